// Orthogonalisation of a weight matrix's update by Newton-Schulz products: the step of an optimiser that moves a matrix
// along the nearest semi-orthogonal matrix to its (averaged) gradient G,
//   X = G / ||G||_F;  `steps` times:  A = X X^T,  B = b A + c A^2,  X = a X + B X,
// X taken with its short side as rows (m <= n; a tall G transposed). Each step maps every singular value s of X to
// a s + b s^3 + c s^5 and leaves the singular vectors alone.
//
// All three products run on v_mfma_f32_32x32x16_f16. float16 and not bf16: every matrix here is bounded (singular
// values stay near 1 or below, checked on the host for the coefficients given), so bf16's range buys nothing and its
// three bits fewer cost: on a gradient with a few strong directions the bf16 iteration ends 3e-2 from the exact one,
// float16 4e-3. X is held as two float16 parts, X = hi + lo (22 bits): the products read hi, and a X, the term that
// carries the small singular values, takes both, so a rounding of X is not multiplied by a in every step: 1e-3 and
// below. All sums are float32. X, A and B are stored times 2^10 (exact), which keeps entries of 1e-4, as a normalised
// large matrix has, clear of float16's smallest normal number; the largest entries, below 8, stay below 2^13.
//
// A's and B's entries are largest on the diagonal (near 1 and 2 at the end), and with few rows their rounding to float16
// there moves a whole singular direction (2e-3 to 4e-3 at 1 to 7 rows, more than the result's own rounding). The
// diagonals are therefore kept in float32 beside the matrices, and what float16 took of them is put back entry by entry:
// with A = Ah + E, E diagonal, A^2 = Ah^2 + E A + A E (E^2 is below 2^-24), and with B = Bh + F and X = H + L,
// B X = Bh H + F H + diag(B) L (L's other products stay out, as everywhere). 1 x 900 to 7 x 659: below 7e-4; 1,001 x 333
// 3.0e-4 -> 2.0e-4.
//
// A and B are symmetric: only the tiles on and below the diagonal are computed and each is stored twice. Sizes are
// padded with zeros to tiles, which changes no entry of any product.
#include "common.h"

#include <math.h>

typedef _Float16 lamq_ns_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lamq_ns_f16x4 __attribute__((ext_vector_type(4)));
typedef float lamq_ns_f32x16 __attribute__((ext_vector_type(16)));
typedef short lamq_ns_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lamq_ns_s4 lamq_ns_lds_s4;
typedef __attribute__((address_space(3))) const lamq_ns_f16x8 lamq_ns_lds_f16x8;

#define NS_T 128                     // output tile
#define NS_K 64                      // depth of a stage
#define NS_OPB (NS_T * NS_K * 2)     // bytes of one operand's stage (16 KB)
#define NS_CUS 256                   // compute units: up to as many tiles, one has a unit (and all its LDS) to itself
#define NS_SMALL_M 128               // a matrix up to this goes through in one workgroup, whole
#define NS_SMALL_N 512
#define NS_PARTS 256                 // partial sums of squares a matrix
#define NS_SCALE 1024.0f             // what X, A and B are stored times
#define NS_UNSCALE (1.0f / 1024.0f)

// what float16 takes of a value
__device__ __forceinline__ float ns_rest(float d) { return d - (float)(_Float16)d; }

__device__ __forceinline__ float ns_load(const float* p) { return *p; }
__device__ __forceinline__ float ns_load(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }

// `m` (up to eight) entries at p, any alignment of the type, zeros past them
typedef uint32_t lamq_ns_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float lamq_ns_f4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void ns_load8(const uint16_t* p, int m, float (&v)[8])
{
    if (m == 8) {
        const lamq_ns_u4 x = *reinterpret_cast<const lamq_ns_u4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(x[i] << 16);
            v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < m ? ns_load(p + i) : 0.0f;
    }
}
__device__ __forceinline__ void ns_load8(const float* p, int m, float (&v)[8])
{
    if (m == 8) {
        const lamq_ns_f4 x = reinterpret_cast<const lamq_ns_f4*>(p)[0], y = reinterpret_cast<const lamq_ns_f4*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = x[i];
            v[4 + i] = y[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < m ? ns_load(p + i) : 0.0f;
    }
}

// The sum over the workgroup of 256, in every thread, in a fixed order.
__device__ __forceinline__ double ns_sum(double x)
{
    __shared__ double s[4];
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    return x;
}

// float64 partial sums of squares of each matrix: float32 squares of a gradient can underflow or overflow
template <typename Elt>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Elt* __restrict__ G, int64_t rows, int64_t cols, int64_t ld,
                                                      int64_t stride, double* __restrict__ parts)
{
    const Elt* g = G + blockIdx.y * stride;
    // by groups of eight columns of a row: whole 16-byte loads at any alignment of the type
    double x = 0.0;
    const int64_t groups = (cols + 7) / 8, n = rows * groups;
    int64_t i = blockIdx.x * 256 + threadIdx.x;
    const int64_t by = 256 * (int64_t)gridDim.x;
    int64_t r = i / groups, c = i % groups;
    const int64_t br = by / groups, bc = by % groups;
    for (; i < n; i += by) {
        const Elt* p = g + r * ld + 8 * c;
        const int m = (int)(cols - 8 * c < 8 ? cols - 8 * c : 8);
        float v[8];
        ns_load8(p, m, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = fma((double)v[e], (double)v[e], x);
        r += br;
        c += bc;
        if (c >= groups) {
            c -= groups;
            ++r;
        }
    }
    x = ns_sum(x);
    if (threadIdx.x == 0) parts[blockIdx.y * gridDim.x + blockIdx.x] = x;
}

// X = G / ||G|| (0 for a zero matrix) as hi + lo float16 parts, times 2^10, [mp][np], rows lx apart, zeros past G; a tall G
// transposed. A workgroup takes 64 x 64 entries of X.
template <typename Elt, bool TALL>
__global__ __launch_bounds__(256) void ns_start_kernel(const Elt* __restrict__ G, int64_t rows, int64_t cols, int64_t ld,
                                                       int64_t stride, const double* __restrict__ parts, int nparts,
                                                       int mp, int lx, uint16_t* __restrict__ hi,
                                                       uint16_t* __restrict__ lo)
{
    const int64_t batch = blockIdx.z;
    const double ss = ns_sum((int)threadIdx.x < nparts ? parts[batch * nparts + threadIdx.x] : 0.0);
    const double f = ss > 0.0 ? (double)NS_SCALE / sqrt(ss) : ss;  // NaN stays
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    const Elt* g = G + batch * stride;
    if constexpr (!TALL) {  // eight entries of a row a lane
        const int x = threadIdx.x & 7;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = r0 + 32 * h + (threadIdx.x >> 3), c = c0 + 8 * x;
            float v[8];
            const int64_t left = cols - c;
            if (r < rows && left > 0)
                ns_load8(g + r * ld + c, left < 8 ? (int)left : 8, v);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            lamq_ns_f16x8 hv, lv;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = (float)((double)v[e] * f);
                hv[e] = (_Float16)y;
                lv[e] = (_Float16)(y - (float)hv[e]);
            }
            const int64_t at = (batch * mp + r) * (int64_t)lx + c;
            *reinterpret_cast<lamq_ns_f16x8*>(hi + at) = hv;
            *reinterpret_cast<lamq_ns_f16x8*>(lo + at) = lv;
        }
    } else {  // along G's rows into LDS, then eight entries of a row of X a lane
        __shared__ float tile[64][65];
        const int x = threadIdx.x & 63;
#pragma unroll 4
        for (int y = threadIdx.x >> 6; y < 64; y += 4) {
            const int64_t r = c0 + y, c = r0 + x;
            tile[x][y] = r < rows && c < cols ? (float)((double)ns_load(g + r * ld + c) * f) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int y = 32 * h + (threadIdx.x >> 3), c = 8 * (threadIdx.x & 7);
            lamq_ns_f16x8 hv, lv;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = tile[y][c + e];
                hv[e] = (_Float16)v;
                lv[e] = (_Float16)(v - (float)hv[e]);
            }
            const int64_t at = (batch * mp + r0 + y) * (int64_t)lx + c0 + c;
            *reinterpret_cast<lamq_ns_f16x8*>(hi + at) = hv;
            *reinterpret_cast<lamq_ns_f16x8*>(lo + at) = lv;
        }
    }
}

// One direct global->LDS load, 16 bytes a lane into m + 16 * lane, from a uniform address and a 32-bit byte offset a lane;
// M0 saved and restored around it, with the wait state its write needs (load_lds16).
__device__ __forceinline__ void ns_load_lds(const uint16_t* base, uint32_t off, uint32_t m)
{
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(m)
                 : "memory");
}

// LDS layouts. An operand whose rows run along the product's depth: rows of 64 entries (128 bytes), 16-byte chunks
// XOR-swizzled by row / 2 % 8 (16 rows at one chunk then touch all 64 banks once). One load takes eight rows, lane l the
// slot l % 8 of row l / 8: chunk l % 8 ^ l / 16, ^ 4 in every other eight rows.
__device__ __forceinline__ uint32_t ns_sw(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4)); }
__device__ __forceinline__ uint32_t ns_off(int64_t ld, int lane)
{
    return (uint32_t)(lane >> 3) * (uint32_t)(2 * ld) + 16u * (uint32_t)((lane & 7) ^ (lane >> 4));
}
// One whose rows are the depth: 64 rows, as two panels of 64 columns, 128 bytes a row; chunks swizzled by 4 (row / 2 % 2)
// for the transposing reads (four rows by four chunks at a time).
__device__ __forceinline__ uint32_t ns_tsw(int row, int chunk)
{
    return (uint32_t)(row * 128 + ((chunk ^ (4 * ((row >> 1) & 1))) << 4));
}
__device__ __forceinline__ uint32_t ns_toff(int64_t ld, int lane)
{
    return (uint32_t)(lane >> 3) * (uint32_t)(2 * ld) + 16u * (uint32_t)((lane & 7) ^ (4 * ((lane >> 4) & 1)));
}

enum NSMode { NS_GRAM, NS_POLY, NS_UPDATE, NS_LAST };

struct NSArgs {
    const uint16_t *p, *q;  // operands: p [..][K] rows of the output; q [..][K] columns (gram, poly) or [K][..] (update)
    int64_t ldp, ldq, sp, sq;
    int K, tiles_m, mp, lx, la;  // rows of X lx apart, of A and B la
    uint16_t *out, *out_lo;  // A, B or the next X's hi; lo (read and written in place)
    const uint16_t* in_hi;   // poly: A; update: X's hi
    float* diag;             // gram: A's diagonal, poly: B's, [..][mp]
    const float* in_diag;    // poly: A's, update: B's
    float a, b, c;
    uint16_t* bf;  // last: the caller's matrix
    int64_t ldb, sb;
    int m, n, tall;
};

// C = P Q^T (gram, poly: lower tiles, each stored twice) or P Q (update, last): tiles of 64 MT x 128. Four waves multiply,
// 32 MT x 64 each, fed from a ring of RING LDS stages; four more load, by direct global->LDS loads, and do nothing else: a
// wave that issues its loads itself stands at them until the unit's queue has taken them, and its products with it (Gram
// product of 9,728 x 2,560 99 -> 73 us).
template <int MODE, int MT, int RING>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, RING == 2 ? 4 : 2))) void ns_product_kernel(NSArgs g)
{
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    constexpr bool AHEAD = RING > 3;              // a stage's first fragments are read in the stage before
    constexpr int PB = 64 * MT * 128;             // bytes of P's part of a stage
    constexpr int STAGE = PB + NS_OPB;
    constexpr int LOADS = 2 * MT + 4;             // a loading wave's loads of a stage
    __shared__ __align__(256) uint8_t lds[RING * STAGE];
    const int lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), wv = wave & 3;
    const int li = lane & 31, half = lane >> 5, grp = lane >> 4, i16 = lane & 15;
    const int64_t batch = blockIdx.y;
    const int id = (int)xcd_remap(blockIdx.x, gridDim.x);
    int I, J;
    if (SYM) {  // tile `id` of the lower triangle, row by row
        I = (int)((sqrtf(8.0f * (float)id + 1.0f) - 1.0f) * 0.5f);
        while (I * (I + 1) / 2 > id) --I;
        while ((I + 1) * (I + 2) / 2 <= id) ++I;
        J = id - I * (I + 1) / 2;
    } else {
        I = id % g.tiles_m;
        J = id / g.tiles_m;
    }
    const uint32_t base = lds_addr(lds);
    const int nst = g.K / NS_K;
    if (wave >= 4) {  // uniform
        const uint16_t* P = g.p + batch * g.sp;
        const uint16_t* Q = g.q + batch * g.sq + (SYM ? (int64_t)J * NS_T * g.ldq : (int64_t)J * NS_T);
        const uint32_t poff = ns_off(g.ldp, lane), qoff = SYM ? ns_off(g.ldq, lane) : ns_toff(g.ldq, lane);
        auto stage = [&](int st) {
            const uint32_t buf = base + (uint32_t)((st % RING) * STAGE);
#pragma unroll
            for (int q = 0; q < 2 * MT; ++q) {
                const int r = 16 * MT * wv + 8 * q;  // of the tile; rows past the matrix (mp is a multiple of 128) read its last
                const int row = I * 64 * MT + r < g.mp ? I * 64 * MT + r : g.mp - 8 - 8 * (1 - (q & 1));
                ns_load_lds(P + row * g.ldp + st * NS_K, q & 1 ? poff ^ 64u : poff, buf + (uint32_t)(128 * r));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (SYM)
                    ns_load_lds(Q + (32 * wv + 8 * q) * g.ldq + st * NS_K, q & 1 ? qoff ^ 64u : qoff,
                                buf + (uint32_t)(PB + 128 * (32 * wv + 8 * q)));
                else
                    ns_load_lds(Q + (st * NS_K + 32 * (wv & 1) + 8 * q) * g.ldq + 64 * (wv >> 1), qoff,
                                buf + (uint32_t)(PB + 8192 * (wv >> 1) + 128 * (32 * (wv & 1) + 8 * q)));
        };
#pragma unroll
        for (int st = 0; st < RING - 1; ++st)
            if (st < nst) stage(st);
        for (int st = 0; st < nst; ++st) {
            // this wave's loads of the stage have landed (of the one after it too, where its fragments are read ahead)
            if (RING > 2 && st + RING - 1 <= nst)
                wait_vm<LOADS * (AHEAD ? RING - 3 : RING - 2)>();
            else
                wait_vm<0>();
            __syncthreads();  // every wave's; the buffer of the stage before is free
            if (st + RING - 1 < nst) stage(st + RING - 1);
        }
        __syncthreads();  // the multiplying waves' last stage is done with
        return;
    }
    const int wm = 32 * MT * (wv >> 1), wn = 64 * (wv & 1);
    // LDS addresses of the fragments: chunk 2 ks + half of a row is the first one's address ^ 32 ks, 32 rows on the same
    // 4,096 bytes on; read transposed, 16 rows are 2,048 bytes and 32 columns ^ 64
    const uint32_t pbase = base + ns_sw(wm + li, half);
    const uint32_t qbase = SYM ? base + PB + ns_sw(wn + li, half)
                               : base + PB + (uint32_t)(8192 * (wn >> 6)) + ns_tsw(8 * half + (i16 >> 2), 2 * (grp & 1) + ((i16 & 3) >> 1)) +
                                     8 * (i16 & 1);
    lamq_ns_f32x16 acc[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
    // the fragments of step ks of the stage in buffer `buf`
    auto frags = [&](int buf, int ks, lamq_ns_f16x8 (&pf)[MT], lamq_ns_f16x8 (&qf)[2]) {
        const uint32_t pa = pbase + (uint32_t)(buf * STAGE), qa = qbase + (uint32_t)(buf * STAGE);
#pragma unroll
        for (int i = 0; i < MT; ++i) pf[i] = *(lamq_ns_lds_f16x8*)(uintptr_t)((pa ^ (32u * ks)) + 4096u * i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (SYM) {
                qf[j] = *(lamq_ns_lds_f16x8*)(uintptr_t)((qa ^ (32u * ks)) + 4096u * j);
            } else {
                // depth 16 ks + 8 half + {0..7} of column wn + 32 j + li: two transposing reads of four each, the second
                // four rows on (whose chunks are swizzled alike)
                const uint32_t at = (qa ^ (64u * j)) + 2048u * ks;
                const lamq_ns_s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lamq_ns_lds_s4*)(uintptr_t)at);
                const lamq_ns_s4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lamq_ns_lds_s4*)(uintptr_t)(at + 512));
                const short __attribute__((ext_vector_type(8))) x = __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
                qf[j] = __builtin_bit_cast(lamq_ns_f16x8, x);
            }
        }
    };
    // What the end of the tile reads, A or X there, is asked for before the products where there are registers for it (a
    // tile that has a unit to itself, whose end nothing else covers: 1.5 us of a launch)
    constexpr bool EARLY = RING > 3;
    static_assert(!EARLY || MT == 2, "the early loads are of one 64-row part of a 128-row tile, always inside X");
    lamq_ns_f16x4 A[MODE == NS_POLY && EARLY ? 2 * MT * 4 : 1];
    lamq_ns_f16x8 H[8], L[8];
    float4 dcol[MODE == NS_POLY && EARLY ? 8 : 1];
    float drow[MODE == NS_POLY && EARLY ? MT : 1], dx = 0.0f;
    const float* D = g.in_diag + batch * g.mp;
    const int r8 = lane >> 3, c8 = lane & 7;
    auto a_at = [&](int i, int j, int r) {
        return (batch * g.mp + I * 64 * MT + wm + 32 * i + li) * (int64_t)g.la + J * NS_T + wn + 32 * j + 8 * r + 4 * half;
    };
    auto x_at = [&](int h, int y) {
        return (batch * g.mp + I * 64 * MT + wm + 64 * h + 8 * y + r8) * (int64_t)g.lx + J * NS_T + wn + 8 * c8;
    };
    auto d_row = [&](int i) { return D[I * 64 * MT + wm + 32 * i + li]; };
    auto d_col = [&](int j, int r) { return *reinterpret_cast<const float4*>(D + J * NS_T + wn + 32 * j + 8 * r + 4 * half); };
    if constexpr (EARLY && MODE == NS_POLY) {
#pragma unroll
        for (int i = 0; i < MT; ++i) drow[i] = d_row(i);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) dcol[4 * j + r] = d_col(j, r);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    A[8 * i + 4 * j + r] = *reinterpret_cast<const lamq_ns_f16x4*>(g.in_hi + a_at(i, j, r));
    }
    if constexpr (EARLY && !SYM) {
        dx = D[I * 64 * MT + wm + lane];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            H[y] = *reinterpret_cast<const lamq_ns_f16x8*>(g.in_hi + x_at(0, y));
            L[y] = *reinterpret_cast<const lamq_ns_f16x8*>(g.out_lo + x_at(0, y));
        }
    }
    lamq_ns_f16x8 pf[2][MT], qf[2][2];
    for (int st = 0; st < nst; ++st) {
        __syncthreads();  // the stage has landed
        if (!AHEAD || st == 0) frags(st % RING, 0, pf[0], qf[0]);
#pragma unroll
        for (int ks = 0; ks < NS_K / 16; ++ks) {
            // the next step's fragments are read before this one's products, in that order
            __builtin_amdgcn_sched_barrier(0);
            if (ks + 1 < NS_K / 16)
                frags(st % RING, ks + 1, pf[(ks + 1) & 1], qf[(ks + 1) & 1]);
            else if (AHEAD && st + 1 < nst)
                frags((st + 1) % RING, 0, pf[0], qf[0]);
            __builtin_amdgcn_sched_barrier(0);
            // a lane's four registers in a row are neighbours of a row of C: the operands exchanged
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qf[ks & 1][j], pf[ks & 1][i], acc[i][j], 0, 0, 0);
        }
    }
    __syncthreads();  // every wave's last stage is done with
    // result: lane's row of C wm + 32 i + li, columns wn + 32 j + 8 r + 4 half + {0..3} in registers 4 r .. 4 r + 3
    if constexpr (SYM) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = I * 64 * MT + wm + 32 * i + li;
            const float er = MODE == NS_POLY ? ns_rest(EARLY ? drow[EARLY ? i : 0] : d_row(i)) : 0.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int col = J * NS_T + wn + 32 * j + 8 * r + 4 * half;
                    const int64_t at = a_at(i, j, r);
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = acc[i][j][4 * r + e];
                    if (MODE == NS_POLY) {
                        const float4 d = EARLY ? dcol[EARLY ? 4 * j + r : 0] : d_col(j, r);
                        const float ec[4] = {ns_rest(d.x), ns_rest(d.y), ns_rest(d.z), ns_rest(d.w)};
                        const lamq_ns_f16x4 a =
                            EARLY ? A[EARLY ? 8 * i + 4 * j + r : 0] : *reinterpret_cast<const lamq_ns_f16x4*>(g.in_hi + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float whole = (float)a[e] + (row == col + e ? er : 0.0f);
                            x[e] = fmaf(g.b, whole, g.c * NS_UNSCALE * fmaf(er + ec[e], whole, x[e]));
                        }
                    } else
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] *= NS_UNSCALE;
                    lamq_ns_f16x4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[e] = (_Float16)x[e];
                        if (row == col + e) g.diag[batch * g.mp + row] = x[e];
                    }
                    *reinterpret_cast<lamq_ns_f16x4*>(g.out + at) = o;
                    if (I != J) {
                        uint16_t* t = g.out + (batch * g.mp + col) * (int64_t)g.la + row;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const _Float16 y = o[e];  // a bit cast of the element itself would read the first one's bits
                            t[(int64_t)e * g.la] = __builtin_bit_cast(uint16_t, y);
                        }
                    }
                }
        }
    } else {
        // through LDS (16 KB a wave, chunks of four floats swizzled by the row), so that X is read and written by rows of
        // 128 bytes: eight lanes a row, eight columns a lane
#pragma unroll
        for (int h = 0; h < MT / 2; ++h) {  // 64 rows at a time
            const int m0 = I * 64 * MT + wm + 64 * h;
            if (m0 >= g.mp) break;  // uniform: past the matrix
            if constexpr (!EARLY) {
                dx = D[m0 + lane];
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    H[y] = *reinterpret_cast<const lamq_ns_f16x8*>(g.in_hi + x_at(h, y));
                    L[y] = *reinterpret_cast<const lamq_ns_f16x8*>(g.out_lo + x_at(h, y));
                }
            }
            float4* tile = reinterpret_cast<float4*>(lds) + wv * 1024;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 32 * i + li, chunk = 8 * j + 2 * r + half, a = 2 * h + i;
                        tile[row * 16 + (chunk ^ (row & 15))] =
                            make_float4(acc[a][j][4 * r], acc[a][j][4 * r + 1], acc[a][j][4 * r + 2], acc[a][j][4 * r + 3]);
                    }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const int row = 8 * y + r8;  // of the wave's 64
                float4* t0 = tile + row * 16 + ((2 * c8) ^ (row & 15));
                float4* t1 = tile + row * 16 + ((2 * c8 + 1) ^ (row & 15));
                const float4 u = *t0, w = *t1;
                float x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                const float d = __shfl(dx, row), ah = fmaf(ns_rest(d), NS_UNSCALE, g.a), al = fmaf(d, NS_UNSCALE, g.a);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = fmaf(ah, (float)H[y][e], fmaf(al, (float)L[y][e], x[e] * NS_UNSCALE));
                if constexpr (MODE == NS_UPDATE) {
                    lamq_ns_f16x8 hv, lv;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        hv[e] = (_Float16)x[e];
                        lv[e] = (_Float16)(x[e] - (float)hv[e]);
                    }
                    *reinterpret_cast<lamq_ns_f16x8*>(g.out + x_at(h, y)) = hv;
                    *reinterpret_cast<lamq_ns_f16x8*>(g.out_lo + x_at(h, y)) = lv;
                } else if (g.tall) {  // back where it was, to be read by columns
                    *t0 = make_float4(x[0], x[1], x[2], x[3]);
                    *t1 = make_float4(x[4], x[5], x[6], x[7]);
                } else {
                    const int m = m0 + row, n = J * NS_T + wn + 8 * c8;
                    if (m < g.m)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (n + e < g.n)
                                g.bf[batch * g.sb + (int64_t)m * g.ldb + n + e] =
                                    __builtin_bit_cast(uint16_t, (__bf16)(x[e] * NS_UNSCALE));
                }
            }
            if constexpr (MODE == NS_LAST) {
                if (g.tall) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const int row = 32 * i + li, chunk = c + half;
                            const float4 u = tile[row * 16 + (chunk ^ (row & 15))];
                            const float x[4] = {u.x, u.y, u.z, u.w};
                            const int m = m0 + row, n = J * NS_T + wn + 4 * chunk;
                            if (m < g.m)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (n + e < g.n)
                                        g.bf[batch * g.sb + (int64_t)(n + e) * g.ldb + m] =
                                            __builtin_bit_cast(uint16_t, (__bf16)(x[e] * NS_UNSCALE));
                        }
                }
            }
        }
    }
}

// A small matrix, whole: m <= 128, n <= 512. One workgroup of 16 waves holds X in LDS as float16 (what the products
// read) and, each wave 32 columns of it, in its accumulators as float32 times 2^10 (what a X takes), A and then B in
// LDS; from G to the result nothing else goes through memory, and all steps are one launch. The diagonals are kept where
// LDS has room for them, up to 96 rows; with more, the rounding averages out over the rows (7e-4). 128 x 320: 100 us by the
// products above (17 launches of about 6 us, latencies all of it), 47 us here.
__device__ __forceinline__ int ns_f(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }  // conflict-free both ways
__device__ __forceinline__ uint32_t ns_xat(int row, int chunk)  // 16-byte chunk of X's row in LDS
{
    return (uint32_t)(row * (2 * NS_SMALL_N) + ((chunk ^ ns_f(row)) << 4));
}
__device__ __forceinline__ uint32_t ns_aat(int row, int chunk)  // and of A's
{
    return (uint32_t)(row * (2 * NS_SMALL_M) + ((chunk ^ ns_f(row)) << 4));
}
// four entries at p, any alignment of the type
typedef uint32_t lamq_ns_u2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ void ns_load4(const uint16_t* p, float (&v)[4])
{
    const lamq_ns_u2 x = *reinterpret_cast<const lamq_ns_u2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[2 * i] = __uint_as_float(x[i] << 16);
        v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void ns_load4(const float* p, float (&v)[4])
{
    const lamq_ns_f4 x = *reinterpret_cast<const lamq_ns_f4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
}
// ENTRIES: G and the result an entry a lane (a tall G, whose rows are X's columns, or rows of fewer than four), else by
// rows. MT: tiles of 32 rows that X has room for; up to three, the diagonals are kept.
template <typename Elt, bool ENTRIES, int MT>
__global__ __launch_bounds__(1024) void ns_small_kernel(const Elt* __restrict__ G, int64_t ld, int64_t stride,
                                                        uint16_t* __restrict__ out, int64_t ldo, int64_t so, int m, int n,
                                                        int tall, int steps, float a, float b, float c)
{
    __shared__ __align__(256) uint8_t xs[NS_SMALL_M * NS_SMALL_N * 2];
    __shared__ __align__(256) uint8_t as[NS_SMALL_M * NS_SMALL_M * 2];
    typedef __attribute__((address_space(3))) lamq_ns_f16x4 lds_f16x4;
    const int lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    int li = lane & 31, half = lane >> 5, i16 = lane & 15;
    const int mt = (m + 31) / 32, nt = (n + 31) / 32;  // tiles of 32
    const uint32_t xb = lds_addr(xs), ab = lds_addr(as);
    G += blockIdx.x * stride;
    out += blockIdx.x * so;
    const int c0 = 32 * wave + 4 * half;  // X's rows 32 i + li, columns c0 + 8 r + {0..3}
    constexpr bool EXACT = MT < NS_SMALL_M / 32;
    lamq_ns_f32x16 X[MT];
    double ss = 0.0;
    // No load is conditional (a branch would wait for each in turn): past the matrix the address is held inside it and the
    // value left out.
    if constexpr (ENTRIES) {
        const int64_t sr = tall ? 1 : ld, sc = tall ? ld : 1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = 32 * i + li;
            const Elt* g = G + (row < m ? row : m - 1) * sr;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int col = c0 + 8 * (v >> 2) + (v & 3);
                X[i][v] = ns_load(g + (col < n ? col : n - 1) * sc);
            }
        }
    } else {
        // eight lanes a row of 32 columns, then into the lanes' own places through LDS, 64 rows (8 KB a wave) at a time
        const int cc = 32 * wave + 4 * (lane & 7), at = cc < n - 4 ? cc : n - 4, shift = cc - at;  // past the row by `shift`
        float4* t = reinterpret_cast<float4*>(xs) + 512 * wave;
#pragma unroll
        for (int h = 0; h < (MT + 1) / 2; ++h) {
            __builtin_amdgcn_sched_barrier(0);
            float x[8][4];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int row = 64 * h + 8 * q + (lane >> 3);
                ns_load4(G + (row < m ? row : m - 1) * ld + at, x[q]);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int y = 8 * q + (lane >> 3);
                const float s0 = shift & 1 ? x[q][1] : x[q][0], s1 = shift & 1 ? x[q][2] : x[q][1],
                            s2 = shift & 1 ? x[q][3] : x[q][2], s3 = x[q][3];
                // (what moves past the end is left out below, whatever it is)
                t[8 * y + ((lane & 7) ^ (y & 7))] = make_float4(shift & 2 ? s2 : s0, shift & 2 ? s3 : s1, s2, s3);
            }
#pragma unroll
            for (int i = 0; i < 2 && 2 * h + i < MT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int y = 32 * i + li;
                    const float4 v = t[8 * y + ((2 * r + half) ^ (y & 7))];
                    X[2 * h + i][4 * r] = v.x;
                    X[2 * h + i][4 * r + 1] = v.y;
                    X[2 * h + i][4 * r + 2] = v.z;
                    X[2 * h + i][4 * r + 3] = v.w;
                }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            X[i][v] = 32 * i + li < m && c0 + 8 * (v >> 2) + (v & 3) < n ? X[i][v] : 0.0f;
            ss = fma((double)X[i][v], (double)X[i][v], ss);
        }
    {
        double* sums = reinterpret_cast<double*>(as);
        for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
        if (lane == 0) sums[wave] = ss;
        __syncthreads();
        ss = 0.0;
        for (int w = 0; w < 16; ++w) ss += sums[w];
    }
    const double f = ss > 0.0 ? (double)NS_SCALE / sqrt(ss) : ss;  // NaN stays
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) X[i][v] = (float)((double)X[i][v] * f);
    const int ti = wave >> 2, tj = wave & 3;  // this wave's tile of A and B
    const bool mine = ti < mt && tj < mt, cols = wave < nt;  // uniform
    float* dA = reinterpret_cast<float*>(as + (NS_SMALL_M - 32) * NS_SMALL_M * 2);  // A's and B's diagonals, where A has no rows
    float* dB = dA + NS_SMALL_M;
    for (int step = 0; step < steps; ++step) {
        asm volatile("" : "+v"(li), "+v"(half), "+v"(i16));  // addresses are formed where they are used, not kept around the loop
        if (cols)  // X as float16
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (i < mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        lamq_ns_f16x4 h;
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = (_Float16)X[i][4 * r + e];
                        *(lds_f16x4*)(uintptr_t)(xb + ns_xat(32 * i + li, 4 * wave + r) + 8 * half) = h;
                    }
        __syncthreads();  // X is there; B of the step before (and the sums) are read
        lamq_ns_f32x16 T;
        auto at = [&](int r) { return (lds_f16x4*)(uintptr_t)(ab + ns_aat(32 * ti + li, 4 * tj + r) + 8 * half); };
        if (mine) {
#pragma unroll
            for (int v = 0; v < 16; ++v) T[v] = 0.0f;
            for (int ks = 0; ks < 2 * nt; ++ks) {
                const lamq_ns_f16x8 p = *(lamq_ns_lds_f16x8*)(uintptr_t)(xb + ns_xat(32 * ti + li, 2 * ks + half));
                const lamq_ns_f16x8 q = *(lamq_ns_lds_f16x8*)(uintptr_t)(xb + ns_xat(32 * tj + li, 2 * ks + half));
                T = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, p, T, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                lamq_ns_f16x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    T[4 * r + e] *= NS_UNSCALE;
                    h[e] = (_Float16)T[4 * r + e];
                    if (EXACT && ti == tj && li == 8 * r + 4 * half + e) dA[32 * ti + li] = T[4 * r + e];
                }
                *at(r) = h;
            }
        }
        __syncthreads();
        if (mine) {
#pragma unroll
            for (int v = 0; v < 16; ++v) T[v] = 0.0f;
            for (int ks = 0; ks < 2 * mt; ++ks) {
                const lamq_ns_f16x8 p = *(lamq_ns_lds_f16x8*)(uintptr_t)(ab + ns_aat(32 * ti + li, 2 * ks + half));
                const lamq_ns_f16x8 q = *(lamq_ns_lds_f16x8*)(uintptr_t)(ab + ns_aat(32 * tj + li, 2 * ks + half));
                T = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, p, T, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const lamq_ns_f16x4 h = *at(r);
                if constexpr (EXACT) {
                    const float er = ns_rest(dA[32 * ti + li]);
                    const float4 d = *reinterpret_cast<const float4*>(dA + 32 * tj + 8 * r + 4 * half);
                    const float ec[4] = {ns_rest(d.x), ns_rest(d.y), ns_rest(d.z), ns_rest(d.w)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool on = ti == tj && li == 8 * r + 4 * half + e;
                        const float whole = (float)h[e] + (on ? er : 0.0f);
                        T[4 * r + e] = fmaf(b, whole, c * NS_UNSCALE * fmaf(er + ec[e], whole, T[4 * r + e]));
                        if (on) dB[32 * ti + li] = T[4 * r + e];
                    }
                } else
#pragma unroll
                    for (int e = 0; e < 4; ++e) T[4 * r + e] = fmaf(b, (float)h[e], c * (T[4 * r + e] * NS_UNSCALE));
            }
        }
        __syncthreads();  // A is read
        if (mine)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                lamq_ns_f16x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = (_Float16)T[4 * r + e];
                *at(r) = h;
            }
        __syncthreads();
        if (cols) {  // X = a X + B X, onto 2^10 a X
#pragma unroll
            for (int i = 0; i < MT; ++i)
                if (EXACT) {  // and F H + diag(B) (X - H), F = diag(B) - Bh's (rows from 32 mt on are never read)
                    const float d = dB[32 * i + li], up = fmaf(a, NS_SCALE, d), dh = -(float)(_Float16)d;
#pragma unroll
                    for (int v = 0; v < 16; ++v) X[i][v] = fmaf(up, X[i][v], dh * (float)(_Float16)X[i][v]);
                } else
#pragma unroll
                    for (int v = 0; v < 16; ++v) X[i][v] *= a * NS_SCALE;
            for (int ks = 0; ks < 2 * mt; ++ks) {
                // depth 16 ks + 8 half + {0..7} of a column: two transposing reads of four rows each
                const int row = 16 * ks + 8 * half + (i16 >> 2), chunk = 4 * wave + 2 * (li >> 4) + ((i16 & 3) >> 1);
                const lamq_ns_s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lamq_ns_lds_s4*)(uintptr_t)(xb + ns_xat(row, chunk) + 8 * (i16 & 1)));
                const lamq_ns_s4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lamq_ns_lds_s4*)(uintptr_t)(xb + ns_xat(row + 4, chunk) + 8 * (i16 & 1)));
                const short __attribute__((ext_vector_type(8))) y = __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
                const lamq_ns_f16x8 q = __builtin_bit_cast(lamq_ns_f16x8, y);
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    if (i < mt) {
                        const lamq_ns_f16x8 p = *(lamq_ns_lds_f16x8*)(uintptr_t)(ab + ns_aat(32 * i + li, 2 * ks + half));
                        X[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, p, X[i], 0, 0, 0);
                    }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) X[i][v] *= NS_UNSCALE;
        }
        __syncthreads();  // X and B are read
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 32 * i + li, col = c0 + 8 * r;
            uint16_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_bit_cast(uint16_t, (__bf16)(X[i][4 * r + e] * NS_UNSCALE));
            if (!ENTRIES && row < m && col + 4 <= n) {
                const lamq_ns_u2 w = {(uint32_t)y[0] | ((uint32_t)y[1] << 16), (uint32_t)y[2] | ((uint32_t)y[3] << 16)};
                *reinterpret_cast<lamq_ns_u2*>(out + row * ldo + col) = w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row < m && col + e < n) out[tall ? (col + e) * ldo + row : row * ldo + col + e] = y[e];
            }
        }
}

// G as bf16: the result of no step at all
template <typename Elt>
__global__ __launch_bounds__(256) void ns_copy_kernel(const Elt* __restrict__ G, int64_t rows, int64_t cols, int64_t ld,
                                                      int64_t stride, const double* __restrict__ parts, int nparts,
                                                      uint16_t* __restrict__ out, int64_t ldo, int64_t so)
{
    const double ss = ns_sum((int)threadIdx.x < nparts ? parts[blockIdx.y * nparts + threadIdx.x] : 0.0);
    const double f = ss > 0.0 ? 1.0 / sqrt(ss) : ss;
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += 256 * (int64_t)gridDim.x) {
        const int64_t r = i / cols, c = i % cols;
        const float v = (float)((double)ns_load(G + blockIdx.y * stride + r * ld + c) * f);
        out[blockIdx.y * so + r * ldo + c] = __builtin_bit_cast(uint16_t, (__bf16)v);
    }
}

struct NSPlan {
    int64_t m, n, mp, np, lx, la;
    size_t x, aa, total;  // bytes of one [mp][lx] and [mp][la] array over the batch, and of everything
};
static NSPlan ns_plan(int64_t batch, int64_t rows, int64_t cols)
{
    NSPlan p;
    p.m = rows < cols ? rows : cols;
    p.n = rows < cols ? cols : rows;
    p.mp = cdiv(p.m, NS_T) * NS_T;
    p.np = cdiv(p.n, NS_T) * NS_T;
    // rows an odd number of 128 bytes apart: at a multiple of 256 the eight rows a load takes fall on few of the memory's
    // channels
    p.lx = p.np + 64;
    p.la = p.mp + 64;
    p.x = (size_t)batch * p.mp * p.lx * 2;
    p.aa = (size_t)batch * p.mp * p.la * 2;
    p.total = (size_t)batch * NS_PARTS * sizeof(double) + 3 * p.x + 2 * p.aa + 2 * (size_t)batch * p.mp * sizeof(float);
    return p;
}

extern "C" size_t lamq_orthogonalize_workspace_size(int64_t batch, int64_t rows, int64_t cols)
{
    if (batch < 1 || rows < 1 || cols < 1) return 0;
    return ns_plan(batch, rows, cols).total;
}

// The largest singular value that any step reaches from [0, 1], on a grid of them: what the float16 range is checked
// against.
static double ns_reach(int steps, double a, double b, double c)
{
    double s[256], top = 1.0;
    for (int i = 0; i < 256; ++i) s[i] = (i + 1) / 256.0;
    for (int k = 0; k < steps && top < 1e6; ++k)
        for (int i = 0; i < 256; ++i) {
            s[i] = s[i] * (a + s[i] * s[i] * (b + s[i] * s[i] * c));
            top = fabs(s[i]) <= top ? top : fabs(s[i]) < 1e6 ? fabs(s[i]) : 1e6;  // a NaN counts as past it
        }
    return top;
}

template <typename Elt>
static int ns_launch(const Elt* G, int64_t batch, int64_t rows, int64_t cols, int64_t ld, int64_t stride, int steps, float a,
                     float b, float c, uint16_t* out, int64_t ldo, int64_t so, void* workspace, size_t workspace_bytes,
                     void* stream)
{
    if (!G || !out || batch < 0 || rows < 0 || cols < 0 || steps < 0 || ld < cols || ldo < cols) return LAMQ_EINVAL;
    if (batch > 1 && (stride < 0 || so < rows * ldo)) return LAMQ_EINVAL;
    if ((uintptr_t)G % sizeof(Elt) || (uintptr_t)out % 2) return LAMQ_EINVAL;
    if (!(ns_reach(steps, a, b, c) <= 8.0)) return LAMQ_EINVAL;
    if (batch == 0 || rows == 0 || cols == 0) return LAMQ_OK;
    if (batch > 65535 || rows > (1 << 20) || cols > (1 << 20)) return LAMQ_EUNSUP;
    const NSPlan p = ns_plan(batch, rows, cols);
    if (p.mp * p.np > ((int64_t)1 << 36)) return LAMQ_EUNSUP;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < p.total) return LAMQ_EINVAL;
    hipStream_t st = as_stream(stream);
    const bool tall = rows > cols;
    if (p.m <= NS_SMALL_M && p.n <= NS_SMALL_N && steps > 0) {
        const bool entries = tall || p.n < 4, few = p.m <= 96;
        hipLaunchKernelGGL((few ? entries ? ns_small_kernel<Elt, true, 3> : ns_small_kernel<Elt, false, 3>
                            : entries ? ns_small_kernel<Elt, true, 4> : ns_small_kernel<Elt, false, 4>),
                           dim3((unsigned)batch), dim3(1024), 0, st, G, ld, stride, out, ldo, so, (int)p.m, (int)p.n, (int)tall,
                           steps, a, b, c);
        LAMQ_LAUNCH_CHECK();
        return LAMQ_OK;
    }
    double* parts = reinterpret_cast<double*>(workspace);
    uint8_t* at = reinterpret_cast<uint8_t*>(parts + batch * NS_PARTS);
    uint16_t* hi[2] = {reinterpret_cast<uint16_t*>(at), reinterpret_cast<uint16_t*>(at + p.x)};
    uint16_t* lo = reinterpret_cast<uint16_t*>(at + 2 * p.x);
    uint16_t* A = reinterpret_cast<uint16_t*>(at + 3 * p.x);
    uint16_t* Bm = reinterpret_cast<uint16_t*>(at + 3 * p.x + p.aa);
    float* dA = reinterpret_cast<float*>(at + 3 * p.x + 2 * p.aa);
    float* dB = dA + batch * p.mp;
    const int64_t want = cdiv(rows * cols, 4096);
    const int nparts = (int)(want < NS_PARTS ? want : NS_PARTS);
    hipLaunchKernelGGL(ns_norm_kernel<Elt>, dim3(nparts, (unsigned)batch), dim3(256), 0, st, G, rows, cols, ld, stride, parts);
    LAMQ_LAUNCH_CHECK();
    if (steps == 0) {
        hipLaunchKernelGGL(ns_copy_kernel<Elt>, dim3(nparts, (unsigned)batch), dim3(256), 0, st, G, rows, cols, ld, stride,
                           parts, nparts, out, ldo, so);
        LAMQ_LAUNCH_CHECK();
        return LAMQ_OK;
    }
    const dim3 sg((unsigned)(p.np / 64), (unsigned)(p.mp / 64), (unsigned)batch);
    if (tall)
        hipLaunchKernelGGL((ns_start_kernel<Elt, true>), sg, dim3(256), 0, st, G, rows, cols, ld, stride, parts, nparts,
                           (int)p.mp, (int)p.lx, hi[0], lo);
    else
        hipLaunchKernelGGL((ns_start_kernel<Elt, false>), sg, dim3(256), 0, st, G, rows, cols, ld, stride, parts, nparts,
                           (int)p.mp, (int)p.lx, hi[0], lo);
    LAMQ_LAUNCH_CHECK();
    const int tm = (int)(p.mp / NS_T), tn = (int)(p.np / NS_T);
    NSArgs x{};
    x.lx = (int)p.lx;
    x.la = (int)p.la;
    x.mp = (int)p.mp;
    x.a = a;
    x.b = b;
    x.c = c;
    x.out_lo = lo;
    x.bf = out;
    x.ldb = ldo;
    x.sb = so;
    x.m = (int)p.m;
    x.n = (int)p.n;
    x.tall = tall;
    const dim3 lower((unsigned)(tm * (tm + 1) / 2), (unsigned)batch);
    // A ring of four stages (all of a unit's LDS) where every tile has a unit to itself, two where two tiles share one (X X^T,
    // four / two: 6 tiles 10.9 / 14.7 us, 72 19.2 / 29.4, 210 74 / 98, 300 56 / 46; updates: 144 tiles 18.5 / 20.6, 320 25.4 /
    // 20.0). Updates take tiles of 256 rows, a third less of X and B through LDS, where two rounds of them fill the chip
    // (9,728 x 2,560, 760 tiles: 134 us, of 128 rows 137; 2 x 1,024 x 2,560, 160 tiles: 21.9 us, of 128 rows 19.6)
    const int64_t tiles = (int64_t)tm * tn * batch, tall_tiles = (int64_t)((tm + 1) / 2) * tn * batch;
    const bool alone = (int64_t)lower.x * batch <= NS_CUS, wide = tall_tiles >= 2 * NS_CUS, apart = tiles <= NS_CUS;
    x.tiles_m = wide ? (tm + 1) / 2 : tm;
    const dim3 full((unsigned)(x.tiles_m * tn), (unsigned)batch), wg(512);
    for (int k = 0; k < steps; ++k) {
        NSArgs y = x;
        y.p = y.q = hi[k & 1];
        y.ldp = y.ldq = p.lx;
        y.sp = y.sq = p.mp * p.lx;
        y.K = (int)p.np;
        y.out = A;
        y.diag = dA;
        hipLaunchKernelGGL((alone ? ns_product_kernel<NS_GRAM, 2, 4> : ns_product_kernel<NS_GRAM, 2, 2>), lower, wg, 0, st, y);
        LAMQ_LAUNCH_CHECK();
        y.p = y.q = y.in_hi = A;
        y.ldp = y.ldq = p.la;
        y.sp = y.sq = p.mp * p.la;
        y.K = (int)p.mp;
        y.out = Bm;
        y.in_diag = dA;
        y.diag = dB;
        hipLaunchKernelGGL((alone ? ns_product_kernel<NS_POLY, 2, 4> : ns_product_kernel<NS_POLY, 2, 2>), lower, wg, 0, st, y);
        LAMQ_LAUNCH_CHECK();
        y.p = Bm;
        y.q = y.in_hi = hi[k & 1];
        y.ldq = p.lx;
        y.sq = p.mp * p.lx;
        y.in_diag = dB;
        y.out = hi[1 - (k & 1)];
        if (k + 1 < steps)
            hipLaunchKernelGGL((wide ? ns_product_kernel<NS_UPDATE, 4, 3> : apart ? ns_product_kernel<NS_UPDATE, 2, 4> : ns_product_kernel<NS_UPDATE, 2, 2>), full, wg, 0,
                               st, y);
        else
            hipLaunchKernelGGL((wide ? ns_product_kernel<NS_LAST, 4, 3> : apart ? ns_product_kernel<NS_LAST, 2, 4> : ns_product_kernel<NS_LAST, 2, 2>), full, wg, 0, st,
                               y);
        LAMQ_LAUNCH_CHECK();
    }
    return LAMQ_OK;
}

extern "C" int lamq_orthogonalize_bf16(const uint16_t* G, int64_t batch, int64_t rows, int64_t cols, int64_t ld,
                                       int64_t stride, int steps, float a, float b, float c, uint16_t* out, int64_t ldo,
                                       int64_t so, void* workspace, size_t workspace_bytes, void* stream)
{
    return ns_launch(G, batch, rows, cols, ld, stride, steps, a, b, c, out, ldo, so, workspace, workspace_bytes, stream);
}

extern "C" int lamq_orthogonalize_f32(const float* G, int64_t batch, int64_t rows, int64_t cols, int64_t ld,
                                      int64_t stride, int steps, float a, float b, float c, uint16_t* out, int64_t ldo,
                                      int64_t so, void* workspace, size_t workspace_bytes, void* stream)
{
    return ns_launch(G, batch, rows, cols, ld, stride, steps, a, b, c, out, ldo, so, workspace, workspace_bytes, stream);
}
