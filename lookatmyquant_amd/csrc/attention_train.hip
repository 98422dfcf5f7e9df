// The causal grouped-query attention of training: a forward that takes the sequences' lengths and keeps the log-sum-exp
// of every query's scores, and the backward pass, which recomputes the probabilities from it tile by tile; they never
// reach memory.
//
// With S = scale Q K^T over u <= t < len, lse_t = log sum_u exp S_tu, P = exp(S - lse), O = P V and dO the gradient of O:
//   delta_t = sum_d dO_td O_td,  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,  dK and dV summed over a key/value head's query heads.
//
// The forward owns 128 queries a workgroup and walks the keys with a running maximum and sum. The backward is two
// kernels, so that each gradient has one owner and its sums one order (no atomics): attention_dq_kernel owns 128
// queries and walks the keys up to them, forming S^T, dP^T and dQ^T += K^T dS^T; attention_dkdv_kernel owns 64 keys and
// walks the query heads and queries from them on, forming S, dP, dV^T += dO^T P and dK^T += Q^T dS. Seven products where
// five would do with one pass; the two formed twice cost less than a float32 dQ added up in memory (a read and a
// write of 4 bytes per query, head dim and key block) and keep the results the same from run to run.
//
// Operand layouts (32x32x16 bf16 MFMA): A[m][k] has lane l holding m = l % 32 and k = 8 (l / 32) .. + 7; B[k][n] has lane
// l holding n = l % 32 and the same k; the result has lane l holding column l % 32 and rows 8 (v / 4) + 4 (l / 32) + v % 4 of
// register v. With the owned rows as columns of the result, S^T (or S)
// and dP come out as the second product's B operand as they stand, and that product's A operand is the walked tile read
// transposed (ds_read_b64_tr_b16) in the result's own order. A walked tile is read both ways, so its 16-byte chunks are
// XOR-swizzled by at_f(row), the row's two low bit pairs exchanged: 16 rows at one chunk touch 16 different chunk
// slots, and so do the four rows and four chunks a transposing read serves at once.
//
// P is rounded to bf16 for dV as the forward rounds it for O, dS to bf16 for dQ and dK, the operand type of the matrix
// instructions; scores, dP, delta and every sum are float32, each gradient rounded once at its end. delta is a sum of
// products with O, and where dP - delta is small beside either, O's own rounding would show in dQ and dK (two or three
// times the rounding of the result, over sequences of a few tokens): the forward leaves what the rounding took, a second
// bf16 part, for it. Over short sequences the roundings of P and dS stay as large as the results' own, or larger where
// few terms cancel; up to 128 tokens, where launches and latencies set the time, P and dS go into their products as two
// bf16 parts.
#include "common.h"

typedef __bf16 lamq_at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float lamq_at_f32x16 __attribute__((ext_vector_type(16)));
typedef short lamq_at_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lamq_at_s4 lamq_at_lds_s4;
typedef __attribute__((address_space(3))) const lamq_at_bf16x8 lamq_at_lds_frag;

#define AT_GRID_X (1 << 22)
#define AT_D 128                        // head dim
#define AT_LOG2E 1.4426950408889634f

// the larger of this lane's value and lane ^ 32's (one swap of the wave's halves, no LDS)
__device__ __forceinline__ float at_max32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_sum32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// what bf16 takes of a value, as bf16 (nothing of an infinity)
__device__ __forceinline__ __bf16 at_second(float x)
{
    const float r = x - (float)(__bf16)x;
    return (__bf16)(r == r ? r : 0.0f);
}

// the length of sequence b, 0 .. T (all T without lengths)
__device__ __forceinline__ int at_length(const int32_t* __restrict__ lens, int b, int T)
{
    if (!lens) return T;
    const int n = __builtin_amdgcn_readfirstlane(lens[b]);
    return n < 0 ? 0 : n < T ? n : T;
}

// zeros into rows first .. last - 1 of 128 bf16 at `row` (a workgroup of 256, eight bytes a lane: the alignment asked
// of outputs)
__device__ __forceinline__ void at_zero_rows(uint16_t* base, int64_t stride, int first, int last)
{
    for (int i = (int)threadIdx.x; i < (last - first) * (AT_D / 4); i += 256)
        *reinterpret_cast<uint2*>(base + (int64_t)(first + i / (AT_D / 4)) * stride + 4 * (i % (AT_D / 4))) =
            make_uint2(0u, 0u);
}

// One operand by its (batch, head, token) strides in elements, the head dim contiguous.
struct AtView {
    const uint16_t* p;
    int64_t sb, sh, st;
};
struct AtOut {
    uint16_t* p;
    int64_t sb, sh, st;
};

// One direct global->LDS load (16 bytes a lane into m0 + 16 * lane) from a uniform address and a 32-bit byte offset a
// lane; M0 saved and restored around it, with the wait state its write needs (load_lds16).
__device__ __forceinline__ void at_load_lds16(const uint16_t* base, uint32_t off, uint32_t m)
{
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(m)
                 : "memory");
}

#define AG_LAZY 8.0f                  // log 2 of how far the forward's maximum may lag
#define AG_R 32                       // rows a wave owns
#define AG_W 64                       // rows of a walked block
#define AG_OWN 128                    // queries a workgroup owns
#define AG_KEYS 64                    // keys a workgroup owns
#define AG_OPB (AG_W * AT_D * 2)      // bytes of one operand's block (16 KB)
#define AG_HALF (AG_OPB / 2)          // ... and of 32 of its rows

__device__ __forceinline__ int at_f(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }
__device__ __forceinline__ uint32_t at_fsw(int row, int chunk)
{
    return (uint32_t)(row * (AT_D * 2) + ((chunk ^ at_f(row)) << 4));
}

// A block of walked rows into LDS (at_load_lds16): wave wv's instruction q fills rows 16 wv + 4 q .. + 3, lane l the
// slot l % 16 of row 16 wv + 4 q + l / 16 with the chunk that belongs there. Of fewer than 64 rows the ones past the
// last read the last one (and meet probabilities of 0).
__device__ __forceinline__ void ag_load_block(const uint16_t* block, int64_t st, int rows, int wv, int lane, uint32_t buf)
{
    const int sub = lane >> 4;
    uint32_t chunk = 16u * (uint32_t)((lane & 15) ^ (sub << 2));  // of q = 0; q's is chunk ^ 16 q
    uint32_t off = (uint32_t)sub * (uint32_t)(2 * st);
    asm volatile("" : "+v"(chunk), "+v"(off));  // formed here, not kept in eight registers around the loop
    if (rows >= AG_W) {
        const uint16_t* p = block + 16 * wv * st;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            at_load_lds16(p + 4 * q * st, off + (chunk ^ (16u * q)), buf + (uint32_t)((4 * wv + q) * 1024));
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = 16 * wv + 4 * q + sub;
            at_load_lds16(block, (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)(2 * st) + (chunk ^ (16u * q)),
                          buf + (uint32_t)((4 * wv + q) * 1024));
        }
    }
}

// LDS addresses of a lane's operand fragments in a block (64 rows of 256 bytes, aligned to 256), from two bases:
// A operand of a product over the head dim: row `row` (32 hf + li), head dims 16 j + 8 hi .. + 7, chunk 2 j + hi.
__device__ __forceinline__ uint32_t ag_frag_base(int row, int hi) { return at_fsw(row, hi); }
__device__ __forceinline__ lamq_at_bf16x8 ag_frag(uint32_t base, int j, uint32_t block)
{
    return *(lamq_at_lds_frag*)(uintptr_t)((base ^ (32u * j)) + block);
}
// A operand of a product over the walked rows: head dims 32 t + li, rows 32 hf + 16 mi + 4 hi + {0..3} and + 8 (the row
// eight further on differs by 2 in at_f, the one sixteen further on not at all).
__device__ __forceinline__ uint32_t ag_tr_base(int hf, int lane)
{
    const int i16 = lane & 15, col = 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
    return at_fsw(32 * hf + 4 * (lane >> 5) + (i16 >> 2), col >> 3) + 8 * ((col >> 2) & 1);
}
__device__ __forceinline__ lamq_at_bf16x8 ag_tr_frag(uint32_t base, int mi, int t, uint32_t block)
{
    const uint32_t a0 = (base ^ (64u * t)) + block + 4096u * mi, a1 = (base ^ (64u * t) ^ 32u) + block + 4096u * mi + 2048u;
    const lamq_at_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lamq_at_lds_s4*)(uintptr_t)a0);
    const lamq_at_s4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lamq_at_lds_s4*)(uintptr_t)a1);
    const short __attribute__((ext_vector_type(8))) w = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(lamq_at_bf16x8, w);
}

// eight consecutive head-dim values of a row
__device__ __forceinline__ lamq_at_bf16x8 ag_row8(const uint16_t* p)
{
    return *reinterpret_cast<const lamq_at_bf16x8*>(p);
}

// the waits of the loads behind these fragments, before the loop whose own waits the compiler does not see
__device__ __forceinline__ void ag_settle(lamq_at_bf16x8 (&f)[8])
{
    asm volatile("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]), "+v"(f[4]), "+v"(f[5]), "+v"(f[6]), "+v"(f[7]));
}

// O's second part is kept by blocks of 32 queries, [16 chunks of 8 head dims][32 queries][8]: the writer's 8 bytes a lane
// and the reader's 16 are 512 bytes in a row a load or store. The offset of a query's first chunk.
__device__ __forceinline__ int64_t ag_rest(int head, int T, int q0, int li)
{
    return ((int64_t)head * ((T + 31) / 32) + q0 / 32) * (32 * AT_D) + 8 * li;
}

// a transposed 128 x 32 result (four tiles: head dims 32 t + 8 r + 4 hi + {0..3} of the lane's row) times `scale`, as
// bf16 (nearest, ties to even) into the row; what the rounding leaves of it, as bf16 again, into `rest` if there is one
__device__ __forceinline__ void ag_store_row(uint16_t* row, const lamq_at_f32x16 (&acc)[4], float scale, int hi,
                                             uint16_t* rest = nullptr)
{
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            uint32_t w2[2], l2[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f0 = acc[t][4 * r + 2 * e] * scale, f1 = acc[t][4 * r + 2 * e + 1] * scale;
                const __bf16 x0 = (__bf16)f0, x1 = (__bf16)f1;
                const __bf16 y0 = (__bf16)(f0 - (float)x0), y1 = (__bf16)(f1 - (float)x1);
                w2[e] = (uint32_t)__builtin_bit_cast(uint16_t, x0) | ((uint32_t)__builtin_bit_cast(uint16_t, x1) << 16);
                l2[e] = (uint32_t)__builtin_bit_cast(uint16_t, y0) | ((uint32_t)__builtin_bit_cast(uint16_t, y1) << 16);
            }
            *reinterpret_cast<uint2*>(row + 32 * t + 8 * r + 4 * hi) = make_uint2(w2[0], w2[1]);
            if (rest) *reinterpret_cast<uint2*>(rest + (4 * t + r) * 256) = make_uint2(l2[0], l2[1]);
        }
}

// workgroup -> (pair of sequence and key/value head, index in the pair's `per`): the pairs spread over the XCDs, so that
// those that read the same keys and values run on one XCD together. False past the last workgroup.
__device__ __forceinline__ bool ag_place(int pairs, int per, int& pair, int& rem)
{
    const int id = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if ((unsigned)id >= (unsigned)pairs * (unsigned)per) return false;
    if (pairs % LAMQ_XCDS == 0) {
        const int y = id / LAMQ_XCDS;
        pair = y / per * LAMQ_XCDS + id % LAMQ_XCDS;
        rem = y % per;
    } else {
        pair = id / per;
        rem = id % per;
    }
    return true;
}

// The forward: O and the log-sum-exp. Per block of 64 keys a wave forms S^T = K Q^T (two tiles of 32 keys x 32 queries),
// the block's maxima, P = exp2(scale S - m) and O^T += V^T P^T. m is the running maximum as of the last time some query's
// maximum had grown by more than 2^AG_LAZY: until then P is at most that, which bf16 and the float32 sums take as they
// are, and the 64 products that rescale O are left out (with the exact maximum some query of 32 grows in most blocks).
// The sums of a query's two lanes are added at the end. 4 x 32 heads x 2,048: 195 -> 162 us against the exact maximum and
// 32 keys a step.
template <bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_lse_kernel(
    AtView Q, AtView K, AtView V, AtOut O, uint16_t* __restrict__ rest, float* __restrict__ lse,
    const int32_t* __restrict__ lens, int rep, int Hkv, int pairs, int Tall, float scale_log2)
{
    __shared__ __align__(256) uint8_t lds[2][2][AG_OPB];  // [buffer][K, V]
    const int nqb = (Tall + AG_OWN - 1) / AG_OWN;
    int pair, rem;
    if (!ag_place(pairs, nqb * rep, pair, rem)) return;
    const int qb = nqb - 1 - rem / rep;  // the longest query blocks first
    const int b = pair / Hkv, hk = pair % Hkv, h = hk * rep + rem % rep;
    const int lane = (int)(threadIdx.x & 63), wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int li = lane & 31, hi = lane >> 5;
    const int T = at_length(lens, b, Tall);
    uint16_t* Op = O.p + b * O.sb + (int64_t)h * O.sh;
    float* L = lse + ((int64_t)b * Hkv * rep + h) * Tall;
    const int own0 = qb * AG_OWN, own1 = own0 + AG_OWN < Tall ? own0 + AG_OWN : Tall;
    if (own1 > T) {
        const int first = own0 > T ? own0 : T;
        at_zero_rows(Op, O.st, first, own1);
        for (int t = first + (int)threadIdx.x; t < own1; t += 256) L[t] = -__builtin_inff();
        if (own0 >= T) return;  // uniform, before any barrier
    }
    const int q0 = own0 + AG_R * wv, myq = q0 + li, qrow = myq < T ? myq : T - 1;
    const uint16_t* Kp = K.p + b * K.sb + (int64_t)hk * K.sh;
    const uint16_t* Vp = V.p + b * V.sb + (int64_t)hk * V.sh;
    const uint32_t base = lds_addr(lds);
    const int nblk = ((own1 < T ? own1 : T) - 1) / AG_W + 1;
    const int my_last = q0 < T ? (q0 + AG_R < T ? q0 + AG_R : T) - 1 : -1;
    auto load_block = [&](int kb) {
        const uint32_t buf = base + (uint32_t)((kb & 1) * 2 * AG_OPB);
        const int r0 = kb * AG_W;
        ag_load_block(Kp + r0 * K.st, K.st, T - r0, wv, lane, buf);
        ag_load_block(Vp + r0 * V.st, V.st, T - r0, wv, lane, buf + AG_OPB);
    };
    load_block(0);
    lamq_at_bf16x8 qf[8];
    {
        const uint16_t* Qr = Q.p + b * Q.sb + (int64_t)h * Q.sh + (int64_t)qrow * Q.st + 8 * hi;
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[j] = ag_row8(Qr + 16 * j);
    }
    ag_settle(qf);
    lamq_at_f32x16 o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] = 0.0f;
    float m = -__builtin_inff(), sum = 0.0f;  // in units of log 2; this lane's keys' part of the sum
    for (int kb = 0; kb < nblk; ++kb) {
        wait_vm<0>();     // this wave's loads of block kb have landed
        __syncthreads();  // everyone's; the other buffer is free
        if (kb + 1 < nblk) load_block(kb + 1);
        const int k0 = kb * AG_W;
        if (k0 > my_last) continue;  // uniform: this wave's queries end before these keys
        uint32_t fb = base + (uint32_t)((kb & 1) * 2 * AG_OPB) + ag_frag_base(li, hi);
        uint32_t tb = base + (uint32_t)((kb & 1) * 2 * AG_OPB) + AG_OPB + ag_tr_base(0, lane);
        asm volatile("" : "+v"(fb), "+v"(tb));  // the fragments' addresses formed here, not kept around the loop
        lamq_at_f32x16 s[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int v = 0; v < 16; ++v) s[hf][v] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                s[hf] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_frag(fb, j, hf * AG_HALF), qf[j], s[hf], 0, 0, 0);
        lamq_at_bf16x8 vf[2][2][4];  // V's fragments read under the softmax
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int mi = 0; mi < 2; ++mi)
#pragma unroll
                for (int t = 0; t < 4; ++t) vf[hf][mi][t] = ag_tr_frag(tb, mi, t, hf * AG_HALF);
        if (k0 + AG_W - 1 > q0) {  // the causal mask, only where the block reaches past the wave's first query
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    s[hf][v] = k0 + 32 * hf + 8 * (v >> 2) + 4 * hi + (v & 3) <= myq ? s[hf][v] : -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int v = 1; v < 32; ++v) mx = fmaxf(mx, s[v >> 4][v & 15]);
        mx = at_max32(mx) * scale_log2;
        if (__builtin_amdgcn_ballot_w64(mx > m + AG_LAZY)) {  // uniform
            const float up = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - up);  // 0 at the first block
            sum *= alpha;
            m = up;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[t][v] *= alpha;
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (hf && k0 + 32 > my_last) break;  // uniform: past this wave's queries
            lamq_at_bf16x8 pf[2], pl[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[hf][v], scale_log2, -m));
                sum += p;
                pf[v >> 3][v & 7] = (__bf16)p;
                if (TWO) pl[v >> 3][v & 7] = at_second(p);
            }
#pragma unroll
            for (int mi = 0; mi < 2; ++mi)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[hf][mi][t], pf[mi], o[t], 0, 0, 0);
                    if (TWO) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[hf][mi][t], pl[mi], o[t], 0, 0, 0);
                }
        }
    }
    if (myq >= T) return;
    sum = at_sum32(sum);
    ag_store_row(Op + (int64_t)myq * O.st, o, 1.0f / sum, hi,
                 rest ? rest + ag_rest(b * Hkv * rep + h, Tall, q0, li) + 4 * hi : nullptr);
    if (hi == 0) L[myq] = (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// dQ, and per query the log-sum-exp in units of log 2 and delta for the other kernel (rows [B, H, T] of stats and
// stats + B H T).
template <bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_dq_kernel(
    AtView Q, AtView K, AtView V, AtView O, AtView dO, AtOut dQ, const uint16_t* __restrict__ rest,
    const float* __restrict__ lse,
    const int32_t* __restrict__ lens, float* __restrict__ stats, int64_t nstats, int rep, int Hkv, int pairs, int Tall,
    float scale, float scale_log2)
{
    __shared__ __align__(256) uint8_t lds[2][2][AG_OPB];  // [buffer][K, V]
    const int nqb = (Tall + AG_OWN - 1) / AG_OWN;
    int pair, rem;
    if (!ag_place(pairs, nqb * rep, pair, rem)) return;
    const int qb = nqb - 1 - rem / rep;  // the longest query blocks first
    const int b = pair / Hkv, hk = pair % Hkv, h = hk * rep + rem % rep;
    const int lane = (int)(threadIdx.x & 63), wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int li = lane & 31, hi = lane >> 5;
    const int T = at_length(lens, b, Tall);
    uint16_t* dQp = dQ.p + b * dQ.sb + (int64_t)h * dQ.sh;
    const int own0 = qb * AG_OWN, own1 = own0 + AG_OWN < Tall ? own0 + AG_OWN : Tall;
    if (own1 > T) {
        at_zero_rows(dQp, dQ.st, own0 > T ? own0 : T, own1);
        if (own0 >= T) return;  // uniform, before any barrier
    }
    const int q0 = own0 + AG_R * wv, myq = q0 + li, qrow = myq < T ? myq : T - 1;
    const uint16_t* Kp = K.p + b * K.sb + (int64_t)hk * K.sh;
    const uint16_t* Vp = V.p + b * V.sb + (int64_t)hk * V.sh;
    const uint32_t base = lds_addr(lds);
    const int wg_last = (own1 < T ? own1 : T) - 1;
    const int nblk = wg_last / AG_W + 1;
    const int my_last = q0 < T ? (q0 + AG_R < T ? q0 + AG_R : T) - 1 : -1;
    auto load_block = [&](int kb) {
        const uint32_t buf = base + (uint32_t)((kb & 1) * 2 * AG_OPB);
        const int r0 = kb * AG_W;
        ag_load_block(Kp + r0 * K.st, K.st, T - r0, wv, lane, buf);
        ag_load_block(Vp + r0 * V.st, V.st, T - r0, wv, lane, buf + AG_OPB);
    };
    load_block(0);
    lamq_at_bf16x8 qf[8], df[8];
    float delta = 0.0f, lse2;
    {
        const uint16_t* Qr = Q.p + b * Q.sb + (int64_t)h * Q.sh + (int64_t)qrow * Q.st + 8 * hi;
        const uint16_t* Dr = dO.p + b * dO.sb + (int64_t)h * dO.sh + (int64_t)qrow * dO.st + 8 * hi;
        const uint16_t* Or = O.p + b * O.sb + (int64_t)h * O.sh + (int64_t)qrow * O.st + 8 * hi;
        const uint16_t* Lr = rest + ag_rest(b * Hkv * rep + h, Tall, q0, li) + 256 * hi;
        const int64_t at = ((int64_t)b * Hkv * rep + h) * Tall + qrow;
        lse2 = lse[at] * AT_LOG2E;
        lamq_at_bf16x8 of[8], lf[8];
        // O's second part has blocks only up to T, and rows only up to the length
        const bool second = rest && myq < T;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            qf[j] = ag_row8(Qr + 16 * j);
            df[j] = ag_row8(Dr + 16 * j);
            of[j] = ag_row8(Or + 16 * j);
            lf[j] = of[j];
        }
        if (second)
#pragma unroll
            for (int j = 0; j < 8; ++j) lf[j] = ag_row8(Lr + 512 * j);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf((float)df[j][e], (float)of[j][e], delta);
        if (second)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) delta = fmaf((float)df[j][e], (float)lf[j][e], delta);
        delta = at_sum32(delta);
        if (hi == 0 && myq < T) {
            stats[at] = lse2;
            stats[nstats + at] = delta;
        }
    }
    ag_settle(qf);
    ag_settle(df);
    lamq_at_f32x16 acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[t][v] = 0.0f;
    for (int kb = 0; kb < nblk; ++kb) {
        wait_vm<0>();     // this wave's loads of block kb have landed
        __syncthreads();  // everyone's; the other buffer is free
        if (kb + 1 < nblk) load_block(kb + 1);
        const int k0 = kb * AG_W;
        uint32_t fb = base + (uint32_t)((kb & 1) * 2 * AG_OPB) + ag_frag_base(li, hi);
        uint32_t tb = base + (uint32_t)((kb & 1) * 2 * AG_OPB) + ag_tr_base(0, lane);
        asm volatile("" : "+v"(fb), "+v"(tb));  // the fragments' addresses formed here, not kept around the loop
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (k0 + 32 * hf > my_last) continue;  // uniform: past this wave's queries
            lamq_at_f32x16 s, dp;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                s[v] = 0.0f;
                dp[v] = -delta;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_frag(fb, j, hf * AG_HALF), qf[j], s, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_frag(fb, j, AG_OPB + hf * AG_HALF), df[j], dp, 0, 0, 0);
            }
            if (k0 + 32 * hf + 31 > q0) {  // the causal mask, only where the half reaches past the wave's first query
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    s[v] = k0 + 32 * hf + 8 * (v >> 2) + 4 * hi + (v & 3) <= myq ? s[v] : -__builtin_inff();
            }
            lamq_at_bf16x8 dsf[2], dsl[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float ds = __builtin_amdgcn_exp2f(fmaf(s[v], scale_log2, -lse2)) * dp[v];
                dsf[v >> 3][v & 7] = (__bf16)ds;
                if (TWO) dsl[v >> 3][v & 7] = at_second(ds);
            }
#pragma unroll
            for (int mi = 0; mi < 2; ++mi)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const lamq_at_bf16x8 kt = ag_tr_frag(tb, mi, t, hf * AG_HALF);
                    acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, dsf[mi], acc[t], 0, 0, 0);
                    if (TWO) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, dsl[mi], acc[t], 0, 0, 0);
                }
        }
    }
    if (myq < T) ag_store_row(dQp + (int64_t)myq * dQ.st, acc, scale, hi);
}

// dK and dV of 64 keys of a key/value head, over its query heads and the queries from the keys on. Two waves own 32 keys
// each, two more the same keys: of a walked block of 64 queries the first pair takes the first 32, the second the
// others, and their sums are joined in LDS at the end. A wave's walk is as long as the heads and the queries are many,
// so with 128 keys a workgroup four sequences of 2,048 had 512 workgroups, one for every slot of the chip, the first
// keys' with twice the mean walk: 606 us; halved walks of half the keys go out longest first and fill each other's
// tails. The queries are walked from the last one down, so that workgroups that start together read the same blocks.
template <bool TWO>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_dkdv_kernel(
    AtView Q, AtView K, AtView V, AtView dO, AtOut dK, AtOut dV, const int32_t* __restrict__ lens,
    const float* __restrict__ stats, int64_t nstats, int rep, int Hkv, int pairs, int Tall, float scale, float scale_log2)
{
    __shared__ __align__(256) uint8_t lds[2][2][AG_OPB];  // [buffer][Q, dO]; at the end [wave][64 registers][64 lanes]
    __shared__ __align__(16) float row_stats[2][2][AG_W];  // [buffer][lse, delta]
    const int nkb = (Tall + AG_KEYS - 1) / AG_KEYS;
    // workgroup -> (key block, pair): the first keys, whose walks are the longest, go out first
    const int id = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if ((unsigned)id >= (unsigned)pairs * (unsigned)nkb) return;
    const int pair = id % pairs, kb = id / pairs;
    const int b = pair / Hkv, hk = pair % Hkv;
    const int lane = (int)(threadIdx.x & 63), wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int li = lane & 31, hi = lane >> 5, kw = wv >> 1, qw = wv & 1;
    const int T = at_length(lens, b, Tall);
    uint16_t* dKp = dK.p + b * dK.sb + (int64_t)hk * dK.sh;
    uint16_t* dVp = dV.p + b * dV.sb + (int64_t)hk * dV.sh;
    const int own0 = kb * AG_KEYS, own1 = own0 + AG_KEYS < Tall ? own0 + AG_KEYS : Tall;
    if (own1 > T) {
        const int first = own0 > T ? own0 : T;
        at_zero_rows(dKp, dK.st, first, own1);
        at_zero_rows(dVp, dV.st, first, own1);
        if (own0 >= T) return;  // uniform, before any barrier
    }
    const int k0 = own0 + AG_R * kw, myk = k0 + li, krow = myk < T ? myk : T - 1;
    const uint32_t base = lds_addr(lds), sbase = lds_addr(row_stats);
    const int b0 = own0 / AG_W, b1 = (T - 1) / AG_W;  // the walked blocks, from b1 down to b0
    auto load_block = [&](int h, int blk, int to) {
        const int r0 = blk * AG_W;
        const uint32_t buf = base + (uint32_t)(to * 2 * AG_OPB);
        ag_load_block(Q.p + b * Q.sb + (int64_t)h * Q.sh + r0 * Q.st, Q.st, T - r0, wv, lane, buf);
        ag_load_block(dO.p + b * dO.sb + (int64_t)h * dO.sh + r0 * dO.st, dO.st, T - r0, wv, lane, buf + AG_OPB);
        if (wv < 2) {
            const int row = r0 + lane < T ? r0 + lane : T - 1;
            load_lds4(stats + wv * nstats + ((int64_t)b * Hkv * rep + h) * Tall + row,
                      sbase + (uint32_t)((to * 2 + wv) * AG_W * 4));
        }
    };
    const int h1 = hk * rep + rep;
    int h = hk * rep, blk = b1;
    load_block(h, blk, 0);
    lamq_at_bf16x8 kf[8], vf[8];
    {
        const uint16_t* Kr = K.p + b * K.sb + (int64_t)hk * K.sh + (int64_t)krow * K.st + 8 * hi;
        const uint16_t* Vr = V.p + b * V.sb + (int64_t)hk * V.sh + (int64_t)krow * V.st + 8 * hi;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            kf[j] = ag_row8(Kr + 16 * j);
            vf[j] = ag_row8(Vr + 16 * j);
        }
    }
    ag_settle(kf);
    ag_settle(vf);
    lamq_at_f32x16 dk[4], dv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) dk[t][v] = dv[t][v] = 0.0f;
    for (int cur = 0; h < h1; cur ^= 1) {
        wait_vm<0>();     // this wave's loads of the block have landed
        __syncthreads();  // everyone's; the other buffer is free
        const int q0 = blk * AG_W + 32 * qw;  // this wave's queries of the block
        if (--blk < b0) {
            blk = b1;
            ++h;
        }
        if (h < h1) load_block(h, blk, cur ^ 1);
        if (q0 + 31 < k0 || q0 >= T) continue;  // uniform: no query here sees this wave's keys
        uint32_t fb = base + (uint32_t)(cur * 2 * AG_OPB) + ag_frag_base(32 * qw + li, hi);
        uint32_t tb = base + (uint32_t)(cur * 2 * AG_OPB) + ag_tr_base(qw, lane);
        asm volatile("" : "+v"(fb), "+v"(tb));  // the fragments' addresses formed here, not kept around the loop
        const float* sl = &row_stats[cur][0][32 * qw + 4 * hi];
        lamq_at_f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float4 dl4 = *reinterpret_cast<const float4*>(sl + AG_W + 8 * r);
            dp[4 * r] = -dl4.x;
            dp[4 * r + 1] = -dl4.y;
            dp[4 * r + 2] = -dl4.z;
            dp[4 * r + 3] = -dl4.w;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_frag(fb, j, 0), kf[j], s, 0, 0, 0);
            dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_frag(fb, j, AG_OPB), vf[j], dp, 0, 0, 0);
        }
        if (q0 < k0 + 31 || q0 + 31 >= T) {  // the causal mask and the queries past the length
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int q = q0 + 8 * (v >> 2) + 4 * hi + (v & 3);
                s[v] = myk <= q && q < T ? s[v] : -__builtin_inff();
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float4 ls4 = *reinterpret_cast<const float4*>(sl + 8 * r);
            const float ls[4] = {ls4.x, ls4.y, ls4.z, ls4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = 4 * r + e;
                s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], scale_log2, -ls[e]));
                dp[v] *= s[v];
            }
        }
#pragma unroll
        for (int part = 0; part < (TWO ? 2 : 1); ++part) {
            if (part) asm volatile("" : "+v"(tb));  // the transposed tiles are read again: no registers are left to keep them
            lamq_at_bf16x8 pf[2], dsf[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                pf[v >> 3][v & 7] = part ? at_second(s[v]) : (__bf16)s[v];
                dsf[v >> 3][v & 7] = part ? at_second(dp[v]) : (__bf16)dp[v];
            }
#pragma unroll
            for (int mi = 0; mi < 2; ++mi)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    dv[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_tr_frag(tb, mi, t, AG_OPB), pf[mi], dv[t], 0, 0, 0);
                    dk[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ag_tr_frag(tb, mi, t, 0), dsf[mi], dk[t], 0, 0, 0);
                }
        }
    }
    // the two halves of the queries: the first pair of waves takes the other's dK and ends with it, the second dV
    __syncthreads();  // everyone's last block is done with
    float* mine = reinterpret_cast<float*>(lds) + wv * 64 * 64 + lane;
    const float* other = reinterpret_cast<float*>(lds) + (wv ^ 1) * 64 * 64 + lane;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) mine[64 * (16 * t + v)] = qw ? dk[t][v] : dv[t][v];
    __syncthreads();
    if (qw) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) dv[t][v] = other[64 * (16 * t + v)] + dv[t][v];
        if (myk < T) ag_store_row(dVp + (int64_t)myk * dV.st, dv, 1.0f, hi);
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) dk[t][v] += other[64 * (16 * t + v)];
        if (myk < T) ag_store_row(dKp + (int64_t)myk * dK.st, dk, scale, hi);
    }
}

// A tensor by its strides: 16-byte loads of inputs, 8-byte stores of outputs, 64 rows within a 32-bit byte offset
static int at_heads(const lamq_heads* x, int64_t T, int align)
{
    if (!x || !x->data || (uintptr_t)x->data % align) return LAMQ_EINVAL;
    for (int64_t s : {x->sb, x->sh, x->st})
        if (s < 0 || s % 8 != 0) return LAMQ_EINVAL;
    return T > 1 && x->st > 0xffffff ? LAMQ_EUNSUP : LAMQ_OK;
}

static int at_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t D, float scale)
{
    if (B < 0 || H < 1 || Hkv < 1 || T < 0 || H % Hkv != 0) return LAMQ_EINVAL;
    if (D != AT_D) return LAMQ_EUNSUP;
    if (!(scale > 0.0f) || !(scale < 3.0e38f)) return LAMQ_EINVAL;
    if (B > 65535 || H > 65535 || T > 0x7fffff) return LAMQ_EUNSUP;
    return cdiv(T, AG_KEYS) * H * B > 0x7fffffff ? LAMQ_EUNSUP : LAMQ_OK;
}

// a grid's work items along x must stay below 2^32, so past 2^22 workgroups they go out in rows
static dim3 at_grid(int64_t wgs)
{
    const int64_t gx = wgs < AT_GRID_X ? wgs : AT_GRID_X;
    return dim3((unsigned)gx, (unsigned)cdiv(wgs, gx));
}

// P and dS in two parts where one block of queries is all there is. 45 tokens x 32 heads: 28 -> 36 us on the device, 37 us a
// call from the host either way, and the error over that of the results' own rounding 1.46 -> 1.00 (2 to 5 tokens: up to
// 1.97 -> 1.00); 4 x 32 heads x 2,048: 695 -> 1,102 us, 1.43 -> 1.00
static bool at_two(int64_t T) { return T <= AG_OWN; }

static AtView at_view(const lamq_heads* x) { return AtView{x->data, x->sb, x->sh, x->st}; }
static AtOut at_out(const lamq_heads* x) { return AtOut{x->data, x->sb, x->sh, x->st}; }

extern "C" int lamq_attention_causal_lse_bf16(const lamq_heads* q, const lamq_heads* k, const lamq_heads* v,
                                              const lamq_heads* out, uint16_t* rest, float* lse, const int32_t* lens,
                                              int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t D, float scale,
                                              void* stream)
{
    int rc = at_sizes(B, H, Hkv, T, D, scale);
    for (const lamq_heads* x : {q, k, v})
        if (rc == LAMQ_OK) rc = at_heads(x, T, 16);
    if (rc == LAMQ_OK) rc = at_heads(out, T, 8);
    if (rc != LAMQ_OK) return rc;
    if (!lse || (uintptr_t)rest % 16) return LAMQ_EINVAL;
    if (B == 0 || T == 0) return LAMQ_OK;
    hipLaunchKernelGGL((at_two(T) ? attention_lse_kernel<true> : attention_lse_kernel<false>), at_grid(cdiv(T, AG_OWN) * H * B), dim3(256), 0, as_stream(stream), at_view(q),
                       at_view(k), at_view(v), at_out(out), rest, lse, lens, (int)(H / Hkv), (int)Hkv, (int)(B * Hkv), (int)T,
                       scale * AT_LOG2E);
    LAMQ_LAUNCH_CHECK();
    return LAMQ_OK;
}

extern "C" size_t lamq_attention_causal_grad_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t T)
{
    if (B < 1 || H < 1 || Hkv < 1 || T < 1) return 0;
    return (size_t)B * H * T * 2 * sizeof(float);
}

extern "C" int lamq_attention_causal_grad_bf16(const lamq_heads* q, const lamq_heads* k, const lamq_heads* v,
                                               const lamq_heads* out, const uint16_t* rest, const float* lse,
                                               const lamq_heads* dout,
                                               const int32_t* lens, const lamq_heads* dq, const lamq_heads* dk,
                                               const lamq_heads* dv, int64_t B, int64_t H, int64_t Hkv, int64_t T,
                                               int64_t D, float scale, void* workspace, size_t workspace_bytes,
                                               void* stream)
{
    int rc = at_sizes(B, H, Hkv, T, D, scale);
    for (const lamq_heads* x : {q, k, v, out, dout})
        if (rc == LAMQ_OK) rc = at_heads(x, T, 16);
    for (const lamq_heads* x : {dq, dk, dv})
        if (rc == LAMQ_OK) rc = at_heads(x, T, 8);
    if (rc != LAMQ_OK) return rc;
    if (!lse || (uintptr_t)rest % 16) return LAMQ_EINVAL;
    if (B == 0 || T == 0) return LAMQ_OK;
    if (!workspace || (uintptr_t)workspace % 4 ||
        workspace_bytes < lamq_attention_causal_grad_workspace_size(B, H, Hkv, T))
        return LAMQ_EINVAL;
    float* stats = reinterpret_cast<float*>(workspace);
    const int64_t nstats = B * H * T;
    hipStream_t s = as_stream(stream);
    const bool two = at_two(T);
    hipLaunchKernelGGL((two ? attention_dq_kernel<true> : attention_dq_kernel<false>), at_grid(cdiv(T, AG_OWN) * H * B), dim3(256), 0, s, at_view(q), at_view(k),
                       at_view(v), at_view(out), at_view(dout), at_out(dq), rest, lse, lens, stats, nstats, (int)(H / Hkv),
                       (int)Hkv, (int)(B * Hkv), (int)T, scale, scale * AT_LOG2E);
    LAMQ_LAUNCH_CHECK();
    hipLaunchKernelGGL((two ? attention_dkdv_kernel<true> : attention_dkdv_kernel<false>), at_grid(cdiv(T, AG_KEYS) * Hkv * B), dim3(256), 0, s, at_view(q), at_view(k),
                       at_view(v), at_view(dout), at_out(dk), at_out(dv), lens, stats, nstats, (int)(H / Hkv), (int)Hkv,
                       (int)(B * Hkv), (int)T, scale, scale * AT_LOG2E);
    LAMQ_LAUNCH_CHECK();
    return LAMQ_OK;
}
