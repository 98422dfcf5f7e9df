// The KL loss of distillation with its gradient (the loss finetune.py's distillation descends; compiler.py:177-188
// measures the same KL): for rows t of reference logits r and student logits q with weights w,
//   kl_t = sum_v p_v (log p_v - log s_v),  p = softmax(r_t), s = softmax(q_t),
//   loss = sum_t w_t kl_t / sum_t w_t,     dq_t = w_t / sum(w) (s - p).
// A row of weight 0 is left out: its kl and gradient are 0 and its logits are not read.
//
// kl_t = (sum_v e^(r_v - m_r) (r_v - q_v)) / s_r - lse_r + lse_q needs the row's maxima and three sums; the gradient
// needs both sums, so a row is read for them and again for the gradient. What bounds it is memory: three elements a
// logit cannot be done without. The sums of 8 logits are float32, the running ones float64 (they cancel in kl where
// the two distributions are close), merged in a fixed order.
//
// A logit of -inf (a masked word) has weight 0 in its distribution: where r is -inf the term is 0, where only q is, kl
// is +inf. A row with no finite logit has no distribution, and its kl and gradient are NaN.
#include "common.h"

#define KG_NT 256      // threads of a workgroup
#define KG_SPLIT 256   // rows from which on a workgroup takes a row of its own

__device__ __forceinline__ float kg_inf() { return __builtin_inff(); }

// Eight logits at any alignment of their type (rows of an odd length start anywhere; the hardware takes 16-byte
// accesses at element alignment), as they are and as float32.
typedef uint32_t kg_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float kg_f4 __attribute__((ext_vector_type(4), aligned(4)));
struct KGChunk {
    float v[8];
};
template <typename Elt>
struct KGRaw;
template <>
struct KGRaw<uint16_t> {
    uint4 x[1];
};
template <>
struct KGRaw<float> {
    uint4 x[2];
};
__device__ __forceinline__ KGRaw<uint16_t> kg_raw(const uint16_t* p)
{
    const kg_u4 x = *reinterpret_cast<const kg_u4*>(p);
    return KGRaw<uint16_t>{{make_uint4(x[0], x[1], x[2], x[3])}};
}
__device__ __forceinline__ KGRaw<float> kg_raw(const float* p)
{
    const kg_f4 x = reinterpret_cast<const kg_f4*>(p)[0], y = reinterpret_cast<const kg_f4*>(p)[1];
    auto u = [](kg_f4 a) {
        return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
    };
    return KGRaw<float>{{u(x), u(y)}};
}
__device__ __forceinline__ KGChunk kg_wide(const KGRaw<uint16_t>& r)
{
    const uint32_t x[4] = {r.x[0].x, r.x[0].y, r.x[0].z, r.x[0].w};
    KGChunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c.v[2 * i] = __uint_as_float(x[i] << 16);
        c.v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
    }
    return c;
}
__device__ __forceinline__ KGChunk kg_wide(const KGRaw<float>& r)
{
    KGChunk c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        c.v[4 * h] = __uint_as_float(r.x[h].x);
        c.v[4 * h + 1] = __uint_as_float(r.x[h].y);
        c.v[4 * h + 2] = __uint_as_float(r.x[h].z);
        c.v[4 * h + 3] = __uint_as_float(r.x[h].w);
    }
    return c;
}
template <typename Elt>
__device__ __forceinline__ KGChunk kg_load8(const Elt* p)
{
    return kg_wide(kg_raw(p));
}
__device__ __forceinline__ float kg_load1(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ float kg_load1(const float* p) { return *p; }

// float32 to bf16, nearest with ties to even
__device__ __forceinline__ uint16_t kg_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ void kg_store8(uint16_t* p, const KGChunk& c)
{
    kg_u4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (uint32_t)kg_bf16(c.v[2 * i]) | ((uint32_t)kg_bf16(c.v[2 * i + 1]) << 16);
    *reinterpret_cast<kg_u4*>(p) = x;
}
__device__ __forceinline__ void kg_store8(float* p, const KGChunk& c)
{
#pragma unroll
    for (int h = 0; h < 2; ++h)
        reinterpret_cast<kg_f4*>(p)[h] = kg_f4{c.v[4 * h], c.v[4 * h + 1], c.v[4 * h + 2], c.v[4 * h + 3]};
}
__device__ __forceinline__ void kg_store1(uint16_t* p, float x) { *p = kg_bf16(x); }
__device__ __forceinline__ void kg_store1(float* p, float x) { *p = x; }

// A part of a row: both maxima in units of log 2 (log2(e) times the largest logit, rounded: the sums' common reference
// and nothing else), s_r and s_q relative to them, and a = sum e^(r - m_r) (r - q)
struct KGPart {
    float mr, mq;
    double sr, ar, sq;
};
#define KG_L2E 1.4426950408889634f
#define KG_FAR 1e30f  // logits beyond it (-inf, the types' lowest and largest values) are taken by the careful form

__device__ __forceinline__ float kg_exp(float x, float m) { return __builtin_amdgcn_exp2f(fmaf(x, KG_L2E, -m)); }
// The same where x or m may be infinite or too large to multiply: differences first, -inf gives 0 (also against -inf).
__device__ __forceinline__ float kg_exp_far(float x, float m)
{
    return x == -kg_inf() ? 0.0f : __builtin_amdgcn_exp2f((x - m * (1.0f / KG_L2E)) * KG_L2E);
}
// log2(e) x for a maximum, kept finite
__device__ __forceinline__ float kg_log2(float x)
{
    return x == -kg_inf() ? x : fminf(fmaxf(x * KG_L2E, -3.0e38f), 3.0e38f);
}
// a times a factor that may have underflowed, +inf where a is: it stays so
__device__ __forceinline__ double kg_keep_inf(double a, double f) { return a == (double)kg_inf() ? a : a * f; }

// the first N of eight logits into a part
template <int N>
__device__ __forceinline__ void kg_add(KGPart& p, const KGChunk& r, const KGChunk& q)
{
    float cr = r.v[0], cq = q.v[0], lo = fminf(r.v[0], q.v[0]);
#pragma unroll
    for (int e = 1; e < N; ++e) {
        cr = fmaxf(cr, r.v[e]);
        cq = fmaxf(cq, q.v[e]);
        lo = fminf(lo, fminf(r.v[e], q.v[e]));
    }
    const bool far = lo < -KG_FAR || cr > KG_FAR || cq > KG_FAR;
    const float br = kg_log2(cr), bq = kg_log2(cq);
    if (br > p.mr) {
        const double f = p.mr == -kg_inf() ? 0.0 : (double)__builtin_amdgcn_exp2f(p.mr - br);
        p.sr *= f;
        p.ar = kg_keep_inf(p.ar, f);
        p.mr = br;
    }
    if (bq > p.mq) {
        p.sq *= p.mq == -kg_inf() ? 0.0 : (double)__builtin_amdgcn_exp2f(p.mq - bq);
        p.mq = bq;
    }
    float sr = 0.0f, ar = 0.0f, sq = 0.0f;
    if (far) {  // masked words, by -inf or the type's lowest value: the terms that would be 0 times infinity
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float er = kg_exp_far(r.v[e], p.mr);
            sr += er;
            if (r.v[e] != -kg_inf() && q.v[e] == -kg_inf())
                ar = kg_inf();
            else if (!(er == 0.0f))
                ar += er * (r.v[e] - q.v[e]);
            sq += kg_exp_far(q.v[e], p.mq);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float er = kg_exp(r.v[e], p.mr);
            sr += er;
            ar = fmaf(er, r.v[e] - q.v[e], ar);
            sq += kg_exp(q.v[e], p.mq);
        }
    }
    p.sr += (double)sr;
    p.ar += (double)ar;
    p.sq += (double)sq;
}

// x times 2^(m - M), for a part's sum and maximum against a larger maximum
__device__ __forceinline__ double kg_scaled(double x, float m, float M)
{
    return m == -kg_inf() ? 0.0 : m == M ? x : kg_keep_inf(x, exp2((double)m - (double)M));
}

// The sum of the workgroup's parts, in every thread: the maxima, then the sums by waves and over them, in a fixed order.
template <int NT = KG_NT>
__device__ __forceinline__ KGPart kg_reduce(KGPart p)
{
    __shared__ float m[2][NT / 64];
    __shared__ double s[3][NT / 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float mr = p.mr, mq = p.mq;
    for (int o = 32; o; o >>= 1) {
        mr = fmaxf(mr, __shfl_xor(mr, o));
        mq = fmaxf(mq, __shfl_xor(mq, o));
    }
    if (lane == 0) {
        m[0][wave] = mr;
        m[1][wave] = mq;
    }
    __syncthreads();
    KGPart t;
    t.mr = m[0][0];
    t.mq = m[1][0];
    for (int w = 1; w < NT / 64; ++w) {
        t.mr = fmaxf(t.mr, m[0][w]);
        t.mq = fmaxf(t.mq, m[1][w]);
    }
    double x[3] = {kg_scaled(p.sr, p.mr, t.mr), kg_scaled(p.ar, p.mr, t.mr), kg_scaled(p.sq, p.mq, t.mq)};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        for (int o = 32; o; o >>= 1) x[i] += __shfl_xor(x[i], o);
        if (lane == 0) s[i][wave] = x[i];
    }
    __syncthreads();
    t.sr = t.ar = t.sq = 0.0;
    for (int w = 0; w < NT / 64; ++w) {
        t.sr += s[0][w];
        t.ar += s[1][w];
        t.sq += s[2][w];
    }
    __syncthreads();  // the arrays are free again
    return t;
}

__device__ __forceinline__ double kg_kl(const KGPart& t)
{
    // mean of r - q under p, minus the log-sum-exps, whose references are in log 2
    return t.ar / t.sr + 0.6931471805599453 * ((double)t.mq - (double)t.mr) + (log(t.sq) - log(t.sr));
}

// this thread's share of logits v0 .. v1 - 1 of a row
template <typename Elt>
__device__ __forceinline__ KGPart kg_part(const Elt* r, const Elt* q, int64_t v0, int64_t v1)
{
    KGPart p{-kg_inf(), -kg_inf(), 0.0, 0.0, 0.0};
    int64_t v = v0 + 8 * (int64_t)threadIdx.x;
    for (; v + 8 <= v1; v += 8 * KG_NT) kg_add<8>(p, kg_load8(r + v), kg_load8(q + v));
    for (; v < v1; ++v) {  // the last ones, in the one thread they fall to
        KGChunk a, b;
        a.v[0] = kg_load1(r + v);
        b.v[0] = kg_load1(q + v);
        kg_add<1>(p, a, b);
    }
    return p;
}

// The gradient fq e^(q - m_q) - fr e^(r - m_r), fq = coef / s_q and fr = coef / s_r, of a chunk of logits
struct KGCoef {
    float fr, fq, mr, mq;
    bool far;  // a maximum no product of the fast form reaches
};
__device__ __forceinline__ KGCoef kg_coef(const KGPart& t, double coef)
{
    return KGCoef{(float)(coef / t.sr), (float)(coef / t.sq), t.mr, t.mq, !(fabsf(t.mr) < KG_FAR && fabsf(t.mq) < KG_FAR)};
}
__device__ __forceinline__ float kg_grad1(float r, float q, const KGCoef& k)
{
    if (k.far) return fmaf(kg_exp_far(q, k.mq), k.fq, -(kg_exp_far(r, k.mr) * k.fr));  // uniform
    // a logit of -inf or far below a maximum of ordinary size: the multiply-add gives -inf, its exponential 0
    return fmaf(kg_exp(q, k.mq), k.fq, -(kg_exp(r, k.mr) * k.fr));
}
__device__ __forceinline__ KGChunk kg_grad8(const KGChunk& a, const KGChunk& b, const KGCoef& k)
{
    KGChunk c;
#pragma unroll
    for (int e = 0; e < 8; ++e) c.v[e] = kg_grad1(a.v[e], b.v[e], k);
    return c;
}
template <typename Elt>
__device__ __forceinline__ void kg_grad(const Elt* r, const Elt* q, Elt* g, int64_t v0, int64_t v1, const KGCoef& k)
{
    int64_t v = v0 + 8 * (int64_t)threadIdx.x;
    for (; v + 8 <= v1; v += 8 * KG_NT) kg_store8(g + v, kg_grad8(kg_load8(r + v), kg_load8(q + v), k));
    for (; v < v1; ++v) kg_store1(g + v, kg_grad1(kg_load1(r + v), kg_load1(q + v), k));
}

template <int NT, typename Elt>
__device__ __forceinline__ void kg_zero(Elt* g, int64_t v0, int64_t v1)
{
    KGChunk z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z.v[e] = 0.0f;
    int64_t v = v0 + 8 * (int64_t)threadIdx.x;
    for (; v + 8 <= v1; v += 8 * NT) kg_store8(g + v, z);
    for (; v < v1; ++v) kg_store1(g + v, 0.0f);
}

// the workgroup's sum of x, in every thread, in a fixed order
template <int NT>
__device__ __forceinline__ double kg_sum(double x)
{
    __shared__ double s[NT / 64];
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < NT / 64; ++w) t += s[w];
    __syncthreads();
    return t;
}

// sum w (T without weights) over all T, in every thread
template <int NT>
__device__ __forceinline__ double kg_weights(const float* __restrict__ w, int64_t T)
{
    if (!w) return (double)T;
    double x = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += NT) x += (double)w[t];
    return kg_sum<NT>(x);
}

__global__ __launch_bounds__(1024) void kl_weights_kernel(const float* __restrict__ w, int64_t T, double* __restrict__ total)
{
    const double x = kg_weights<1024>(w, T);
    if (threadIdx.x == 0) *total = x;
}

// loss = sum w kl / sum w, of float64 kl's
__global__ __launch_bounds__(1024) void kl_loss_kernel(const double* __restrict__ kl, const float* __restrict__ w, int64_t T,
                                                       float* __restrict__ loss)
{
    double x = 0.0, y = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        const double wt = w ? (double)w[t] : 1.0;
        x += wt * kl[t];
        y += wt;
    }
    x = kg_sum<1024>(x);
    y = kg_sum<1024>(y);
    if (threadIdx.x == 0) *loss = (float)(x / y);
}

// Many rows: a workgroup of NT threads a row, read once: of a thread's chunks the first REGS stay in its registers and the
// next LDS in its places of the unit's LDS until the gradient is formed; what a longer row has beyond them is read
// again, from the caches as far as the rows in flight (one a unit: 155 MB at 151,936 bf16 words) fit there.
template <typename Elt, int NT, int REGS, int LDS>
__global__ __launch_bounds__(NT) void kl_grad_rows_kernel(const Elt* __restrict__ ref, const Elt* __restrict__ q, int64_t V,
                                                          int64_t ldr, int64_t ldq, const float* __restrict__ w,
                                                          const double* __restrict__ total, float* __restrict__ kl,
                                                          double* __restrict__ kl64, Elt* __restrict__ grad, int64_t ldg)
{
    constexpr int N16 = sizeof(KGRaw<Elt>) / 16;
    __shared__ uint4 held[LDS * 2 * N16 * NT + 1];
    const int64_t t = blockIdx.x;
    const double wt = w ? (double)w[t] : 1.0;
    Elt* g = grad + t * ldg;
    if (wt == 0.0) {
        kg_zero<NT>(g, 0, V);
        if (threadIdx.x == 0) {
            kl[t] = 0.0f;
            kl64[t] = 0.0;
        }
        return;
    }
    const Elt *r = ref + t * ldr, *s = q + t * ldq;
    const int64_t nv = V / 8;  // whole chunks; this thread's: threadIdx.x + NT c
    KGPart p{-kg_inf(), -kg_inf(), 0.0, 0.0, 0.0};
    KGRaw<Elt> a[REGS], b[REGS];
#pragma unroll
    for (int c = 0; c < REGS; ++c) {
        const int64_t i = threadIdx.x + (int64_t)NT * c;
        if (i < nv) {
            a[c] = kg_raw(r + 8 * i);
            b[c] = kg_raw(s + 8 * i);
        }
    }
    auto place = [&](int c, int half, int k) -> uint4& { return held[((c * 2 + half) * N16 + k) * NT + threadIdx.x]; };
    if constexpr (LDS > 0) {
        KGRaw<Elt> x[LDS], y[LDS];
#pragma unroll
        for (int c = 0; c < LDS; ++c) {
            const int64_t i = threadIdx.x + (int64_t)NT * (REGS + c);
            if (i < nv) {
                x[c] = kg_raw(r + 8 * i);
                y[c] = kg_raw(s + 8 * i);
            }
        }
#pragma unroll
        for (int c = 0; c < REGS; ++c)
            if (threadIdx.x + (int64_t)NT * c < nv) kg_add<8>(p, kg_wide(a[c]), kg_wide(b[c]));
#pragma unroll
        for (int c = 0; c < LDS; ++c)
            if (threadIdx.x + (int64_t)NT * (REGS + c) < nv) {
                kg_add<8>(p, kg_wide(x[c]), kg_wide(y[c]));
#pragma unroll
                for (int k = 0; k < N16; ++k) {
                    place(c, 0, k) = x[c].x[k];
                    place(c, 1, k) = y[c].x[k];
                }
            }
    } else {
#pragma unroll
        for (int c = 0; c < REGS; ++c)
            if (threadIdx.x + (int64_t)NT * c < nv) kg_add<8>(p, kg_wide(a[c]), kg_wide(b[c]));
    }
    constexpr int64_t kept = (int64_t)NT * (REGS + LDS);
#pragma unroll 2
    for (int64_t i = threadIdx.x + kept; i < nv; i += NT) kg_add<8>(p, kg_load8(r + 8 * i), kg_load8(s + 8 * i));
    const int64_t tail = 8 * nv + threadIdx.x;  // up to seven logits past the whole chunks, one a thread
    if (tail < V) {
        KGChunk x, y;
        x.v[0] = kg_load1(r + tail);
        y.v[0] = kg_load1(s + tail);
        kg_add<1>(p, x, y);
    }
    p = kg_reduce<NT>(p);
    const KGCoef k = kg_coef(p, wt / *total);
#pragma unroll
    for (int c = 0; c < REGS; ++c) {
        const int64_t i = threadIdx.x + (int64_t)NT * c;
        if (i < nv) kg_store8(g + 8 * i, kg_grad8(kg_wide(a[c]), kg_wide(b[c]), k));
    }
#pragma unroll
    for (int c = 0; c < LDS; ++c) {
        const int64_t i = threadIdx.x + (int64_t)NT * (REGS + c);
        if (i < nv) {
            KGRaw<Elt> x, y;
#pragma unroll
            for (int e = 0; e < N16; ++e) {
                x.x[e] = place(c, 0, e);
                y.x[e] = place(c, 1, e);
            }
            kg_store8(g + 8 * i, kg_grad8(kg_wide(x), kg_wide(y), k));
        }
    }
#pragma unroll 2
    for (int64_t i = threadIdx.x + kept; i < nv; i += NT)
        kg_store8(g + 8 * i, kg_grad8(kg_load8(r + 8 * i), kg_load8(s + 8 * i), k));
    if (tail < V) kg_store1(g + tail, kg_grad1(kg_load1(r + tail), kg_load1(s + tail), k));
    if (threadIdx.x == 0) {
        const double x = kg_kl(p);
        kl[t] = (float)x;
        kl64[t] = x;
    }
}

// Few rows: `split` workgroups a row. The first launch leaves each one's part ...
template <typename Elt>
__global__ __launch_bounds__(KG_NT) void kl_part_kernel(const Elt* __restrict__ ref, const Elt* __restrict__ q, int64_t V,
                                                        int64_t ldr, int64_t ldq, const float* __restrict__ w,
                                                        int64_t span, int split, KGPart* __restrict__ parts)
{
    const int64_t t = blockIdx.x / split, s = blockIdx.x % split;
    if (w && w[t] == 0.0f) return;
    const int64_t v0 = s * span, v1 = v0 + span < V ? v0 + span : V;
    const KGPart p = kg_reduce(kg_part(ref + t * ldr, q + t * ldq, v0, v1));
    if (threadIdx.x == 0) parts[blockIdx.x] = p;
}

// ... and the second joins a row's parts (each thread takes one; split <= KG_NT) and writes its span of the gradient.
template <typename Elt>
__global__ __launch_bounds__(KG_NT) void kl_grad_part_kernel(const Elt* __restrict__ ref, const Elt* __restrict__ q,
                                                             int64_t T, int64_t V, int64_t ldr, int64_t ldq,
                                                             const float* __restrict__ w, int64_t span, int split,
                                                             const KGPart* __restrict__ parts, float* __restrict__ kl,
                                                             double* __restrict__ kl64, Elt* __restrict__ grad, int64_t ldg)
{
    const int64_t t = blockIdx.x / split, s = blockIdx.x % split;
    const int64_t v0 = s * span, v1 = v0 + span < V ? v0 + span : V;
    const double wt = w ? (double)w[t] : 1.0;
    double x = 0.0;
    if (wt == 0.0) {
        kg_zero<KG_NT>(grad + t * ldg, v0, v1);
    } else {
        KGPart p{-kg_inf(), -kg_inf(), 0.0, 0.0, 0.0};
        if ((int)threadIdx.x < split) p = parts[t * split + threadIdx.x];
        p = kg_reduce(p);
        kg_grad(ref + t * ldr, q + t * ldq, grad + t * ldg, v0, v1, kg_coef(p, wt / kg_weights<KG_NT>(w, T)));
        x = kg_kl(p);
    }
    if (s == 0 && threadIdx.x == 0) {
        kl[t] = (float)x;
        kl64[t] = x;
    }
}

// workgroups a row for T rows of V logits: enough to fill the chip with a few, at least 2,048 logits each; one where there
// is a row for every unit (151,936 bf16 words, several workgroups a row / one: 64 rows 30 / 53 us, 128 45 / 55, 255 73 / 68)
static int kg_splits(int64_t T, int64_t V)
{
    if (T >= KG_SPLIT) return 1;
    const int64_t want = cdiv(1024, T), most = cdiv(V, 2048);
    const int64_t s = want < most ? want : most;
    return (int)(s < KG_NT ? s : KG_NT);
}

extern "C" size_t lamq_kl_rows_grad_workspace_size(int64_t T, int64_t V)
{
    if (T < 1 || V < 1) return 0;
    return 16 + (size_t)T * sizeof(double) + (size_t)T * kg_splits(T, V) * sizeof(KGPart);
}

template <typename Elt>
static int kl_grad_launch(const Elt* ref, const Elt* q, int64_t T, int64_t V, int64_t ldr, int64_t ldq, const float* w,
                          float* kl, float* loss, Elt* grad, int64_t ldg, void* workspace, size_t workspace_bytes,
                          void* stream)
{
    if (!ref || !q || !kl || !loss || !grad || T < 0 || V < 1 || ldr < V || ldq < V || ldg < V) return LAMQ_EINVAL;
    if ((uintptr_t)ref % sizeof(Elt) || (uintptr_t)q % sizeof(Elt) || (uintptr_t)grad % sizeof(Elt)) return LAMQ_EINVAL;
    if (T == 0) return LAMQ_OK;
    if (T > 0xffffff) return LAMQ_EUNSUP;  // the grid's work items stay below 2^32
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < lamq_kl_rows_grad_workspace_size(T, V))
        return LAMQ_EINVAL;
    hipStream_t st = as_stream(stream);
    double* total = reinterpret_cast<double*>(workspace);
    double* kl64 = total + 2;
    KGPart* parts = reinterpret_cast<KGPart*>(kl64 + T);
    const int split = kg_splits(T, V);
    if (split == 1) {
        hipLaunchKernelGGL(kl_weights_kernel, dim3(1), dim3(1024), 0, st, w, T, total);
        LAMQ_LAUNCH_CHECK();
        // Rows up to 96 KB: 256 threads, four rows a unit in flight to cover each other's sums, what their registers do not
        // hold read again from the caches. Longer ones, which pass the caches so: 1,024 threads and most of a unit's LDS.
        // 2,048 rows bf16, 256 / 1,024 threads: of 32,000 words 103 / 134 us, 49,152 179 / 181, 65,536 245 / 234, 151,936
        // 614 / 499 (on a slower box); 1,024 rows float32: 16,384 words 50 / 57, 65,536 257 / 208
        constexpr int R = sizeof(Elt) == 2 ? 4 : 2;
        if (V * (int64_t)sizeof(Elt) <= 96 * 1024)
            hipLaunchKernelGGL((kl_grad_rows_kernel<Elt, 256, R, 0>), dim3((unsigned)T), dim3(256), 0, st, ref, q, V, ldr, ldq,
                               w, total, kl, kl64, grad, ldg);
        else
            hipLaunchKernelGGL((kl_grad_rows_kernel<Elt, 1024, R, R>), dim3((unsigned)T), dim3(1024), 0, st, ref, q, V, ldr,
                               ldq, w, total, kl, kl64, grad, ldg);
        LAMQ_LAUNCH_CHECK();
    } else {
        const int64_t span = cdiv(cdiv(V, split), 8) * 8;  // the last spans may be empty
        const dim3 grid((unsigned)(T * split));
        hipLaunchKernelGGL(kl_part_kernel<Elt>, grid, dim3(KG_NT), 0, st, ref, q, V, ldr, ldq, w, span, split, parts);
        LAMQ_LAUNCH_CHECK();
        hipLaunchKernelGGL(kl_grad_part_kernel<Elt>, grid, dim3(KG_NT), 0, st, ref, q, T, V, ldr, ldq, w, span, split,
                           parts, kl, kl64, grad, ldg);
        LAMQ_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(kl_loss_kernel, dim3(1), dim3(1024), 0, st, kl64, w, T, loss);
    LAMQ_LAUNCH_CHECK();
    return LAMQ_OK;
}

extern "C" int lamq_kl_rows_grad(const uint16_t* ref, const uint16_t* q, int64_t T, int64_t V, int64_t ldr, int64_t ldq,
                                 const float* w, float* kl, float* loss, uint16_t* grad, int64_t ldg, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    return kl_grad_launch(ref, q, T, V, ldr, ldq, w, kl, loss, grad, ldg, workspace, workspace_bytes, stream);
}

extern "C" int lamq_kl_rows_grad_f32(const float* ref, const float* q, int64_t T, int64_t V, int64_t ldr, int64_t ldq,
                                     const float* w, float* kl, float* loss, float* grad, int64_t ldg, void* workspace,
                                     size_t workspace_bytes, void* stream)
{
    return kl_grad_launch(ref, q, T, V, ldr, ldq, w, kl, loss, grad, ldg, workspace, workspace_bytes, stream);
}
