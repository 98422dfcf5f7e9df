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
// accesses at element alignment), as float32.
typedef uint32_t kg_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float kg_f4 __attribute__((ext_vector_type(4), aligned(4)));
struct KGChunk {
    float v[8];
};
__device__ __forceinline__ KGChunk kg_load8(const uint16_t* p)
{
    const kg_u4 x = *reinterpret_cast<const kg_u4*>(p);
    KGChunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c.v[2 * i] = __uint_as_float(x[i] << 16);
        c.v[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
    }
    return c;
}
__device__ __forceinline__ KGChunk kg_load8(const float* p)
{
    const kg_f4 x = reinterpret_cast<const kg_f4*>(p)[0], y = reinterpret_cast<const kg_f4*>(p)[1];
    KGChunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c.v[i] = x[i];
        c.v[4 + i] = y[i];
    }
    return c;
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

// A part of a row: both maxima, s_r and s_q relative to them, and a = sum e^(r - m_r) (r - q)
struct KGPart {
    float mr, mq;
    double sr, ar, sq;
};

// a maximum to subtract, 0 where there is none yet (every logit so far -inf: their exponentials are 0)
__device__ __forceinline__ float kg_base(float m) { return m == -kg_inf() ? 0.0f : m; }
// e^(x - base): the difference first, which no logit and maximum of the type can make overflow upwards
__device__ __forceinline__ float kg_exp(float x, float base)
{
    return __builtin_amdgcn_exp2f((x - base) * 1.4426950408889634f);
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
    if (cr > p.mr) {
        const double f = p.mr == -kg_inf() ? 0.0 : (double)__expf(p.mr - cr);
        p.sr *= f;
        p.ar = kg_keep_inf(p.ar, f);
        p.mr = cr;
    }
    if (cq > p.mq) {
        p.sq *= p.mq == -kg_inf() ? 0.0 : (double)__expf(p.mq - cq);
        p.mq = cq;
    }
    const float br = kg_base(p.mr), bq = kg_base(p.mq);
    float sr = 0.0f, ar = 0.0f, sq = 0.0f;
    if (lo < -1e30f) {  // masked words, by -inf or the type's lowest value: the terms that would be 0 times infinity
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float er = kg_exp(r.v[e], br);
            sr += er;
            if (r.v[e] != -kg_inf() && q.v[e] == -kg_inf())
                ar = kg_inf();
            else if (er > 0.0f)
                ar += er * (r.v[e] - q.v[e]);
            sq += kg_exp(q.v[e], bq);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float er = kg_exp(r.v[e], br);
            sr += er;
            ar = fmaf(er, r.v[e] - q.v[e], ar);
            sq += kg_exp(q.v[e], bq);
        }
    }
    p.sr += (double)sr;
    p.ar += (double)ar;
    p.sq += (double)sq;
}

// x times e^(m - M), for a part's sum and maximum against a larger maximum
__device__ __forceinline__ double kg_scaled(double x, float m, float M)
{
    return m == -kg_inf() ? 0.0 : m == M ? x : kg_keep_inf(x, exp((double)m - (double)M));
}

// The sum of the workgroup's parts, in every thread: the maxima, then the sums by waves and over them, in a fixed order.
__device__ __forceinline__ KGPart kg_reduce(KGPart p)
{
    __shared__ float m[2][KG_NT / 64];
    __shared__ double s[3][KG_NT / 64];
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
    for (int w = 1; w < KG_NT / 64; ++w) {
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
    for (int w = 0; w < KG_NT / 64; ++w) {
        t.sr += s[0][w];
        t.ar += s[1][w];
        t.sq += s[2][w];
    }
    __syncthreads();  // the arrays are free again
    return t;
}

__device__ __forceinline__ double kg_kl(const KGPart& t)
{
    return t.ar / t.sr - ((double)t.mr + log(t.sr)) + ((double)t.mq + log(t.sq));
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

// The gradient of those logits: fq e^(q - m_q) - fr e^(r - m_r), fq = coef / s_q and fr = coef / s_r
template <typename Elt>
__device__ __forceinline__ void kg_grad(const Elt* r, const Elt* q, Elt* g, int64_t v0, int64_t v1, const KGPart& t,
                                        double coef)
{
    const float fr = (float)(coef / t.sr), fq = (float)(coef / t.sq), br = kg_base(t.mr), bq = kg_base(t.mq);
    int64_t v = v0 + 8 * (int64_t)threadIdx.x;
    for (; v + 8 <= v1; v += 8 * KG_NT) {
        const KGChunk a = kg_load8(r + v), b = kg_load8(q + v);
        KGChunk c;
#pragma unroll
        for (int e = 0; e < 8; ++e) c.v[e] = fmaf(kg_exp(b.v[e], bq), fq, -(kg_exp(a.v[e], br) * fr));
        kg_store8(g + v, c);
    }
    for (; v < v1; ++v)
        kg_store1(g + v, fmaf(kg_exp(kg_load1(q + v), bq), fq, -(kg_exp(kg_load1(r + v), br) * fr)));
}

template <typename Elt>
__device__ __forceinline__ void kg_zero(Elt* g, int64_t v0, int64_t v1)
{
    KGChunk z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z.v[e] = 0.0f;
    int64_t v = v0 + 8 * (int64_t)threadIdx.x;
    for (; v + 8 <= v1; v += 8 * KG_NT) kg_store8(g + v, z);
    for (; v < v1; ++v) kg_store1(g + v, 0.0f);
}

// the workgroup's sum of x, in every thread, in a fixed order
__device__ __forceinline__ double kg_sum(double x)
{
    __shared__ double s[KG_NT / 64];
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < KG_NT / 64; ++w) t += s[w];
    __syncthreads();
    return t;
}

// sum w (T without weights) over all T, in every thread
__device__ __forceinline__ double kg_weights(const float* __restrict__ w, int64_t T)
{
    if (!w) return (double)T;
    double x = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += KG_NT) x += (double)w[t];
    return kg_sum(x);
}

__global__ __launch_bounds__(KG_NT) void kl_weights_kernel(const float* __restrict__ w, int64_t T,
                                                           double* __restrict__ total)
{
    const double x = kg_weights(w, T);
    if (threadIdx.x == 0) *total = x;
}

// loss = sum w kl / total, of float64 kl's
__global__ __launch_bounds__(KG_NT) void kl_loss_kernel(const double* __restrict__ kl, const float* __restrict__ w,
                                                        int64_t T, const double* __restrict__ total,
                                                        float* __restrict__ loss)
{
    double x = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += KG_NT) x += (w ? (double)w[t] : 1.0) * kl[t];
    x = kg_sum(x);
    if (threadIdx.x == 0) *loss = (float)(x / *total);
}

// Many rows: a workgroup a row, read for the sums and again (from the caches, where they hold what is in flight) for
// the gradient.
template <typename Elt>
__global__ __launch_bounds__(KG_NT) void kl_grad_rows_kernel(const Elt* __restrict__ ref, const Elt* __restrict__ q,
                                                             int64_t V, int64_t ldr, int64_t ldq,
                                                             const float* __restrict__ w, const double* __restrict__ total,
                                                             float* __restrict__ kl, double* __restrict__ kl64,
                                                             Elt* __restrict__ grad, int64_t ldg)
{
    const int64_t t = blockIdx.x;
    const double wt = w ? (double)w[t] : 1.0;
    Elt* g = grad + t * ldg;
    if (wt == 0.0) {
        kg_zero(g, 0, V);
        if (threadIdx.x == 0) {
            kl[t] = 0.0f;
            kl64[t] = 0.0;
        }
        return;
    }
    const Elt *r = ref + t * ldr, *s = q + t * ldq;
    const KGPart p = kg_reduce(kg_part(r, s, 0, V));
    kg_grad(r, s, g, 0, V, p, wt / *total);
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
        kg_zero(grad + t * ldg, v0, v1);
    } else {
        KGPart p{-kg_inf(), -kg_inf(), 0.0, 0.0, 0.0};
        if ((int)threadIdx.x < split) p = parts[t * split + threadIdx.x];
        p = kg_reduce(p);
        kg_grad(ref + t * ldr, q + t * ldq, grad + t * ldg, v0, v1, p, wt / kg_weights(w, T));
        x = kg_kl(p);
    }
    if (s == 0 && threadIdx.x == 0) {
        kl[t] = (float)x;
        kl64[t] = x;
    }
}

// workgroups a row for T rows of V logits: enough to fill the chip with a few, at least 2,048 logits each
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
    hipLaunchKernelGGL(kl_weights_kernel, dim3(1), dim3(KG_NT), 0, st, w, T, total);
    LAMQ_LAUNCH_CHECK();
    if (split == 1) {
        hipLaunchKernelGGL(kl_grad_rows_kernel<Elt>, dim3((unsigned)T), dim3(KG_NT), 0, st, ref, q, V, ldr, ldq, w, total,
                           kl, kl64, grad, ldg);
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
    hipLaunchKernelGGL(kl_loss_kernel, dim3(1), dim3(KG_NT), 0, st, kl64, w, T, total, loss);
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
