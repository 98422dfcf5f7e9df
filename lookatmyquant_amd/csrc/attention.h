// What the attention kernels share: the MFMA operand types, the lane combines and the grids' rows.
#pragma once
#include "common.h"

typedef __bf16 lamq_at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float lamq_at_f32x16 __attribute__((ext_vector_type(16)));
typedef short lamq_at_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lamq_at_s4 lamq_at_lds_s4;

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
