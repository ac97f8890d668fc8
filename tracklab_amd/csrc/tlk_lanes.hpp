// tlk_lanes.hpp -- reductions across the lanes of a wavefront without LDS: DPP within 16 lanes, the row swaps of gfx950 between them (a __shfl_xor is an
// LDS round trip of ~100 cycles; these are one or two VALU instructions).  Every lane ends with the result, in the same order on every run.
#pragma once
#include "tlk_common.hpp"

namespace tlk {

struct LaneAdd { static __device__ __forceinline__ float op(float a, float b) { return a + b; } };
struct LaneMax { static __device__ __forceinline__ float op(float a, float b) { return fmaxf(a, b); } };

template <int CTRL> __device__ __forceinline__ float lane_dpp(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }

// over lanes that differ in bit 4 / bit 5: both operands of a swap hold v, so its two results hold the even and the odd rows (halves)
template <class OP> __device__ __forceinline__ float lanes_16(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    return OP::op(__int_as_float(r[0]), __int_as_float(r[1]));
}
template <class OP> __device__ __forceinline__ float lanes_32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return OP::op(__int_as_float(r[0]), __int_as_float(r[1]));
}
// over runs of N = 16, 32 or 64 lanes
template <class OP, int N> __device__ __forceinline__ float lanes_all(float v)
{
    v = OP::op(v, lane_dpp<0xB1>(v));               // lane ^ 1
    v = OP::op(v, lane_dpp<0x4E>(v));               // lane ^ 2
    v = OP::op(v, lane_dpp<0x141>(v));              // 7 - lane of 8: the other four
    v = OP::op(v, lane_dpp<0x140>(v));              // 15 - lane of 16: the other eight
    if (N >= 32) v = lanes_16<OP>(v);
    if (N >= 64) v = lanes_32<OP>(v);
    return v;
}

// a barrier for LDS alone: __syncthreads() would also wait for loads from HBM that are on their way to registers
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);             // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace tlk
