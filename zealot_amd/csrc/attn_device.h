// attn_device.h -- device helpers the decode attention kernels share.
#pragma once

#include <cmath>

#include "zk_common.h"

namespace zk {

// Lane l ^ 16 / l ^ 32's value, on the VALU: v_permlane16_swap exchanges the
// odd 16-lane rows of its first operand with the even rows of its second, and
// v_permlane32_swap the upper half of the first with the lower half of the
// second; with both operands v, a lane's partner value lands in the second
// result on the even rows (lower half) and in the first elsewhere.  (Unlike
// ds_swizzle / ds_bpermute they are not LDS instructions, so they never wait
// behind outstanding LDS or scalar loads.)
__device__ __forceinline__ float xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Another lane's value of the same 16 by the VALU's lane permutations: 0xb1 lane ^
// 1, 0x4e lane ^ 2, 0x141 / 0x140 mirrored in 8 / 16 lanes, 0x120 + n rotated by n.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Two f32 -> packed bf16, round to nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t bf16x2_rne(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2_t));
}

// scale / l for a row of maximum m: 0 where it saw no keys (m = -inf), NaN where
// all their scores were -inf (l = 0 at the lowest finite m).
__device__ __forceinline__ float inverse_sum(float l, float m, float scale = 1.0f) {
    return l > 0.0f ? scale / l : m == -INFINITY ? 0.0f : NAN;
}

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes per lane from global memory straight into LDS at lds + 16 * lane
// (global_load_lds_dwordx4; no VGPRs, counted by vmcnt).  Cache policy NT
// (nontemporal, aux bit 1): every K/V byte is read exactly once, and the
// streaming hint measured ~9% faster than the default policy on C2.
constexpr int kCachePolicyNT = 2;
__device__ __forceinline__ void g2l16(const void *g, lds_void *l) {
    __builtin_amdgcn_global_load_lds(g, l, 16, 0, kCachePolicyNT);
}
// s_waitcnt vmcnt(N) alone (gfx9 encoding: expcnt 7 and lgkmcnt 15 mean "no wait").
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N <= 63, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
// What the wave's lanes wrote to LDS before is what its lanes read after: nothing
// moves across in the compiler (the LDS unit keeps a wave's accesses in order, so no
// instruction comes of it).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xc07f); }

}  // namespace zk
