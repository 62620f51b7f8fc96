// What the prompt kernels (fh_attention_prefill.hip, fh_paged_prompt.hip) share: scores and outputs are 32 x 32 accumulators whose
// column, lane % 32, is the lane's query; g = lane / 32.
#pragma once
#include "fh_blocks.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float ap_swap32_max(float v) {
    const uint32_t u = __float_as_uint(v);
    auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float ap_swap32_sum(float v) {
    const uint32_t u = __float_as_uint(v);
    auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ void ap_store4(float *p, float a, float b, float c, float d) {
    *(float4 *)p = make_float4(a, b, c, d);
}
__device__ __forceinline__ void ap_store4(fh_half *p, float a, float b, float c, float d) {
    const fh_half h[4] = {(fh_half)a, (fh_half)b, (fh_half)c, (fh_half)d};
    uint2 u;
    __builtin_memcpy(&u, h, 8);
    *(uint2 *)p = u;
}
__device__ __forceinline__ void ap_store4(__bf16 *p, float a, float b, float c, float d) {
    const __bf16 h[4] = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    uint2 u;
    __builtin_memcpy(&u, h, 8);
    *(uint2 *)p = u;
}

typedef short short4v __attribute__((ext_vector_type(4)));
// Eight halfs of the V^T operand: keys k .. k+7 of the dim this lane stands for (two transposing loads of 4 keys).
__device__ __forceinline__ half8 ap_vt8(const fh_half *p, int row_stride) {
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v *)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
    const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v *)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)(p + 4 * row_stride));
    half8 r;
    __builtin_memcpy(&r, &a, 8);
    __builtin_memcpy((char *)&r + 8, &b, 8);
    return r;
}

// The second group of wavefronts hands its statistics and output over: [value][query wavefront][lane] floats in the tile buffers (the barrier
// that ended the last step has passed: nobody reads them any more).
template <int D, int QW>
__device__ __forceinline__ void ap_merge(float *sm, int wave, int lane, int kset, float &m_run, float &l_run, floatx16 (&acc)[D / 32]) {
    constexpr int NQ = 64 * QW, DT = D / 32;
    const int slot = (wave % QW) * 64 + lane;
    if (kset == 1) {
        sm[slot] = m_run;
        sm[NQ + slot] = l_run;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r++) sm[(2 + dt * 16 + r) * NQ + slot] = acc[dt][r];
    }
    __syncthreads();
    if (kset == 1) return;
    const float m1 = sm[slot], l1 = sm[NQ + slot];
    const float mm = fmaxf(m_run, m1), ref = mm == -INFINITY ? 0.f : mm;
    const float f0 = __builtin_amdgcn_exp2f(m_run - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
    m_run = mm, l_run = l_run * f0 + l1 * f1;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[dt][r] = acc[dt][r] * f0 + sm[(2 + dt * 16 + r) * NQ + slot] * f1;
}

// lane = query, register r of d-tile dt is d = 32 dt + 8 (r / 4) + 4 g + r % 4
template <int D, typename TQ>
__device__ __forceinline__ void ap_store(TQ *op, int g, float inv, const floatx16 (&acc)[D / 32]) {
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++)
            ap_store4(op + 32 * dt + 8 * r4 + 4 * g, acc[dt][4 * r4] * inv, acc[dt][4 * r4 + 1] * inv, acc[dt][4 * r4 + 2] * inv,
                      acc[dt][4 * r4 + 3] * inv);
}

