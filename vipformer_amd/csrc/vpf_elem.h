// vpf_elem.h -- element types of the block operators (rotary.hip, gated_norm.hip, window_attention.hip): fp32, fp16 and bf16 tensors are
// chosen per CALL by the VPF_T_* codes of the C ABI (the library-wide operand type h16 of vpf_common.h is a build switch).
// Arithmetic is fp32; a store rounds once, to nearest even.
#pragma once
#include "vpf_common.h"

typedef _Float16 vpf_f16;
typedef __bf16 vpf_bf16;

static inline bool vpf_elem_ok(int code) { return code == VPF_T_F32 || code == VPF_T_F16 || code == VPF_T_BF16; }
static inline bool vpf_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// N consecutive elements as one access of N * sizeof(T) bytes (16-byte pieces where it is larger); the caller guarantees the alignment
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) VpfPack { T e[N]; };
template <typename T, int N> __device__ __forceinline__ void vpf_store(T* p, const float* v)
{
    VpfPack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.e[i] = (T)v[i];
    *reinterpret_cast<VpfPack<T, N>*>(p) = r;
}
// The same N elements unconverted, in whole registers: a load whose value is first needed much later (converting it at once would make the
// wave wait right behind the load; so would a branch around it -- load from a clamped address and drop the value instead).
template <typename T, int N> struct VpfRaw {
    static constexpr int BYTES = N * (int)sizeof(T), WORDS = (BYTES + 3) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (BYTES == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
        else if constexpr (BYTES == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
        else w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return (float)__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
    }
};
