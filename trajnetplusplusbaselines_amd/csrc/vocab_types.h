// Element types of the vocabulary operators (token_embed.hip, vocab_ce.hip): fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include "tnp_internal.h"

namespace tnp {

struct bf16_t { uint16_t bits; };
typedef _Float16 half_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(half_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ half_t from_f32<half_t>(float v) { return (half_t)v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
    const __bf16 b = (__bf16)v;                       // round to nearest even, NaN stays NaN
    return bf16_t{__builtin_bit_cast(uint16_t, b)};
}

// VE consecutive elements moved as one access of VE * sizeof(T) bytes; the address must be a multiple of that
template <typename T, int VE> struct alignas(VE * sizeof(T)) Pack { T v[VE]; };

static constexpr int VOCAB_MAX_DEVICES = 64;      // per-device caches of kernel attributes
inline size_t dtype_bytes(int dtype) { return dtype == TNP_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == TNP_F32 || dtype == TNP_BF16 || dtype == TNP_F16; }

}  // namespace tnp
