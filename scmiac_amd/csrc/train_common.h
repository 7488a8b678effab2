// Shared by the training-side kernels (dense layer, distillation, top logits): element types,
// 16-byte vectors, wave reductions.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace scmiac {
namespace train {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef _Float16 f16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    return static_cast<float>(v);
}
// round to nearest even (a float that is too large for fp16 becomes an infinity)
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);
}

// the elements of one 16-byte vector, as floats
template <typename T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    u32x4 raw;
    __device__ __forceinline__ float get(int i) const;
    __device__ __forceinline__ void set(const float (&v)[N]);
};
template <>
__device__ __forceinline__ float Vec16<float>::get(int i) const {
    return __builtin_bit_cast(f32x4, raw)[i];
}
template <>
__device__ __forceinline__ void Vec16<float>::set(const float (&v)[4]) {
    f32x4 t = {v[0], v[1], v[2], v[3]};
    raw = __builtin_bit_cast(u32x4, t);
}
template <>
__device__ __forceinline__ float Vec16<bf16>::get(int i) const {
    const uint32_t w = raw[i >> 1];
    return __builtin_bit_cast(float, (i & 1) ? (w & 0xffff0000u) : (w << 16));
}
template <>
__device__ __forceinline__ void Vec16<bf16>::set(const float (&v)[8]) {
    bf16x8 t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = static_cast<bf16>(v[i]);
    raw = __builtin_bit_cast(u32x4, t);
}
template <>
__device__ __forceinline__ float Vec16<f16>::get(int i) const {
    return static_cast<float>(__builtin_bit_cast(f16x8, raw)[i]);
}
template <>
__device__ __forceinline__ void Vec16<f16>::set(const float (&v)[8]) {
    f16x8 t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = static_cast<f16>(v[i]);
    raw = __builtin_bit_cast(u32x4, t);
}

// 16 bytes that start at any element (the memory pipe takes unaligned addresses; a load then touches one line more)
template <typename T>
__device__ __forceinline__ Vec16<T> load_vec(const T* p) {
    Vec16<T> v;
    __builtin_memcpy(&v.raw, p, 16);
    return v;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// the wave's number in its block, known to be the same in all lanes
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// lanes for which b holds (straight from the comparison's mask)
__device__ __forceinline__ unsigned long long ballot(bool b) { return __builtin_amdgcn_ballot_w64(b); }
__device__ __forceinline__ bool any_lane(bool b) { return ballot(b) != 0; }

// Between LDS writes and reads of different lanes of one wave (which the LDS serves in order): keeps the
// compiler from moving one across the other.
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}

// a value that is the same in all lanes, known to be
__device__ __forceinline__ float uniform(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

static inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
static inline long long round_up(long long a, long long b) { return ceil_div(a, b) * b; }

}  // namespace train
}  // namespace scmiac
