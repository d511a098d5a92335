// Shared by the kernels of the decoder layer around the experts (norm, rotary positions, paged cache): element types,
// 16-byte vectors of them, and the launch parameters that the C entries fill in.
#pragma once

#include "layer_params.h"
#include "moe_common.h"

namespace cmoe {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));  // a vector at any element's address: global accesses
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));  // of gfx950 need no alignment beyond the element's

// Two fp32 values as two 16-bit ones, rounded to nearest even, in one conversion (low half = a).
__device__ __forceinline__ uint32_t cvt_bf16x2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ uint32_t cvt_f16x2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

struct TypeBf16 {
    typedef uint16_t raw;
    typedef u32x4_a2 loose;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(raw v) { return bf16_bits_to_f32(v); }
    static __device__ __forceinline__ raw put(float v) { return f32_to_bf16_bits(v); }
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(r[i]), f[2 * i + 1] = bf16_hi(r[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        return u32x4{cvt_bf16x2(f[0], f[1]), cvt_bf16x2(f[2], f[3]), cvt_bf16x2(f[4], f[5]), cvt_bf16x2(f[6], f[7])};
    }
};

struct TypeF16 {
    typedef uint16_t raw;
    typedef u32x4_a2 loose;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
        const f16x8 h = __builtin_bit_cast(f16x8, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        return u32x4{cvt_f16x2(f[0], f[1]), cvt_f16x2(f[2], f[3]), cvt_f16x2(f[4], f[5]), cvt_f16x2(f[6], f[7])};
    }
};

struct TypeF32 {
    typedef float raw;
    typedef u32x4_a4 loose;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float get(raw v) { return v; }
    static __device__ __forceinline__ raw put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const u32x4& r, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* f) {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
};

template <class T>
__device__ __forceinline__ u32x4 load_vec(const typename T::raw* p) {
    return *reinterpret_cast<const typename T::loose*>(p);
}
template <class T>
__device__ __forceinline__ void store_vec(typename T::raw* p, const u32x4& v) {
    *reinterpret_cast<typename T::loose*>(p) = v;
}

}  // namespace cmoe
