// Matrix fragments of the sequence operators (band.hip, cache.hip) for the three storage types: 0 = f32, 1 = bf16, 2 = fp16.
//
// One product step contracts eight elements per lane.  With 16-bit operands that is one v_mfma_f32_16x16x32: lane (n = lane & 15,
// g = lane >> 4) holds row n and the contracted slots 8 g .. 8 g + 7.  With f32 operands the same eight elements go through eight
// v_mfma_f32_16x16x4: step i contracts element i of the four lanes g, so over the eight steps every slot (g, i) meets its partner --
// the order of a sum is free as long as both operands use the same one.  The accumulator of both: column n, rows 4 g + r.
#pragma once
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define SEQ_LOG2E 1.4426950408889634f
// exponents are taken to base 2: a scale whose product with log2(e) is no finite float32 would turn scores of zero into NaN
static inline bool seq_scale_ok(float scale) { return scale * SEQ_LOG2E < INFINITY && scale * SEQ_LOG2E > -INFINITY; }

template <int DT> struct SeqT { typedef unsigned short elem; static constexpr int bytes = 2, words = 4; };   // words: registers of eight elements
template <> struct SeqT<0> { typedef float elem; static constexpr int bytes = 4, words = 8; };

template <int DT> struct Frag { unsigned w[SeqT<DT>::words]; };

template <int DT> __device__ __forceinline__ f32x4 seq_mma(const Frag<DT>& a, const Frag<DT>& b, f32x4 c) {
    if constexpr (DT == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[i]), __uint_as_float(b.w[i]), c, 0, 0, 0);
        return c;
    } else {
        const u32x4 x = {a.w[0], a.w[1], a.w[2], a.w[3]}, y = {b.w[0], b.w[1], b.w[2], b.w[3]};
        if constexpr (DT == 1) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    }
}

// two f32 -> one register of two 16-bit values, rounded to nearest even
template <int DT> __device__ __forceinline__ unsigned seq_pack(float a, float b) {
    if constexpr (DT == 1) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(unsigned, v);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(unsigned, v);
    }
}
template <int DT> __device__ __forceinline__ float seq_lo(unsigned w) {
    if constexpr (DT == 1) return __uint_as_float(w << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)(w & 0xffffu));
}
template <int DT> __device__ __forceinline__ float seq_hi(unsigned w) {
    if constexpr (DT == 1) return __uint_as_float(w & 0xffff0000u);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
}
// x less the lower / upper of two 16-bit values.  fp16: one v_fma_mix_f32 that reads the half where it is (written as a conversion and a
// difference the compiler rounds x a second time instead of taking the half out of its register).  x must not be a matrix instruction's own
// result: the compiler puts no wait for that before the instruction.
template <int DT> __device__ __forceinline__ float seq_less_lo(float x, unsigned w) {
    if constexpr (DT == 1) return x - seq_lo<DT>(w);
#ifdef __HIP_DEVICE_COMPILE__
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(x));
    return r;
#else
    return x - seq_lo<DT>(w);
#endif
}
template <int DT> __device__ __forceinline__ float seq_less_hi(float x, unsigned w) {
    if constexpr (DT == 1) return x - seq_hi<DT>(w);
#ifdef __HIP_DEVICE_COMPILE__
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(x));
    return r;
#else
    return x - seq_hi<DT>(w);
#endif
}
template <int DT> __device__ __forceinline__ void seq_store1(void* p, int64_t i, float x) {
    if constexpr (DT == 0) static_cast<float*>(p)[i] = x;
    else static_cast<unsigned short*>(p)[i] = (unsigned short)(seq_pack<DT>(x, 0.f) & 0xffffu);
}

__device__ __forceinline__ float seq_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// maximum / sum over the four lanes g of a column n: the two row swaps leave every lane with its own and its partner's value
__device__ __forceinline__ float seq_max_g(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float seq_sum_g(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
