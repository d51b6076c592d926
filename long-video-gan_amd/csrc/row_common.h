// row_common.h -- pieces shared by the kernels on matrices of rows (rms_norm.hip, token_*.hip): masked vector access to rows that may start at
// any element, e4m3 conversion, the activations in float32 with their derivatives.
#pragma once
#include "lvg_common.h"
#include <algorithm>
#include <string.h>

namespace {

constexpr int64_t kGridBlocks = ((int64_t)1 << 24) - 1;  // workgroups of 256: a grid holds fewer than 2^32 threads
constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 5.421010862427522e-20f;     // 2^-64: the scale of a row of zeros; its reciprocal is still finite

__device__ __forceinline__ float row_load(float v)  { return v; }
__device__ __forceinline__ float row_load(f16_t v)  { return to_acc(v); }
__device__ __forceinline__ float row_load(bf16_t v) { return to_acc(v); }

// n of the V elements at p (the others zero). A row starts wherever its stride puts it, so the full access is an unaligned 16-byte one, which
// the global memory path takes; only the last vector of a row goes element by element.
template <class T> __device__ __forceinline__ void load_row(const T* p, int64_t n, float* v)
{
    constexpr int V = Elem<T>::kVec;
    if (n >= V)
    {
        T r[V];
        __builtin_memcpy(r, p, 16);
        #pragma unroll
        for (int i = 0; i < V; i++) v[i] = row_load(r[i]);
    }
    else
    {
        #pragma unroll
        for (int i = 0; i < V; i++) v[i] = i < n ? row_load(p[i]) : 0.f;
    }
}

// The same in two steps, for loads that are to be on their way early: the raw vector, then its values.
template <class T> struct RawRow { T v[Elem<T>::kVec]; };
// once: 16-byte aligned rows of more than the caches hold, read by nobody else.
template <class T> __device__ __forceinline__ RawRow<T> load_raw(const T* p, int64_t n, bool once = false)
{
    constexpr int V = Elem<T>::kVec;
    RawRow<T> r;
    if (n >= V && once)
    {
        typedef uint32_t vec __attribute__((ext_vector_type(4)));
        const vec w = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p));
        __builtin_memcpy(&r, &w, 16);
    }
    else if (n >= V) __builtin_memcpy(&r, p, 16);
    else
    {
        __builtin_memset(&r, 0, 16);
        #pragma unroll
        for (int i = 0; i < V; i++) if (i < n) r.v[i] = p[i];
    }
    return r;
}

// past: 16-byte aligned rows of a result larger than the caches, stored past them.
template <class T> __device__ __forceinline__ void store_row(T* p, int64_t n, const float* v, bool past = false)
{
    constexpr int V = Elem<T>::kVec;
    T r[V];
    #pragma unroll
    for (int i = 0; i < V; i++) r[i] = from_acc<T>(v[i]);
    if (n >= V && past)
    {
        typedef uint32_t vec __attribute__((ext_vector_type(4)));
        vec w;
        __builtin_memcpy(&w, r, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<vec*>(p));
    }
    else if (n >= V) __builtin_memcpy(p, r, 16);
    else
    {
        #pragma unroll
        for (int i = 0; i < V; i++) if (i < n) p[i] = r[i];
    }
}

// Four values to e4m3 (round to nearest even), clamped to the finite range; a NaN stays one.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d)
{
    auto bound = [](float v) { return v != v ? v : fminf(fmaxf(v, -kE4m3Max), kE4m3Max); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(bound(a), bound(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(bound(c), bound(d), w, true);
    return (uint32_t)w;
}

// Two bits beside a rounded value: what rounding v to T left, in units of two thirds of half a step: -1, 0 or 1 (+ 1), a third of it at most is lost.
// A half step is 2^(exponent - 11) of float16 (its subnormals' is larger: theirs stay within the half step itself); bfloat16 is the upper half of a
// float32, a half step 0x8000 of its lower half (zeros, infinities and NaNs stay what they are: nothing is left of them, or it stays within their patterns).
__device__ __forceinline__ float half_step(float rounded) { return __uint_as_float(__float_as_uint(rounded) & 0x7f800000u) * 0.00048828125f; }
template <class T> __device__ __forceinline__ uint32_t rest_code(float v)
{
    if constexpr (__is_same(T, bf16_t))
    {
        const int left = (int)(__float_as_uint(v) - ((uint32_t)from_acc<bf16_t>(v).bits << 16));
        return left > 0x2aaa ? 2u : left < -0x2aaa ? 0u : 1u;
    }
    const float r = to_acc(from_acc<f16_t>(v)), left = v - r, third = half_step(r) * (1.f / 3.f);
    return left > third ? 2u : left < -third ? 0u : 1u;
}
template <class T> __device__ __forceinline__ float with_rest(float rounded, uint32_t code)
{
    if constexpr (__is_same(T, bf16_t)) return __uint_as_float(__float_as_uint(rounded) + code * 0x5555u - 0x5555u);
    return code == 1u ? rounded : fmaf((float)(int)(code - 1u), half_step(rounded) * (2.f / 3.f), rounded);
}

__device__ __forceinline__ float wave_total(float v)
{
    #pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Largest magnitude as bits: integers order like the floats they are, with infinity above every number and NaN above infinity, so a NaN is kept.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_largest(uint32_t v)
{
    #pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// scale = largest / 448, at least 2^-64 (a NaN stays one).
__device__ __forceinline__ float row_scale(uint32_t largest)
{
    const float s = __uint_as_float(largest) / kE4m3Max;
    return s < kScaleMin ? kScaleMin : s;
}

// Quotients by one scale, rounded as a division rounds them. The reciprocal and what its rounding left give a quotient within one unit in the last
// place; the exact remainder corrects it to the nearest value (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).
// Values of 16 bits meet e4m3's ties often: with the rounded reciprocal alone 4 % of the rows of 8192 bfloat16 hold a code that is off by a step. A
// division an element would take three times the instructions.
struct Divisor
{
    float scale, inv, rest;
    __device__ __forceinline__ explicit Divisor(float s) : scale(s), inv(1.f / s), rest(fmaf(-s, inv, 1.f) * inv)
    {
        if (isinf(s)) scale = rest = 0.f;          // finite / infinity = 0, infinity / infinity = NaN
    }
    __device__ __forceinline__ float quotient(float v) const
    {
        const float q = fmaf(v, inv, v * rest);
        return fmaf(fmaf(-q, scale, v), inv, q);
    }
};

} // namespace

// out [width] (type dtype) = gain * sum over the slots of part [slots][width] (rms_norm.hip).
void row_column_sum(const float* part, void* out, int slots, int64_t width, float gain, int dtype, hipStream_t s);
