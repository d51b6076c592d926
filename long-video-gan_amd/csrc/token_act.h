// token_act.h -- what the products of token rows do with their sums before they are stored (token_gemm.h, token_stream.hip, token_finish.hip):
//
//   linear   y = clamp(act(sum * scales + b) * gain) + residual                 slope = gain-free derivative of clamp(act(.)), one a value
//   gated    h = gain * act(g) * u,  g = sum * scales + b of the gate half, u of the up half      slopes dh/dg and dh/du
//
// Everything here is float32; the result is rounded once, to the output's type. The slopes are what the gradient multiplies with. They are kept
// as the forward pass has them, in float32 (or, where the derivative takes only the values 0, 1 and alpha, as one byte that says which): the
// gradient's operand dy * slope then has ONE rounding to 16 bits, and a sum next to a kink keeps the side it was computed on. Saving them in 16
// bits would halve their traffic (7 % of a gated training step at 8192 x 2048 x 8192) and make the error of the weight gradient 1.7 times
// that of its own rounding instead of 1.4.
#pragma once
#include "row_common.h"

enum { LVG_SLOPE_NONE = 0, LVG_SLOPE_F32 = 1, LVG_SLOPE_CODE = 2 };

struct Finish
{
    const float* qs;           // [rows] scales of 8-bit rows, or NULL
    const float* ps;           // [cols] (gated: [2 cols]) scales of 8-bit weights, or NULL
    const void*  bias;         // [cols] (gated: [2 cols]) in the output's type, or NULL
    const void*  residual;     // or NULL
    void*        out;
    void*        slopes;       // [rows][cols] (gated: [rows][2 cols]), or NULL
    int64_t      ldr, ldo;     // elements
    int64_t      rows;
    int64_t      cols;         // of the result; gated: the up half lies cols behind the gate half
    int          act, slopeKind;
    float        alpha, gain, clamp;
    bool         vec;          // the four values of a call may be moved as one vector
};

namespace {

// a = act(v); with WANT also d = act'(v). Branches are uniform over the launch.
__device__ __forceinline__ void act_value(int act, float alpha, float v, bool want, float& a, float& d)
{
    constexpr float kSeluScale = 1.0507009873554804934193349852946f, kSeluAlpha = 1.6732632423543772848170429916717f;
    d = 1.f;
    switch (act)
    {
        case LVG_ACT_RELU:
            // (a NaN stays one)
            a = v <= 0.f ? 0.f : v;
            d = v > 0.f ? 1.f : 0.f;
            break;
        case LVG_ACT_LRELU:
            a = v > 0.f ? v : v * alpha;
            d = v > 0.f ? 1.f : alpha;
            break;
        case LVG_ACT_TANH:
            a = tanhf(v);
            d = fmaf(-a, a, 1.f);
            break;
        case LVG_ACT_SIGMOID:
            a = 1.f / (1.f + expf(-v));
            d = a * (1.f - a);
            break;
        case LVG_ACT_ELU:
            a = v >= 0.f ? v : expm1f(v);
            if (want) d = v >= 0.f ? 1.f : expf(v);
            break;
        case LVG_ACT_SELU:
            a = v >= 0.f ? kSeluScale * v : (kSeluScale * kSeluAlpha) * expm1f(v);
            if (want) d = v >= 0.f ? kSeluScale : (kSeluScale * kSeluAlpha) * expf(v);
            break;
        case LVG_ACT_SOFTPLUS:
            a = fmaxf(v, 0.f) + log1pf(expf(-fabsf(v)));
            if (want) d = 1.f / (1.f + expf(-v));
            break;
        case LVG_ACT_SWISH:
        {
            const float s = 1.f / (1.f + expf(-v));
            a = v * s;
            d = s * fmaf(v, 1.f - s, 1.f);
            break;
        }
        default:
            a = v;
    }
}

template <class T> struct alignas(4 * sizeof(T)) Quad { T v[4]; };

template <class T> __device__ __forceinline__ void quad_load(const T* p, int64_t n, bool vec, float* v)
{
    if (vec && n >= 4)
    {
        const Quad<T> q = *reinterpret_cast<const Quad<T>*>(p);
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = row_load(q.v[i]);
    }
    else
    {
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = i < n ? row_load(p[i]) : 0.f;
    }
}

template <class T> __device__ __forceinline__ void quad_store(T* p, int64_t n, bool vec, const float* v)
{
    Quad<T> q;
    #pragma unroll
    for (int i = 0; i < 4; i++) q.v[i] = from_acc<T>(v[i]);
    if (vec && n >= 4) *reinterpret_cast<Quad<T>*>(p) = q;
    else
    {
        #pragma unroll
        for (int i = 0; i < 4; i++) if (i < n) p[i] = q.v[i];
    }
}

// Four neighbouring sums, row m, columns n .. n + 3 (those below cols): scales and bias. v: sums; gated: v of the gate half, u of the up half.
template <class O, bool GATED> __device__ __forceinline__ void prepare4(const Finish& f, int64_t m, int64_t n, float* v, float* u)
{
    const int64_t left = f.cols - n;
    if (f.qs)
    {
        const float s = f.qs[m];
        #pragma unroll
        for (int i = 0; i < 4; i++) if (i < left)
        {
            v[i] *= s * f.ps[n + i];
            if (GATED) u[i] *= s * f.ps[f.cols + n + i];
        }
    }
    if (f.bias)
    {
        float b[4];
        quad_load(static_cast<const O*>(f.bias) + n, left, f.vec, b);
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] += b[i];
        if (GATED)
        {
            quad_load(static_cast<const O*>(f.bias) + f.cols + n, left, f.vec, b);
            #pragma unroll
            for (int i = 0; i < 4; i++) u[i] += b[i];
        }
    }
}

// The results of four such sums: activation, slopes, residual, store.
template <class O, bool GATED> __device__ __forceinline__ void finish4(const Finish& f, int64_t m, int64_t n, float* v, float* u)
{
    const int64_t left = f.cols - n;
    float a[4], d[4];
    const bool want = f.slopeKind != LVG_SLOPE_NONE;
    #pragma unroll
    for (int i = 0; i < 4; i++) act_value(f.act, f.alpha, v[i], want, a[i], d[i]);
    if (GATED)
    {
        float up[4];
        #pragma unroll
        for (int i = 0; i < 4; i++)
        {
            up[i] = a[i] * f.gain;              // dh/du
            d[i] = d[i] * u[i] * f.gain;        // dh/dg
            a[i] = up[i] * u[i];
        }
        if (want)
        {
            float* s = static_cast<float*>(f.slopes) + m * 2 * f.cols + n;
            quad_store(s, left, f.vec, d);
            quad_store(s + f.cols, left, f.vec, up);
        }
        quad_store(static_cast<O*>(f.out) + m * f.ldo + n, left, f.vec, a);
        return;
    }
    uint32_t code = 0;
    #pragma unroll
    for (int i = 0; i < 4; i++)
    {
        a[i] *= f.gain;
        bool inside = true;
        if (f.clamp >= 0.f)
        {
            inside = !(fabsf(a[i]) >= f.clamp);         // (a NaN is inside: it stays one)
            if (!inside) { a[i] = a[i] > 0.f ? f.clamp : -f.clamp; d[i] = 0.f; }
        }
        // 0: no gradient, 1: alpha (lrelu's lower side; relu has alpha 0), 2: one
        code |= (uint32_t)(!inside ? 0 : (f.act != LVG_ACT_LINEAR && !(v[i] > 0.f)) ? 1 : 2) << (8 * i);
    }
    if (f.slopeKind == LVG_SLOPE_F32) quad_store(static_cast<float*>(f.slopes) + m * f.cols + n, left, f.vec, d);
    else if (f.slopeKind == LVG_SLOPE_CODE)
    {
        uint8_t* s = static_cast<uint8_t*>(f.slopes) + m * f.cols + n;
        if (f.vec && left >= 4) *reinterpret_cast<uint32_t*>(s) = code;
        else
        {
            #pragma unroll
            for (int i = 0; i < 4; i++) if (i < left) s[i] = (uint8_t)(code >> (8 * i));
        }
    }
    if (f.residual)
    {
        float r[4];
        quad_load(static_cast<const O*>(f.residual) + m * f.ldr + n, left, f.vec, r);
        #pragma unroll
        for (int i = 0; i < 4; i++) a[i] += r[i];
    }
    quad_store(static_cast<O*>(f.out) + m * f.ldo + n, left, f.vec, a);
}

} // namespace
