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

// 1 / (1 + exp(-v)). QUICK (results of 16 bits): the hardware's 2^x of the product's rounded value, times 1 + ln 2 * what the rounding left, and its
// reciprocal: three units in the last place in all, where expf and a division take three times the instructions -- and the vector unit's time
// on a tile's results is what a gated product of a short summed index waits for.
template <bool QUICK> __device__ __forceinline__ float sigmoid(float v)
{
    if (!QUICK) return 1.f / (1.f + expf(-v));
    constexpr float kLog2e = 1.44269504088896340736f, kLog2eRest = 1.92596299112661746887e-8f, kLn2 = 0.693147180559945309417f;
    const float h = -v * kLog2e;
    const float rest = fmaf(-v, kLog2eRest, fmaf(-v, kLog2e, -h));
    // an exponent past the range gives infinity or zero; its rest (a NaN of infinities, too) is not looked at
    const float e = __builtin_amdgcn_exp2f(h);
    return __builtin_amdgcn_rcpf(1.f + (fabsf(h) < 126.f ? e * fmaf(rest, kLn2, 1.f) : e));
}

// Four values: a = act(v), d = act'(v) (where `want` is set). ACT = 0: the activation `act`, one branch for the four, uniform over the launch.
template <int ACT, bool QUICK> __device__ __forceinline__ void act4(int act, float alpha, const float* v, bool want, float* a, float* d)
{
    constexpr float kSeluScale = 1.0507009873554804934193349852946f, kSeluAlpha = 1.6732632423543772848170429916717f;
    #define LVG_EACH _Pragma("unroll") for (int i = 0; i < 4; i++)
    switch (ACT ? ACT : act)
    {
        case LVG_ACT_RELU:
            LVG_EACH { a[i] = v[i] <= 0.f ? 0.f : v[i]; d[i] = v[i] > 0.f ? 1.f : 0.f; }      // (a NaN stays one)
            break;
        case LVG_ACT_LRELU:
            LVG_EACH { a[i] = v[i] > 0.f ? v[i] : v[i] * alpha; d[i] = v[i] > 0.f ? 1.f : alpha; }
            break;
        case LVG_ACT_TANH:
            LVG_EACH { a[i] = tanhf(v[i]); d[i] = fmaf(-a[i], a[i], 1.f); }
            break;
        case LVG_ACT_SIGMOID:
            LVG_EACH { a[i] = sigmoid<QUICK>(v[i]); d[i] = a[i] * (1.f - a[i]); }
            break;
        case LVG_ACT_ELU:
            LVG_EACH { a[i] = v[i] >= 0.f ? v[i] : expm1f(v[i]); d[i] = v[i] >= 0.f || !want ? 1.f : expf(v[i]); }
            break;
        case LVG_ACT_SELU:
            LVG_EACH
            {
                a[i] = v[i] >= 0.f ? kSeluScale * v[i] : (kSeluScale * kSeluAlpha) * expm1f(v[i]);
                d[i] = v[i] >= 0.f || !want ? kSeluScale : (kSeluScale * kSeluAlpha) * expf(v[i]);
            }
            break;
        case LVG_ACT_SOFTPLUS:
            LVG_EACH { a[i] = fmaxf(v[i], 0.f) + log1pf(expf(-fabsf(v[i]))); d[i] = want ? sigmoid<QUICK>(v[i]) : 1.f; }
            break;
        case LVG_ACT_SWISH:
            LVG_EACH
            {
                const float s = sigmoid<QUICK>(v[i]);
                a[i] = v[i] * s;
                d[i] = s * fmaf(v[i], 1.f - s, 1.f);
            }
            break;
        default:
            LVG_EACH { a[i] = v[i]; d[i] = 1.f; }
    }
    #undef LVG_EACH
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

template <class O> __device__ __forceinline__ void residual4(const Finish& f, int64_t m, int64_t n, float* r)
{
    #pragma unroll
    for (int i = 0; i < 4; i++) r[i] = 0.f;
    if (f.residual) quad_load(static_cast<const O*>(f.residual) + m * f.ldr + n, f.cols - n, f.vec, r);
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

// Where four results go: the element of the first in each array.
template <class O> struct Place
{
    O*       out;
    float*   slopes;           // (as bytes: LVG_SLOPE_CODE)
    int64_t  left;             // columns from it on
    __device__ __forceinline__ Place(const Finish& f, int64_t m, int64_t n, bool gated)
    {
        left = f.cols - n;
        out = static_cast<O*>(f.out) + m * f.ldo + n;
        const int64_t s = m * (gated ? 2 : 1) * f.cols + n;
        slopes = f.slopeKind == LVG_SLOPE_F32 ? static_cast<float*>(f.slopes) + s
               : f.slopeKind == LVG_SLOPE_CODE ? reinterpret_cast<float*>(static_cast<uint8_t*>(f.slopes) + s) : nullptr;
    }
    // `rows` rows on
    __device__ __forceinline__ Place down(const Finish& f, int rows, bool gated) const
    {
        Place p = *this;
        p.out += rows * f.ldo;
        const int64_t s = rows * (gated ? 2 : 1) * f.cols;
        if (f.slopeKind == LVG_SLOPE_F32) p.slopes += s;
        else if (f.slopeKind == LVG_SLOPE_CODE) p.slopes = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.slopes) + s);
        return p;
    }
};

// The results of four such sums: activation, slopes, residual (four values, or NULL), store.
template <class O, bool GATED> __device__ __forceinline__ void finish4(const Finish& f, const Place<O>& at, const float* v, const float* u, const float* residual)
{
    const int64_t left = at.left;
    float a[4], d[4];
    const bool want = f.slopeKind != LVG_SLOPE_NONE;
    act4<0, sizeof(O) == 2>(f.act, f.alpha, v, want, a, d);
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
            quad_store(at.slopes, left, f.vec, d);
            quad_store(at.slopes + f.cols, left, f.vec, up);
        }
        quad_store(at.out, left, f.vec, a);
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
    if (f.slopeKind == LVG_SLOPE_F32) quad_store(at.slopes, left, f.vec, d);
    else if (f.slopeKind == LVG_SLOPE_CODE)
    {
        uint8_t* s = reinterpret_cast<uint8_t*>(at.slopes);
        if (f.vec && left >= 4) *reinterpret_cast<uint32_t*>(s) = code;
        else
        {
            #pragma unroll
            for (int i = 0; i < 4; i++) if (i < left) s[i] = (uint8_t)(code >> (8 * i));
        }
    }
    if (residual)
    {
        #pragma unroll
        for (int i = 0; i < 4; i++) a[i] += residual[i];
    }
    quad_store(at.out, left, f.vec, a);
}

} // namespace
