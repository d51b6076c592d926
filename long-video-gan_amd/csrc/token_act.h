// token_act.h -- what the products of token rows do with their sums before they are stored (token_gemm.h, token_stream.hip, token_finish.hip):
//
//   linear   y = clamp(act(sum * scales + b) * gain) + residual                 slope = gain-free derivative of clamp(act(.)), one a value
//   gated    h = gain * act(g) * u,  g = sum * scales + b of the gate half, u of the up half      slopes dh/dg and dh/du
//
// Everything here is float32; the result is rounded once, to the output's type. The slopes are what the gradient multiplies with, kept as the
// forward pass has them (smooth ones; where the derivative takes only the values 0, 1 and alpha, one byte says which): float32 for float32 and
// float16, and for bfloat16 its upper 18 bits, a quarter of bfloat16's rounding error. The gradient's operand
// dy * slope then has ONE rounding to 16 bits that counts, and a sum next to a kink keeps the side it was computed on. Slopes of 16 bits would make the
// error of the weight gradient 1.7 times that of its own rounding; it is 1.4 times with float32 and with 18 bits, which take 44 % less
// memory and 40 us less of a bfloat16 training step of 1640 at 8192 x 2048 -> 8192.
#pragma once
#include "row_common.h"

enum { LVG_SLOPE_NONE = 0, LVG_SLOPE_SMOOTH = 1, LVG_SLOPE_CODE = 2 };

struct Finish
{
    const float* qs;           // [rows] scales of 8-bit rows, or NULL
    const float* ps;           // [cols] (gated: [2 cols]) scales of 8-bit weights, or NULL
    const void*  bias;         // [cols] (gated: [2 cols]) in the output's type, or NULL
    const void*  residual;     // or NULL
    void*        out;
    void*        slopes;       // [rows][cols] (gated: [rows][2 cols]), or NULL; bfloat16: their two bits behind them, a byte for four columns
    int64_t      ldr, ldo;     // elements
    int64_t      rows;
    int64_t      cols;         // of the result; gated: the up half lies cols behind the gate half
    int          act, slopeKind;
    float        alpha, gain, clamp;
    bool         vec;          // the four values of a call may be moved as one vector
    bool         past;         // gated products of whole tiles: results and derivatives are larger than the caches (64 MB and more) and stored past
                               // them, so that the operands stay there (with norm, 8-bit rows and projection around it, 8 bit 8192 x 4096 -> 8192: 807 ->
                               // 786 us; three bfloat16 blocks forward 16384 x 2048 -> 8192: 4305 -> 4264 us, 8192 x 4096 -> 8192: 4064 -> 4094 us;
                               // products with a plain result gain nothing)
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

// Four 16-bit values past the caches (large results of gated products; see Finish::past).
template <class T> __device__ __forceinline__ void quad_past(T* p, const Quad<T>& q)
{
    typedef uint32_t pair __attribute__((ext_vector_type(2)));
    pair w;
    __builtin_memcpy(&w, &q, 8);
    __builtin_nontemporal_store(w, reinterpret_cast<pair*>(p));
}

// The scale of a row of 8-bit values in two factors, the second a power of two: a sum (0, or 2^-18 to 2^48) times the first, times the column's scale,
// times the second neither overflows nor underflows on the way where the result does not, as the product of the two scales can.
struct RowScale
{
    float most, rest;
    __device__ __forceinline__ explicit RowScale(float s)
    {
        const float m = fabsf(s);
        rest = m > 0x1p70f ? 0x1p64f : m < 0x1p-70f ? 0x1p-64f : 1.f;
        most = m > 0x1p70f ? s * 0x1p-64f : m < 0x1p-70f ? s * 0x1p64f : s;
    }
    __device__ __forceinline__ float of(float v, float column) const { return v * most * column * rest; }
};

// Scales whose product alone will do: it stays in range, and loses two bits at most where both are near 2^-64 (the scale of rows of zeros).
__device__ __forceinline__ bool plain_scale(float s) { return fabsf(s) >= 0x1p-64f && fabsf(s) <= 0x1p60f; }

// Four neighbouring sums, row m, columns n .. n + 3 (those below cols): scales and bias. v: sums; gated: v of the gate half, u of the up half.
template <class O, bool GATED> __device__ __forceinline__ void prepare4(const Finish& f, int64_t m, int64_t n, float* v, float* u)
{
    const int64_t left = f.cols - n;
    if (f.qs)
    {
        const RowScale s(f.qs[m]);
        #pragma unroll
        for (int i = 0; i < 4; i++) if (i < left)
        {
            v[i] = s.of(v[i], f.ps[n + i]);
            if (GATED) u[i] = s.of(u[i], f.ps[f.cols + n + i]);
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

// In a derivative's place: no gradient passes here, whatever it is (what a clamp cut, a gate on relu's lower side). A pattern that no arithmetic
// gives, a signalling NaN, and one that 18 bits hold: a derivative that has merely become zero, of either sign, still makes a NaN of an infinite gradient.
constexpr uint32_t kCutBits = 0xffa54000u;
__device__ __forceinline__ float cut_mark() { return __uint_as_float(kCutBits); }

// A row's derivatives, `cols` for each of H halves: float32 or, for bfloat16, the upper 18 bits of the float32 (rounded; zeros, ones and what else
// bfloat16 holds stay exact): 16 of them as an element of type S, the other two in bytes for four columns each.
template <class O> struct Kept            { typedef float S;  static constexpr bool kBits = false; };
template <> struct Kept<bf16_t>           { typedef bf16_t S; static constexpr bool kBits = true; };
__host__ __device__ __forceinline__ int64_t slope_bytes(int64_t rows, int64_t cols, int halves, int kind, int dtype)
{
    if (kind == LVG_SLOPE_CODE) return rows * cols;
    if (kind == LVG_SLOPE_NONE) return 0;
    return dtype == LVG_BF16 ? rows * halves * (2 * cols + (cols + 3) / 4) : rows * halves * cols * 4;
}

// Where four results go: the element of the first in each array.
template <class O, int H> struct Place
{
    typedef typename Kept<O>::S S;
    O*       out;
    S*       slopes;           // (as bytes: LVG_SLOPE_CODE)
    uint8_t* bits;
    int64_t  left;             // columns from it on
    __device__ __forceinline__ Place(const Finish& f, int64_t m, int64_t n)
    {
        left = f.cols - n;
        out = static_cast<O*>(f.out) + m * f.ldo + n;
        slopes = nullptr;
        bits = nullptr;
        if (f.slopeKind == LVG_SLOPE_SMOOTH)
        {
            slopes = static_cast<S*>(f.slopes) + m * H * f.cols + n;
            if (Kept<O>::kBits) bits = reinterpret_cast<uint8_t*>(static_cast<S*>(f.slopes) + f.rows * H * f.cols) + m * H * ((f.cols + 3) / 4) + n / 4;
        }
        else if (f.slopeKind == LVG_SLOPE_CODE) bits = static_cast<uint8_t*>(f.slopes) + m * f.cols + n;
    }
    // `rows` rows on
    __device__ __forceinline__ Place down(const Finish& f, int rows) const
    {
        Place p = *this;
        p.out += rows * f.ldo;
        if (f.slopeKind == LVG_SLOPE_SMOOTH)
        {
            p.slopes += rows * H * f.cols;
            if (Kept<O>::kBits) p.bits += rows * H * ((f.cols + 3) / 4);
        }
        else if (f.slopeKind == LVG_SLOPE_CODE) p.bits += rows * f.cols;
        return p;
    }
    // four derivatives of half h
    __device__ __forceinline__ void keep(const Finish& f, int h, bool vec, const float* d) const
    {
        if constexpr (!Kept<O>::kBits) quad_store(slopes + h * f.cols, left, vec, d);
        else
        {
            S* const to = slopes + h * f.cols;
            Quad<S> q;
            uint32_t w = 0;
            #pragma unroll
            for (int i = 0; i < 4; i++)
            {
                const uint32_t b = __float_as_uint(d[i]) + 0x2000u;
                q.v[i].bits = (uint16_t)(b >> 16);
                w |= (b >> 14 & 3u) << (2 * i);
            }
            if (vec && left >= 4)
            {
                if (f.past) quad_past(to, q);
                else *reinterpret_cast<Quad<S>*>(to) = q;
            }
            else
            {
                #pragma unroll
                for (int i = 0; i < 4; i++) if (i < left) to[i] = q.v[i];
            }
            bits[h * ((f.cols + 3) / 4)] = (uint8_t)w;
        }
    }
};

// The results of four such sums: activation, slopes, residual (four values, or NULL), store.
template <class O, bool GATED> __device__ __forceinline__ void finish4(const Finish& f, const Place<O, GATED ? 2 : 1>& at, const float* v, const float* u, const float* residual)
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
            d[i] = f.act == LVG_ACT_RELU && v[i] <= 0.f ? cut_mark() : d[i] * u[i] * f.gain;        // dh/dg
            a[i] = up[i] * u[i];
        }
        if (want)
        {
            at.keep(f, 0, f.vec, d);
            at.keep(f, 1, f.vec, up);
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
            if (!inside) { a[i] = a[i] > 0.f ? f.clamp : -f.clamp; d[i] = cut_mark(); }
        }
        // 0: no gradient (cut, or relu's lower side), 1: alpha (lrelu's), 2: one
        code |= (uint32_t)(!inside || (f.act == LVG_ACT_RELU && v[i] <= 0.f) ? 0 : (f.act == LVG_ACT_LRELU && !(v[i] > 0.f)) ? 1 : 2) << (8 * i);
    }
    if (f.slopeKind == LVG_SLOPE_SMOOTH) at.keep(f, 0, f.vec, d);
    else if (f.slopeKind == LVG_SLOPE_CODE)
    {
        uint8_t* s = at.bits;
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
