// token_stream.hip -- forward products of a few token rows (at most 32: decoded tokens, single latents), where the weight's way from memory is all
// that counts. The weight is read once, straight into the matrix instruction's registers: no LDS, no barrier before the sums are joined.
//
// A workgroup of 8 waves owns 16 columns of the result (gated: of both halves) for up to 16 token rows, or 32 weight rows' columns for up to 32
// token rows: the token rows come from L2 for every workgroup, and as many weight rows as token rows keep that traffic no larger than the weight's. Its
// waves take the summed index's 256-byte spans in turn, so that each has 4 loads of 64 bytes a weight row in flight for this span and 4 for its
// next. The eight partial sums meet in LDS and are added in wave order. Few columns and a long summed index: the spans are split over workgroups, token_finish.hip adds the parts.
// Rows may start anywhere (unaligned 16-byte loads); the last, partial span is loaded under masks.
#include "token_stream.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 8;

// 16 x 16 += 16-byte fragments (e4m3: two of them)
template <class T> __device__ __forceinline__ f32x4 small_product(const uint4& a, const uint4& b, f32x4 c);
template <> __device__ __forceinline__ f32x4 small_product<bf16_t>(const uint4& a, const uint4& b, f32x4 c)
{
    b16x8 av, bv;
    __builtin_memcpy(&av, &a, 16);
    __builtin_memcpy(&bv, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 small_product<f16_t>(const uint4& a, const uint4& b, f32x4 c)
{
    h16x8 av, bv;
    __builtin_memcpy(&av, &a, 16);
    __builtin_memcpy(&bv, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(av, bv, c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 small_product<float>(const uint4& a, const uint4& b, f32x4 c)
{
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 small_product8(const uint4& a0, const uint4& a1, const uint4& b0, const uint4& b1, f32x4 c)
{
    i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
    i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

// 16 bytes of a row of `bytes` bytes, from byte `at` on; zeros past the end.
template <class T> __device__ __forceinline__ uint4 row_bytes(const char* row, int64_t at, int64_t bytes)
{
    uint4 r = make_uint4(0, 0, 0, 0);
    constexpr int kE = 16 / (int)sizeof(T);
    const int64_t n = (bytes - at) / (int64_t)sizeof(T);
    if (n >= kE) __builtin_memcpy(&r, row + at, 16);
    else if (n > 0)
    {
        T e[kE];
        #pragma unroll
        for (int j = 0; j < kE; j++)
        {
            if (j < n) e[j] = reinterpret_cast<const T*>(row + at)[j];
            else __builtin_memset(&e[j], 0, sizeof(T));
        }
        __builtin_memcpy(&r, e, 16);
    }
    return r;
}

// GC groups of 16 columns, GR of 16 rows
template <class T, class O, int GC, int GR, bool GATED>
__global__ __launch_bounds__(kWaves * 64) void token_stream_kernel(StreamArgs a)
{
    constexpr int kH = GATED ? 2 : 1;
    __shared__ float4 sums[kWaves][kH][GC][GR][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * 16 * GC;
    const int first = (int)blockIdx.y * a.spansPerSplit, last = min(first + a.spansPerSplit, a.spans);
    const int64_t in = (lane >> 4) * 16;                   // this lane's bytes of a 64-byte piece

    const char* w[kH][GC];
    const char* x[GR];
    bool has[GR];
    #pragma unroll
    for (int g = 0; g < GC; g++)
    {
        int64_t n = n0 + g * 16 + (lane & 15);
        if (n >= a.cols) n = a.cols - 1;                   // past the end: the last one again, its products are not stored
        #pragma unroll
        for (int h = 0; h < kH; h++) w[h][g] = static_cast<const char*>(a.w) + (n + h * a.cols) * a.ldw;
    }
    #pragma unroll
    for (int g = 0; g < GR; g++)
    {
        const int m = g * 16 + (lane & 15);
        has[g] = m < a.rows;
        x[g] = static_cast<const char*>(a.x) + (has[g] ? m : 0) * a.ldx;
    }

    f32x4 acc[kH][GC][GR];                                  // [half][columns][rows]
    #pragma unroll
    for (int h = 0; h < kH; h++)
        #pragma unroll
        for (int g = 0; g < GC; g++)
            #pragma unroll
            for (int k = 0; k < GR; k++) acc[h][g][k] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Span { uint4 w[kH][GC][4], x[GR][4]; };
    auto load = [&](Span& s, int span)
    {
        const int64_t at = (int64_t)span * 256 + in;
        if ((int64_t)(span + 1) * 256 <= a.bytes)
        {
            #pragma unroll
            for (int j = 0; j < 4; j++)
            {
                #pragma unroll
                for (int g = 0; g < GC; g++)
                    #pragma unroll
                    for (int h = 0; h < kH; h++) __builtin_memcpy(&s.w[h][g][j], w[h][g] + at + j * 64, 16);
                #pragma unroll
                for (int g = 0; g < GR; g++)
                {
                    s.x[g][j] = make_uint4(0, 0, 0, 0);
                    if (has[g]) __builtin_memcpy(&s.x[g][j], x[g] + at + j * 64, 16);
                }
            }
        }
        else
        {
            #pragma unroll
            for (int j = 0; j < 4; j++)
            {
                #pragma unroll
                for (int g = 0; g < GC; g++)
                    #pragma unroll
                    for (int h = 0; h < kH; h++) s.w[h][g][j] = row_bytes<T>(w[h][g], at + j * 64, a.bytes);
                #pragma unroll
                for (int g = 0; g < GR; g++)
                {
                    s.x[g][j] = make_uint4(0, 0, 0, 0);
                    if (has[g]) s.x[g][j] = row_bytes<T>(x[g], at + j * 64, a.bytes);
                }
            }
        }
    };
    auto multiply = [&](const Span& s)
    {
        #pragma unroll
        for (int h = 0; h < kH; h++)
            #pragma unroll
            for (int g = 0; g < GC; g++)
                #pragma unroll
                for (int k = 0; k < GR; k++)
                {
                    if constexpr (sizeof(T) == 1)
                    {
                        acc[h][g][k] = small_product8(s.w[h][g][0], s.w[h][g][1], s.x[k][0], s.x[k][1], acc[h][g][k]);
                        acc[h][g][k] = small_product8(s.w[h][g][2], s.w[h][g][3], s.x[k][2], s.x[k][3], acc[h][g][k]);
                    }
                    else
                    {
                        #pragma unroll
                        for (int j = 0; j < 4; j++) acc[h][g][k] = small_product<T>(s.w[h][g][j], s.x[k][j], acc[h][g][k]);
                    }
                }
    };
    Span one, two;
    int span = first + wave;
    if (span < last) load(one, span);
    while (span < last)
    {
        if (span + kWaves < last) load(two, span + kWaves);
        multiply(one);
        span += kWaves;
        if (span >= last) break;
        if (span + kWaves < last) load(one, span + kWaves);
        multiply(two);
        span += kWaves;
    }

    #pragma unroll
    for (int h = 0; h < kH; h++)
        #pragma unroll
        for (int g = 0; g < GC; g++)
            #pragma unroll
            for (int k = 0; k < GR; k++) sums[wave][h][g][k][lane] = make_float4(acc[h][g][k][0], acc[h][g][k][1], acc[h][g][k][2], acc[h][g][k][3]);
    __syncthreads();
    if (wave >= GC * GR) return;
    // a lane holds row lane & 15, columns 4 (lane / 16) .. + 3 of its block
    const int g = wave / GR, k = wave % GR;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
    #pragma unroll
    for (int i = 0; i < kWaves; i++)
    {
        const float4 s = sums[i][0][g][k][lane];
        v[0] += s.x; v[1] += s.y; v[2] += s.z; v[3] += s.w;
        if (GATED)
        {
            const float4 t = sums[i][kH - 1][g][k][lane];
            u[0] += t.x; u[1] += t.y; u[2] += t.z; u[3] += t.w;
        }
    }
    const int64_t m = k * 16 + (lane & 15), n = n0 + g * 16 + (lane >> 4) * 4;
    if (m >= a.rows || n >= a.cols) return;
    if (a.part)
    {
        float* at = a.part + ((int64_t)blockIdx.y * a.rows + m) * a.ldpart + n;
        *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
        if (GATED) *reinterpret_cast<float4*>(at + a.ldpart / 2) = make_float4(u[0], u[1], u[2], u[3]);
        return;
    }
    prepare4<O, GATED>(a.fin, m, n, v, u);
    float r[4];
    residual4<O>(a.fin, m, n, r);
    finish4<O, GATED>(a.fin, Place<O, GATED ? 2 : 1>(a.fin, m, n), v, u, r);
}

template <class T, class O> int launch(const StreamArgs& a, bool gated, int splits, hipStream_t s)
{
    const bool many = a.rows > 16;
    if (a.cols > kStreamCols) { lvg_set_error("token product of a few rows: %lld columns", (long long)a.cols); return LVG_ERR_INVALID; }
    const dim3 grid((unsigned)lvg_ceil_div(a.cols, many && !gated ? 32 : 16), (unsigned)splits), block(kWaves * 64);
    if (!many)
    {
        if (gated) hipLaunchKernelGGL((token_stream_kernel<T, O, 1, 1, true>), grid, block, 0, s, a);
        else       hipLaunchKernelGGL((token_stream_kernel<T, O, 1, 1, false>), grid, block, 0, s, a);
    }
    else
    {
        if (gated) hipLaunchKernelGGL((token_stream_kernel<T, O, 1, 2, true>), grid, block, 0, s, a);
        else       hipLaunchKernelGGL((token_stream_kernel<T, O, 2, 2, false>), grid, block, 0, s, a);
    }
    return lvg_check_launch("token product of a few rows");
}

} // namespace

// Two workgroups for each of the 256 compute units, but at least two spans a wave.
int token_stream_splits(int64_t rows, int64_t cols, int64_t bytes, bool gated)
{
    const int64_t blocks = lvg_ceil_div(cols, rows > 16 && !gated ? 32 : 16), spans = lvg_ceil_div(bytes, 256);
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(512 / blocks, spans / (2 * kWaves)));
    return want <= 1 ? 1 : (int)lvg_ceil_div(spans, lvg_ceil_div(spans, want));
}

int token_stream_launch(const StreamArgs& a, int dtype, int out_dtype, bool gated, int splits, hipStream_t s)
{
    if (dtype == LVG_F32) return launch<float, float>(a, gated, splits, s);
    if (dtype == LVG_F16) return launch<f16_t, f16_t>(a, gated, splits, s);
    if (dtype == LVG_BF16) return launch<bf16_t, bf16_t>(a, gated, splits, s);
    return out_dtype == LVG_F16 ? launch<e4m3_t, f16_t>(a, gated, splits, s) : launch<e4m3_t, bf16_t>(a, gated, splits, s);
}
