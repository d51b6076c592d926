// rms_norm.hip -- root-mean-square norm of rows with the residual's addition, its gradient, and rows of 8-bit values with one scale each:
//
//   s = x + residual,   r = 1 / sqrt(mean(s^2) + eps),   y = weight * s * r
//   q = y / scale in e4m3,   scale = max |y| of the row / 448               (quantize)
//   ds_in = r (g - n mean(g n)) + ds,   n = s r,   g = weight * dy,   dweight = sum over rows of dy n
//
// (n is about one: the cube of r, which the same gradient can be written with, leaves float32's range from rows of 1e13 and 1e-13 on.)
//
// What a program otherwise spells as add, square, mean, rsqrt, two products, an absolute maximum and a cast: eight passes over the rows where
// one has to read x and residual and write s and y. The gradient reads the sum as it was stored, rounded; two bits a value that the forward pass
// keeps beside it (a third of the rounding's half step up, down, or neither) bring it three times closer to what the norm was taken of, for 3 % of
// the traffic: without them the weight's gradient is 1.5 times as far from the exact one as its own rounding makes it. The sums are float32 and
// their order is fixed.
//
// A row is held in the registers of one wave (up to 2 vectors a lane) or of four (up to 8: 16384 values of 16 bits, 8192 of float32), so each value is
// read once and written once. Wider rows are read again, from L2 where they fit it: twice by the plain norm and by quantisation, three times by the norm
// to 8 bits (mean, maximum, result). The gradient keeps three vectors of a row and of the next one: one wave up to one vector a lane, then four, then
// eight with up to two (8192 values of 16 bits; float32 four, 8192 too); of wider rows a first pass takes the coefficient, a second one
// the columns (4096 rows of 16384 bfloat16 with residual, both directions: 467 us, 1.1 GB at 2.3 TB/s, where 8192 rows of 8192 take 203).
#include "row_common.h"

namespace {

struct NormArgs
{
    const void*  x;
    const void*  residual;     // or NULL
    const void*  weight;       // [width] or NULL
    void*        y;            // T, or e4m3 bytes
    void*        sum;          // T: x + residual, or NULL
    uint16_t*    rest;         // [rows][ceil(width / 8)], 2 bits a value: what the sum's rounding left (16-bit T), or NULL
    float*       rstd;         // [rows] or NULL
    float*       scale;        // [rows], 8-bit results
    int64_t      rows, width, ldx, ldr, ldy;
    float        eps;
    bool         once;         // operands are loaded past the caches
};

struct NormBackArgs
{
    const void*  dy;
    const void*  ds;           // gradient of the sum's other uses, or NULL
    const void*  s;
    const uint16_t* rest;      // as in NormArgs
    const void*  weight;
    const float* rstd;
    void*        dx;
    float*       part;         // [slots][width] or NULL
    float*       coef;         // [rows]: wide rows only
    int64_t      rows, width, lddy, ldds, lds;
    bool         past, once;   // the result is stored past the caches, operands loaded past them
};

template <class T> __device__ __forceinline__ void store_rest(const NormArgs& p, int64_t row, int64_t at, const float* v)
{
    if constexpr (sizeof(T) == 2)
    {
        if (!p.rest || at >= p.width) return;
        uint32_t w = 0;
        #pragma unroll
        for (int i = 0; i < 8; i++) w |= rest_code<T>(v[i]) << (2 * i);
        p.rest[row * ((p.width + 7) / 8) + at / 8] = (uint16_t)w;
    }
}
// the sum's values at `at` (a multiple of the vector), as close as they are kept
template <class T> __device__ __forceinline__ void kept_sum(const NormBackArgs& p, int64_t row, int64_t at, float* v)
{
    if constexpr (sizeof(T) == 2)
    {
        if (!p.rest || at >= p.width) return;
        const uint32_t w = p.rest[row * ((p.width + 7) / 8) + at / 8];
        #pragma unroll
        for (int i = 0; i < 8; i++) v[i] = with_rest<T>(v[i], w >> (2 * i) & 3u);
    }
}

template <int W> __device__ __forceinline__ float row_total(float v, float* lds, int wave)
{
    v = wave_total(v);
    if (W == 1) return v;
    lds[wave] = v;
    __syncthreads();
    float t = 0.f;
    #pragma unroll
    for (int i = 0; i < W; i++) t += lds[i];
    return t;
}

template <int W> __device__ __forceinline__ uint32_t row_largest(uint32_t v, uint32_t* lds, int wave)
{
    v = wave_largest(v);
    if (W == 1) return v;
    lds[wave] = v;
    __syncthreads();
    uint32_t t = 0;
    #pragma unroll
    for (int i = 0; i < W; i++) t = max(t, lds[i]);
    return t;
}

// W waves a row (1: four rows a workgroup of 256), NV vectors a lane; NORM = false: quantisation alone.
template <class T, int W, int NV, bool QUANT, bool NORM>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormArgs p)
{
    constexpr int V = Elem<T>::kVec;
    __shared__ float sums[4];
    __shared__ uint32_t tops[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
    if (W == 1 && row >= p.rows) return;
    const int t = W == 1 ? lane : (int)threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;

    // all loads first: none of them waits behind a store of the sum
    const T* res = NORM && p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    RawRow<T> xr[NV], rr[NV];
    #pragma unroll
    for (int j = 0; j < NV; j++)
    {
        const int64_t at = (int64_t)(j * 64 * W + t) * V;
        xr[j] = load_raw<T>(x + at, p.width - at, p.once);
        if (res) rr[j] = load_raw<T>(res + at, p.width - at, p.once);
    }
    float v[NV][V];
    #pragma unroll
    for (int j = 0; j < NV; j++)
        #pragma unroll
        for (int i = 0; i < V; i++) v[j][i] = row_load(xr[j].v[i]);
    if (NORM)
    {
        if (res)
        {
            #pragma unroll
            for (int j = 0; j < NV; j++)
            {
                const int64_t at = (int64_t)(j * 64 * W + t) * V;
                #pragma unroll
                for (int i = 0; i < V; i++) v[j][i] += row_load(rr[j].v[i]);
                if (p.sum) store_row<T>(static_cast<T*>(p.sum) + row * p.width + at, p.width - at, v[j]);
                store_rest<T>(p, row, at, v[j]);
            }
        }
        float ss = 0.f;
        #pragma unroll
        for (int j = 0; j < NV; j++)
            #pragma unroll
            for (int i = 0; i < V; i++) ss = fmaf(v[j][i], v[j][i], ss);
        ss = row_total<W>(ss, sums, wave);
        const float r = 1.f / sqrtf(ss / (float)p.width + p.eps);
        if (p.rstd && t == 0) p.rstd[row] = r;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t at = (int64_t)(j * 64 * W + t) * V;
            float w[V];
            if (p.weight) load_row<T>(static_cast<const T*>(p.weight) + at, p.width - at, w);
            #pragma unroll
            for (int i = 0; i < V; i++) v[j][i] = p.weight ? v[j][i] * r * w[i] : v[j][i] * r;
        }
    }
    if (QUANT)
    {
        uint32_t top = 0;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t left = p.width - (int64_t)(j * 64 * W + t) * V;
            #pragma unroll
            for (int i = 0; i < V; i++) if (i < left) top = max(top, magnitude(v[j][i]));
        }
        const float scale = row_scale(row_largest<W>(top, tops, wave));
        const Divisor by(scale);
        if (t == 0) p.scale[row] = scale;
        uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.ldy;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t at = (int64_t)(j * 64 * W + t) * V, left = p.width - at;
            uint32_t w[V / 4];
            #pragma unroll
            for (int i = 0; i < V; i += 4) w[i / 4] = pack_e4m3(by.quotient(v[j][i]), by.quotient(v[j][i + 1]), by.quotient(v[j][i + 2]), by.quotient(v[j][i + 3]));
            if (left >= V) __builtin_memcpy(q + at, w, V);
            else
            {
                #pragma unroll
                for (int i = 0; i < V; i++) if (i < left) q[at + i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
            }
        }
    }
    else
    {
        T* y = static_cast<T*>(p.y) + row * p.ldy;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t at = (int64_t)(j * 64 * W + t) * V;
            store_row<T>(y + at, p.width - at, v[j]);
        }
    }
}

// Rows wider than a workgroup's registers: one workgroup a row, the row read again for every statistic.
template <class T, bool QUANT, bool NORM>
__global__ __launch_bounds__(256) void rms_norm_wide_kernel(NormArgs p)
{
    constexpr int V = Elem<T>::kVec;
    __shared__ float sums[4];
    __shared__ uint32_t tops[4];
    const int wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* res = NORM && p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    auto value = [&](int64_t at, float* v)
    {
        load_row<T>(x + at, p.width - at, v);
        if (res)
        {
            float o[V];
            load_row<T>(res + at, p.width - at, o);
            #pragma unroll
            for (int i = 0; i < V; i++) v[i] += o[i];
        }
    };
    float r = 1.f;
    if (NORM)
    {
        float ss = 0.f;
        for (int64_t at = (int64_t)threadIdx.x * V; at < p.width; at += 256 * V)
        {
            float v[V];
            value(at, v);
            #pragma unroll
            for (int i = 0; i < V; i++) ss = fmaf(v[i], v[i], ss);
            if (res && p.sum) store_row<T>(static_cast<T*>(p.sum) + row * p.width + at, p.width - at, v);
            if (res) store_rest<T>(p, row, at, v);
        }
        ss = row_total<4>(ss, sums, wave);
        r = 1.f / sqrtf(ss / (float)p.width + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = r;
    }
    auto result = [&](int64_t at, float* v)
    {
        value(at, v);
        if (!NORM) return;
        float w[V];
        if (p.weight) load_row<T>(static_cast<const T*>(p.weight) + at, p.width - at, w);
        #pragma unroll
        for (int i = 0; i < V; i++) v[i] = p.weight ? v[i] * r * w[i] : v[i] * r;
    };
    float scale = 1.f;
    if (QUANT)
    {
        uint32_t top = 0;
        for (int64_t at = (int64_t)threadIdx.x * V; at < p.width; at += 256 * V)
        {
            float v[V];
            result(at, v);
            #pragma unroll
            for (int i = 0; i < V; i++) if (at + i < p.width) top = max(top, magnitude(v[i]));
        }
        scale = row_scale(row_largest<4>(top, tops, wave));
        if (threadIdx.x == 0) p.scale[row] = scale;
    }
    const Divisor by(scale);
    for (int64_t at = (int64_t)threadIdx.x * V; at < p.width; at += 256 * V)
    {
        float v[V];
        result(at, v);
        if (QUANT)
        {
            uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.ldy + at;
            #pragma unroll
            for (int i = 0; i < V; i += 4)
            {
                const uint32_t w = pack_e4m3(by.quotient(v[i]), by.quotient(v[i + 1]), by.quotient(v[i + 2]), by.quotient(v[i + 3]));
                #pragma unroll
                for (int k = 0; k < 4; k++) if (at + i + k < p.width) q[i + k] = (uint8_t)(w >> (8 * k));
            }
        }
        else store_row<T>(static_cast<T*>(p.y) + row * p.ldy + at, p.width - at, v);
    }
}

// Gradient: a workgroup takes rows blockIdx.x, + gridDim.x, ... (W == 1: its four waves a row each) and keeps the weight's gradient of its
// rows in registers; they go to part[blockIdx.x][width] (W == 1: the four waves' sums meet in LDS in wave order). The next row's three vectors
// are asked for before this one's are used, so that memory does not wait for the row's reduction.
template <class T, int W, int NV>
__global__ __launch_bounds__(W == 8 ? 512 : 256) void rms_norm_back_kernel(NormBackArgs p)
{
    constexpr int V = Elem<T>::kVec;
    static_assert(NV <= 4 && (W != 1 || NV == 1), "two rows fit the registers; one wave a row takes one vector a lane");
    __shared__ float sums[2][W == 1 ? 4 : W];
    __shared__ float cols[W == 1 ? 64 * V : 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int t = W == 1 ? lane : (int)threadIdx.x;
    float dw[NV][V], w[NV][V];
    #pragma unroll
    for (int j = 0; j < NV; j++)
    {
        const int64_t at = (int64_t)(j * 64 * W + t) * V;
        #pragma unroll
        for (int i = 0; i < V; i++) { dw[j][i] = 0.f; w[j][i] = 1.f; }
        if (p.weight) load_row<T>(static_cast<const T*>(p.weight) + at, p.width - at, w[j]);
    }
    struct Row { RawRow<T> g[NV], s[NV], d[NV]; uint32_t rest[NV]; float r; };
    auto load = [&](Row& x, int64_t row)
    {
        const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
        const T* s = static_cast<const T*>(p.s) + row * p.lds;
        const T* ds = static_cast<const T*>(p.ds) + row * p.ldds;
        x.r = p.rstd[row];
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t at = (int64_t)(j * 64 * W + t) * V;
            x.g[j] = load_raw<T>(dy + at, p.width - at, p.once);
            x.s[j] = load_raw<T>(s + at, p.width - at, p.once);
            if (p.ds) x.d[j] = load_raw<T>(ds + at, p.width - at, p.once);
            x.rest[j] = sizeof(T) == 2 && p.rest && at < p.width ? p.rest[row * ((p.width + 7) / 8) + at / 8] : 0x5555u;     // (0x5555: nothing left)
        }
    };
    auto sum_at = [](const Row& x, int j, int i)
    {
        const float s = row_load(x.s[j].v[i]);
        if constexpr (sizeof(T) == 2) return with_rest<T>(s, x.rest[j] >> (2 * i) & 3u);
        else return s;
    };
    const int64_t step = (int64_t)gridDim.x * (W == 1 ? 4 : 1);
    int turn = 0;
    int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
    Row now, next;
    if (row < p.rows) load(now, row);
    for (; row < p.rows; row += step, turn ^= 1)
    {
        if (row + step < p.rows) load(next, row + step);
        const float r = now.r;
        float dot = 0.f;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            #pragma unroll
            for (int i = 0; i < V; i++)
            {
                const float g = row_load(now.g[j].v[i]), n = sum_at(now, j, i) * r;
                dw[j][i] = fmaf(g, n, dw[j][i]);
                dot = fmaf(g * w[j][i], n, dot);
            }
        }
        dot = row_total<W>(dot, sums[turn], wave);         // (two sets: a wave may reach the next row's while another still reads this one's)
        const float c = dot / (float)p.width;
        #pragma unroll
        for (int j = 0; j < NV; j++)
        {
            const int64_t at = (int64_t)(j * 64 * W + t) * V;
            float v[V];
            #pragma unroll
            for (int i = 0; i < V; i++)
            {
                v[i] = fmaf(sum_at(now, j, i) * r, -c, row_load(now.g[j].v[i]) * w[j][i]) * r;
                if (p.ds) v[i] += row_load(now.d[j].v[i]);
            }
            store_row<T>(static_cast<T*>(p.dx) + row * p.width + at, p.width - at, v, p.past);
        }
        now = next;
    }
    if (!p.part) return;
    float* out = p.part + (int64_t)blockIdx.x * p.width;
    if (W == 1)
    {
        for (int k = 0; k < 4; k++)         // the waves add in turn
        {
            if (wave == k)
            {
                #pragma unroll
                for (int i = 0; i < V; i++) cols[lane * V + i] = k == 0 ? dw[0][i] : cols[lane * V + i] + dw[0][i];
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 64 * V; i += 256) if (i < p.width) out[i] = cols[i];
        return;
    }
    #pragma unroll
    for (int j = 0; j < NV; j++)
    {
        const int64_t at = (int64_t)(j * 64 * W + t) * V;
        #pragma unroll
        for (int i = 0; i < V; i++) if (at + i < p.width) out[at + i] = dw[j][i];
    }
}

// Wide rows: the row's coefficient first, then columns.
template <class T>
__global__ __launch_bounds__(256) void rms_norm_back_coef_kernel(NormBackArgs p)
{
    constexpr int V = Elem<T>::kVec;
    __shared__ float sums[4];
    const int64_t row = blockIdx.x;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const T* s = static_cast<const T*>(p.s) + row * p.lds;
    const float r = p.rstd[row];
    float dot = 0.f;
    for (int64_t at = (int64_t)threadIdx.x * V; at < p.width; at += 256 * V)
    {
        float g[V], sv[V], w[V];
        load_row<T>(dy + at, p.width - at, g);
        load_row<T>(s + at, p.width - at, sv);
        kept_sum<T>(p, row, at, sv);
        if (p.weight) load_row<T>(static_cast<const T*>(p.weight) + at, p.width - at, w);
        #pragma unroll
        for (int i = 0; i < V; i++) dot = fmaf(p.weight ? g[i] * w[i] : g[i], sv[i] * r, dot);
    }
    dot = row_total<4>(dot, sums, threadIdx.x >> 6);
    if (threadIdx.x == 0) p.coef[row] = dot / (float)p.width;
}

template <class T>
__global__ __launch_bounds__(256) void rms_norm_back_wide_kernel(NormBackArgs p)
{
    constexpr int V = Elem<T>::kVec;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, left = p.width - at;
    if (left <= 0) return;
    float dw[V], w[V];
    #pragma unroll
    for (int i = 0; i < V; i++) { dw[i] = 0.f; w[i] = 1.f; }
    if (p.weight) load_row<T>(static_cast<const T*>(p.weight) + at, left, w);
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y)
    {
        float g[V], sv[V], d[V];
        load_row<T>(static_cast<const T*>(p.dy) + row * p.lddy + at, left, g);
        load_row<T>(static_cast<const T*>(p.s) + row * p.lds + at, left, sv);
        kept_sum<T>(p, row, at, sv);
        if (p.ds) load_row<T>(static_cast<const T*>(p.ds) + row * p.ldds + at, left, d);
        const float r = p.rstd[row], c = p.coef[row];
        #pragma unroll
        for (int i = 0; i < V; i++)
        {
            const float n = sv[i] * r;
            dw[i] = fmaf(g[i], n, dw[i]);
            g[i] = fmaf(n, -c, g[i] * w[i]) * r + (p.ds ? d[i] : 0.f);
        }
        store_row<T>(static_cast<T*>(p.dx) + row * p.width + at, left, g);
    }
    if (p.part)
    {
        #pragma unroll
        for (int i = 0; i < V; i++) if (i < left) p.part[(int64_t)blockIdx.y * p.width + at + i] = dw[i];
    }
}

// out[c] = sum over the slots of part[slot][c]: 32 columns a workgroup, its 8 rows of threads take every eighth slot and add in their order.
template <class T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* part, T* out, int slots, int64_t width, float gain)
{
    __shared__ float sums[8][32];
    const int group = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.f;
    if (c < width)
    {
        #pragma unroll 8
        for (int s = group; s < slots; s += 8) v += part[(int64_t)s * width + c];
    }
    sums[group][lane] = v;
    __syncthreads();
    if (group != 0 || c >= width) return;
    #pragma unroll
    for (int g = 1; g < 8; g++) v += sums[g][lane];
    out[c] = from_acc<T>(v * gain);
}

int esize(int dtype) { return dtype == LVG_F32 ? 4 : 2; }
bool row_type(int dtype) { return dtype == LVG_F32 || dtype == LVG_F16 || dtype == LVG_BF16; }

// Waves a row and vectors a lane: one wave as long as a lane holds the row in two vectors, then a workgroup of four (16384 rows of 4096 bfloat16
// with residual: 138 us as one wave of 8 vectors a lane, 105 us as four of 2: more waves fit a compute unit).
struct Plan { int waves, vecs; };
Plan plan(int64_t width, int dtype)
{
    const int64_t vecs = lvg_ceil_div(width, 16 / esize(dtype));
    for (int nv : {1, 2}) if (vecs <= 64 * nv) return {1, nv};
    for (int nv : {1, 2, 4, 8}) if (vecs <= 256 * nv) return {4, nv};
    return {0, 0};
}

// Matrices of 64 MB and more, in aligned rows: operands are loaded past the caches, each value is read by one lane, once, and leaves them to what is
// written and read next (four norms with residual in a row, inputs and results in turn, bfloat16: 16384 x 4096 325 us, and 384 with plain loads; 32768 x
// 1024 166 and 169; a norm and the sum of its two results, 16384 x 4096: 137 and 159). Results of the forward pass are stored through the caches, where
// the next operator finds part of them (past them: 357, 187 and 152 us). The gradient is stored past them: four such steps with gradients, 32768 x 1024,
// 429 us, and 441 through the caches; 16384 x 4096 670 and 670; 65536 x 1024 807 and 822.
constexpr int64_t kLarge = (int64_t)64 << 20;
bool aligned_rows(const void* p, int64_t stride, int dtype) { return !p || (lvg_aligned16(p) && stride * esize(dtype) % 16 == 0); }
bool large(int64_t rows, int64_t width, int arrays, int dtype) { return arrays * rows * width * esize(dtype) >= kLarge; }

// Rows of one launch: a grid holds fewer than 2^32 threads.
constexpr int64_t kLaunchRows = (int64_t)1 << 23;

template <class T, bool QUANT, bool NORM> void launch_norm_rows(const NormArgs& a, const Plan& k, hipStream_t s)
{
    const dim3 block(256), grid((unsigned)(k.waves == 1 ? lvg_ceil_div(a.rows, 4) : a.rows));
    #define LVG_ROW(W, NV) if (k.waves == W && k.vecs == NV) { hipLaunchKernelGGL((rms_norm_kernel<T, W, NV, QUANT, NORM>), grid, block, 0, s, a); return; }
    LVG_ROW(1, 1) LVG_ROW(1, 2) LVG_ROW(4, 1) LVG_ROW(4, 2) LVG_ROW(4, 4) LVG_ROW(4, 8)
    #undef LVG_ROW
    hipLaunchKernelGGL((rms_norm_wide_kernel<T, QUANT, NORM>), grid, block, 0, s, a);
}

template <class T, bool QUANT, bool NORM> void launch_norm(const NormArgs& a, const Plan& k, hipStream_t s)
{
    for (int64_t r = 0; r < a.rows; r += kLaunchRows)
    {
        NormArgs b = a;
        b.rows = std::min(kLaunchRows, a.rows - r);
        b.x = static_cast<const T*>(a.x) + r * a.ldx;
        if (a.residual) b.residual = static_cast<const T*>(a.residual) + r * a.ldr;
        b.y = static_cast<char*>(a.y) + r * a.ldy * (QUANT ? 1 : (int64_t)sizeof(T));
        if (a.sum) b.sum = static_cast<T*>(a.sum) + r * a.width;
        if (a.rest) b.rest = a.rest + r * ((a.width + 7) / 8);
        if (a.rstd) b.rstd = a.rstd + r;
        if (a.scale) b.scale = a.scale + r;
        launch_norm_rows<T, QUANT, NORM>(b, k, s);
    }
}

// The gradient keeps more of a row (its three vectors twice and the weight's gradient): a wave a row only as long as a lane holds it in one vector.
Plan back_plan(int64_t width, int dtype)
{
    const int64_t vecs = lvg_ceil_div(width, 16 / esize(dtype));
    if (vecs <= 64) return {1, 1};
    if (vecs <= 256) return {4, 1};
    for (int nv : {1, 2, 4}) if (vecs <= 512 * nv && (nv < 4 || dtype == LVG_F32)) return {8, nv};
    return {0, 0};
}

template <class T> void launch_back(const NormBackArgs& a, const Plan& k, int slots, hipStream_t s)
{
    const dim3 block(256), grid((unsigned)slots);
    #define LVG_ROW(W, NV) if (k.waves == W && k.vecs == NV) { hipLaunchKernelGGL((rms_norm_back_kernel<T, W, NV>), grid, dim3(W == 8 ? 512 : 256), 0, s, a); return; }
    LVG_ROW(1, 1) LVG_ROW(4, 1) LVG_ROW(8, 1) LVG_ROW(8, 2)
    if constexpr (sizeof(T) == 4) { LVG_ROW(8, 4) }
    #undef LVG_ROW
    hipLaunchKernelGGL(rms_norm_back_coef_kernel<T>, dim3((unsigned)a.rows), block, 0, s, a);
    hipLaunchKernelGGL(rms_norm_back_wide_kernel<T>, dim3((unsigned)lvg_ceil_div(a.width, 256 * Elem<T>::kVec), (unsigned)slots), block, 0, s, a);
}

bool rows_ok(int64_t rows, int64_t width) { return rows >= 0 && rows <= 0x7fffffff && width >= 1 && width <= ((int64_t)1 << 40); }

int back_slots(int64_t rows, int64_t width, int dtype)
{
    const Plan k = back_plan(width, dtype);
    // two or four workgroups for each of the 256 compute units: what they write of the weight's gradient is read again
    if (k.waves == 1) return (int)std::min<int64_t>(1024, lvg_ceil_div(rows, 4));
    if (k.waves) return (int)std::min<int64_t>(k.waves == 4 ? 1024 : 512, rows);
    return (int)std::min<int64_t>(64, rows);
}

} // namespace

extern "C" int lvg_rms_norm(const void* x, const void* residual, const void* weight, void* y, void* sum, void* rest, float* rstd, float* scale,
                            int64_t rows, int64_t width, int64_t x_stride, int64_t residual_stride, float eps, int dtype, int quantize, void* stream)
{
    LVG_REQUIRE(row_type(dtype), "lvg_rms_norm: float32 / float16 / bfloat16 only (dtype %d)", dtype);
    LVG_REQUIRE(rows_ok(rows, width), "lvg_rms_norm: bad size (%lld rows of %lld)", (long long)rows, (long long)width);
    if (rows == 0) return LVG_OK;
    LVG_REQUIRE(x && y && (!quantize || scale) && (!sum || residual) && (!rest || sum), "lvg_rms_norm: missing pointer");
    LVG_REQUIRE(x_stride >= 0 && residual_stride >= 0, "lvg_rms_norm: negative row stride");
    LVG_REQUIRE(eps >= 0.f, "lvg_rms_norm: eps must not be negative");
    NormArgs a = {x, residual, weight, y, sum, dtype == LVG_F32 ? nullptr : static_cast<uint16_t*>(rest), rstd, scale, rows, width, x_stride, residual_stride, width, eps, false};
    a.once = large(rows, width, residual ? 2 : 1, dtype) && aligned_rows(x, x_stride, dtype) && aligned_rows(residual, residual_stride, dtype);
    const Plan k = plan(width, dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    #define LVG_TYPE(T) { if (quantize) launch_norm<T, true, true>(a, k, s); else launch_norm<T, false, true>(a, k, s); }
    if (dtype == LVG_F32) LVG_TYPE(float) else if (dtype == LVG_F16) LVG_TYPE(f16_t) else LVG_TYPE(bf16_t)
    #undef LVG_TYPE
    return lvg_check_launch("lvg_rms_norm");
}

extern "C" int lvg_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t width, int64_t x_stride, int dtype, void* stream)
{
    LVG_REQUIRE(row_type(dtype), "lvg_quantize_rows: float32 / float16 / bfloat16 only (dtype %d)", dtype);
    LVG_REQUIRE(rows_ok(rows, width), "lvg_quantize_rows: bad size (%lld rows of %lld)", (long long)rows, (long long)width);
    if (rows == 0) return LVG_OK;
    LVG_REQUIRE(x && q && scale && x_stride >= 0, "lvg_quantize_rows: missing pointer or negative row stride");
    NormArgs a = {x, nullptr, nullptr, q, nullptr, nullptr, nullptr, scale, rows, width, x_stride, 0, width, 0.f, large(rows, width, 1, dtype) && aligned_rows(x, x_stride, dtype)};
    const Plan k = plan(width, dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == LVG_F32) launch_norm<float, true, false>(a, k, s);
    else if (dtype == LVG_F16) launch_norm<f16_t, true, false>(a, k, s);
    else launch_norm<bf16_t, true, false>(a, k, s);
    return lvg_check_launch("lvg_quantize_rows");
}

extern "C" int64_t lvg_rms_norm_backward_work(int64_t rows, int64_t width, int weight, int dtype)
{
    if (!row_type(dtype) || !rows_ok(rows, width)) return LVG_ERR_INVALID;
    if (rows == 0) return 0;
    return (back_plan(width, dtype).waves ? 0 : (rows + 3) / 4 * 16) + (weight ? (int64_t)back_slots(rows, width, dtype) * width * 4 : 0);
}

extern "C" int lvg_rms_norm_backward(const void* dy, const void* dsum, const void* s_in, const void* rest, const void* weight, const float* rstd, void* dx, void* dw,
                                     void* work, int64_t work_size, int64_t rows, int64_t width, int64_t dy_stride, int64_t dsum_stride, int64_t s_stride,
                                     int dtype, void* stream)
{
    LVG_REQUIRE(row_type(dtype), "lvg_rms_norm_backward: float32 / float16 / bfloat16 only (dtype %d)", dtype);
    LVG_REQUIRE(rows_ok(rows, width), "lvg_rms_norm_backward: bad size (%lld rows of %lld)", (long long)rows, (long long)width);
    if (rows == 0)
    {
        if (dw) row_column_sum(nullptr, dw, 0, width, 0.f, dtype, static_cast<hipStream_t>(stream));
        return lvg_check_launch("lvg_rms_norm_backward");
    }
    const Plan k = back_plan(width, dtype);
    const int64_t need = lvg_rms_norm_backward_work(rows, width, dw != nullptr, dtype);
    LVG_REQUIRE(dy && s_in && rstd && dx, "lvg_rms_norm_backward: missing pointer");
    LVG_REQUIRE(need == 0 || (work && lvg_aligned16(work) && work_size >= need), "lvg_rms_norm_backward: the workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
    LVG_REQUIRE(k.waves || rows <= kLaunchRows, "lvg_rms_norm_backward: more than %lld rows of %lld values", (long long)kLaunchRows, (long long)width);
    LVG_REQUIRE(dy_stride >= 0 && dsum_stride >= 0 && s_stride >= 0, "lvg_rms_norm_backward: negative row stride");
    const int slots = back_slots(rows, width, dtype);
    float* const coef = k.waves ? nullptr : static_cast<float*>(work);
    float* const part = dw ? static_cast<float*>(work) + (k.waves ? 0 : (rows + 3) / 4 * 4) : nullptr;
    NormBackArgs a = {dy, dsum, s_in, dtype == LVG_F32 ? nullptr : static_cast<const uint16_t*>(rest), weight, rstd, dx, part, coef, rows, width, dy_stride, dsum_stride, s_stride, false, false};
    a.past = large(rows, width, 1, dtype) && aligned_rows(dx, width, dtype);
    a.once = large(rows, width, 2, dtype) && aligned_rows(dy, dy_stride, dtype) && aligned_rows(dsum, dsum_stride, dtype) && aligned_rows(s_in, s_stride, dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == LVG_F32) launch_back<float>(a, k, slots, s);
    else if (dtype == LVG_F16) launch_back<f16_t>(a, k, slots, s);
    else launch_back<bf16_t>(a, k, slots, s);
    if (dw) row_column_sum(part, dw, slots, width, 1.f, dtype, s);
    return lvg_check_launch("lvg_rms_norm_backward");
}

void row_column_sum(const float* part, void* out, int slots, int64_t width, float gain, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)lvg_ceil_div(width, 32)), block(256);
    if (dtype == LVG_F32) hipLaunchKernelGGL(column_sum_kernel<float>, grid, block, 0, s, part, static_cast<float*>(out), slots, width, gain);
    else if (dtype == LVG_F16) hipLaunchKernelGGL(column_sum_kernel<f16_t>, grid, block, 0, s, part, static_cast<f16_t*>(out), slots, width, gain);
    else hipLaunchKernelGGL(column_sum_kernel<bf16_t>, grid, block, 0, s, part, static_cast<bf16_t*>(out), slots, width, gain);
}
