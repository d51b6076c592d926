// token_finish.hip -- the products of token rows as entry points: how a product is laid out over the chip, the pass that adds the parts of a
// split product, and the element-wise step between a result's gradient and the two products of the backward pass:
//
//   dz[m][n] = dy[m][n] * slope[m][n] * gain,   db[n] = sum over rows of dz
//
// (gated: dy meets both slopes, dz has the gate's columns and then the up half's). One pass: dy and the slopes are read once, dz is written once
// for both products, the column sums stay in registers until a workgroup's rows are done.
#include "token_gemm.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Adding the parts of a split product, in their order.

template <class O, bool GATED>
__global__ __launch_bounds__(256) void token_finish_kernel(const float* part, int splits, int64_t ldpart, Finish f)
{
    const int64_t quads = (f.cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= f.rows * quads) return;
    const int64_t m = i / quads, n = (i - m * quads) * 4;
    const float* at = part + m * ldpart + n;
    const int64_t step = f.rows * ldpart;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
    #pragma unroll 4
    for (int s = 0; s < splits; s++, at += step)
    {
        const float4 a = *reinterpret_cast<const float4*>(at);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        if (GATED)
        {
            const float4 b = *reinterpret_cast<const float4*>(at + ldpart / 2);
            u[0] += b.x; u[1] += b.y; u[2] += b.z; u[3] += b.w;
        }
    }
    prepare4<O, GATED>(f, m, n, v, u);
    float r[4];
    residual4<O>(f, m, n, r);
    finish4<O, GATED>(f, Place<O, GATED ? 2 : 1>(f, m, n), v, u, r);
}

int launch_finish(const float* part, int splits, int64_t ldpart, const Finish& f, int out_dtype, bool gated, hipStream_t s)
{
    const int64_t threads = f.rows * ((f.cols + 3) / 4);
    const dim3 grid((unsigned)lvg_ceil_div(threads, 256)), block(256);
    #define LVG_FINISH(O) { \
        if (gated) hipLaunchKernelGGL((token_finish_kernel<O, true>), grid, block, 0, s, part, splits, ldpart, f); \
        else       hipLaunchKernelGGL((token_finish_kernel<O, false>), grid, block, 0, s, part, splits, ldpart, f); }
    if (out_dtype == LVG_F32) LVG_FINISH(float) else if (out_dtype == LVG_F16) LVG_FINISH(f16_t) else LVG_FINISH(bf16_t)
    #undef LVG_FINISH
    return lvg_check_launch("token product, adding its parts");
}

// ---------------------------------------------------------------------------------------------------------------------
// dy, slopes -> dz and column sums.

struct SlopeArgs
{
    const void* dy;
    const void* slopes;        // [rows][halves * cols] (and their bits), or NULL
    void*       dz;            // or NULL: column sums alone
    float*      part;          // [gridDim.y][halves * cols], or NULL
    int64_t     rows, cols, lddy, lddz;
    int         kind;
    int         lanes;         // threads of a workgroup along the columns, a power of two
    float       alpha, gain;
    bool        once;          // large and aligned: dy, slopes and dz go past the caches
};

// A thread owns one vector of columns (gated: of both halves, dy is read once) and walks down its rows. One row at a time: several rows' loads ahead of
// their use cost more waves than they gain (8192 x 2 x 8192 bfloat16: 314 us with four rows, 172 with one or two; 156 with loads and stores past the
// caches, 4.5 TB/s, and the training step with its products 1594 -> 1553 us; as part of a block's step no difference).
template <class T, int H>
__global__ __launch_bounds__(256) void token_slope_kernel(SlopeArgs p)
{
    typedef typename Kept<T>::S S;
    constexpr int V = Elem<T>::kVec, kE = Elem<S>::kVec;               // kE: derivatives of a 16-byte vector
    const int64_t quads = (p.cols + 3) / 4;
    __shared__ float sums[256][V + 1];
    const int tid = threadIdx.x, cl = tid & (p.lanes - 1), rl = tid / p.lanes, rstep = 256 / p.lanes;
    const int64_t n = ((int64_t)blockIdx.x * p.lanes + cl) * V, left = p.cols - n;
    const int64_t chunk = (p.rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = chunk * blockIdx.y, r1 = min(r0 + chunk, p.rows);
    float db[H][V];
    #pragma unroll
    for (int h = 0; h < H; h++)
        #pragma unroll
        for (int i = 0; i < V; i++) db[h][i] = 0.f;
    // WHOLE: the thread's vector is not cut by the last column
    auto walk = [&](auto isWhole, auto isOnce)
    {
        constexpr bool WHOLE = decltype(isWhole)::value != 0, once = decltype(isOnce)::value != 0;
        const int64_t have = WHOLE ? V : left;
        for (int64_t m = r0 + rl; m < r1; m += rstep)
        {
            const RawRow<T> g = load_raw<T>(static_cast<const T*>(p.dy) + m * p.lddy + n, have, once);
            RawRow<S> d[H][V / kE];
            uint32_t bits[H];
            uint8_t c[V];
            if (p.kind == LVG_SLOPE_SMOOTH)
            {
                #pragma unroll
                for (int h = 0; h < H; h++)
                {
                    const int64_t row = m * H + h;
                    #pragma unroll
                    for (int k = 0; k < V / kE; k++) d[h][k] = load_raw<S>(static_cast<const S*>(p.slopes) + row * p.cols + n + kE * k, have - kE * k, once);
                    if constexpr (Kept<T>::kBits)
                    {
                        const uint8_t* at = reinterpret_cast<const uint8_t*>(static_cast<const S*>(p.slopes) + p.rows * H * p.cols) + row * quads + n / 4;
                        bits[h] = at[0];
                        if (WHOLE || have > 4) bits[h] |= (uint32_t)at[1] << 8;
                    }
                }
            }
            else if (p.kind == LVG_SLOPE_CODE)
            {
                const uint8_t* s = static_cast<const uint8_t*>(p.slopes) + m * p.cols + n;
                if (WHOLE) __builtin_memcpy(c, s, V);
                else
                {
                    #pragma unroll
                    for (int i = 0; i < V; i++) c[i] = i < have ? s[i] : (uint8_t)0;
                }
            }
            #pragma unroll
            for (int h = 0; h < H; h++)
            {
                float v[V];
                #pragma unroll
                for (int i = 0; i < V; i++)
                {
                    v[i] = row_load(g.v[i]);
                    if (p.kind == LVG_SLOPE_SMOOTH)
                    {
                        float s = row_load(d[h][i / kE].v[i % kE]);
                        if constexpr (Kept<T>::kBits) s = __uint_as_float(__float_as_uint(s) | (bits[h] >> (2 * i) & 3u) << 14);
                        // (the mark stops infinities and NaNs too; nothing cuts a gated unit's up half)
                        v[i] = h == 0 && __float_as_uint(s) == kCutBits ? 0.f : v[i] * s;
                    }
                    else if (p.kind == LVG_SLOPE_CODE) v[i] = c[i] == 2 ? v[i] : c[i] == 1 ? v[i] * p.alpha : 0.f;
                    v[i] *= p.gain;
                    db[h][i] += v[i];
                }
                if (p.dz) store_row<T>(static_cast<T*>(p.dz) + m * p.lddz + h * p.cols + n, have, v, once);
            }
        }
    };
    // (with `once` every vector is whole and aligned)
    if (p.once && left >= V) walk(Const<1>(), Const<1>());
    else if (left >= V) walk(Const<1>(), Const<0>());
    else if (left > 0) walk(Const<0>(), Const<0>());
    if (!p.part) return;
    #pragma unroll
    for (int h = 0; h < H; h++)
    {
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < V; i++) sums[tid][i] = db[h][i];
        __syncthreads();
        if (rl == 0 && left > 0)
        {
            float v[V];
            #pragma unroll
            for (int i = 0; i < V; i++) v[i] = db[h][i];
            for (int k = 1; k < rstep; k++)
            {
                #pragma unroll
                for (int i = 0; i < V; i++) v[i] += sums[k * p.lanes + cl][i];
            }
            float* out = p.part + ((int64_t)blockIdx.y * H + h) * p.cols + n;
            #pragma unroll
            for (int i = 0; i < V; i++) if (i < left) out[i] = v[i];
        }
    }
}

int slope_lanes(int64_t cols, int esize)
{
    const int64_t vecs = lvg_ceil_div(cols, 16 / esize);
    int lanes = 1;
    while (lanes < 256 && lanes < vecs) lanes *= 2;
    return lanes;
}

// Row chunks: about eight workgroups for each compute unit, at least four rows a thread.
int slope_slots(int64_t rows, int64_t cols, int esize)
{
    const int lanes = slope_lanes(cols, esize);
    const int64_t across = lvg_ceil_div(lvg_ceil_div(cols, 16 / esize), lanes);
    const int64_t most = lvg_ceil_div(rows, 4 * (256 / lanes));
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, std::max<int64_t>(1, 2048 / across)));
}

int esize_of(int dtype) { return dtype == LVG_F32 ? 4 : dtype == LVG_E4M3 ? 1 : 2; }
bool float_type(int dtype) { return dtype == LVG_F32 || dtype == LVG_F16 || dtype == LVG_BF16; }
bool size_ok(int64_t v) { return v >= 0 && v <= (int64_t)0x7fffffff; }

int64_t part_pitch(int64_t cols, bool gated) { return (cols + 3) / 4 * 4 * (gated ? 2 : 1); }

bool streams(int64_t rows, int64_t cols, int form) { return rows <= kStreamRows && cols <= kStreamCols && (form == LVG_TOKEN_FORWARD || form == LVG_TOKEN_GATED); }

int layout_p(int form) { return form == LVG_TOKEN_ROW_GRAD || form == LVG_TOKEN_WEIGHT_GRAD ? DOWN : ALONG; }
int layout_q(int form) { return form == LVG_TOKEN_WEIGHT_GRAD ? DOWN : ALONG; }

int64_t pad16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// ---------------------------------------------------------------------------------------------------------------------
// Layout of a product over the 256 compute units, from its sizes alone: the same answer sizes the workspace and launches.
//
// A step of a tile costs `cycles` of a compute unit that holds as many workgroups as fit (1 / 2 / 3 of the 256 / 128 / 64-row tiles), and `alone` if
// it has one; measured at 2.1 GHz on direct operands: 256 rows 1.45 us; 128: 0.48 and 0.7 us; 64: 0.33 and 0.57 us. Rows that go through registers
// cost 1.8 times as much (float32: 1.25). Splitting the summed index fills the chip when there are few tiles, and costs the float32 parts' way to memory and back and
// one more launch (about 4 us). Operands whose sizes make their rows start at odd places are repacked first, in one launch for both, where the
// product is long enough to pay for it (3000 x 1501 -> 3000, bfloat16: 62 us, and 79 us through registers; 1237 x 771 -> 515: 19 and 14 us). A linear
// layer's backward pass reads dy as it is: in odd rows it takes both operands through registers, where the repacked other one still pays, by aligned
// loads and whole chunks at its edge (8192 x 1501 -> 3001, bfloat16, training step: 636 us, and 896 without; 1536 -> 3001: 535 us, counted as direct or
// as slow steps).

constexpr int64_t kPackBlocks = (int64_t)1 << 23;         // of a repacking launch, 4 KiB each: more than 32 GiB go through registers as they are

struct TokenPlan { int tile, splits; bool pack; };

// Workspace: the parts, then the repacked operands.
struct Work { int64_t part, p, q, all; };

Work work_of(const TokenPlan& k, int64_t rows, int64_t cols, int64_t inner, int es, int form)
{
    const bool gated = form == LVG_TOKEN_GATED;
    Work w = {0, 0, 0, 0};
    if (k.splits > 1) w.part = (int64_t)k.splits * rows * part_pitch(cols, gated) * 4;
    if (k.pack)
    {
        w.p = layout_p(form) == ALONG ? cols * (gated ? 2 : 1) * pad16(inner * es) : inner * pad16(cols * es);
        if (layout_q(form) == ALONG && form != LVG_TOKEN_ROW_GRAD) w.q = rows * pad16(inner * es);
    }
    w.all = w.part + w.p + w.q;
    return w;
}

TokenPlan token_plan(int64_t rows, int64_t cols, int64_t inner, int es, int form)
{
    static const struct { int bm, bn, held; double cycles[2], alone[2], more; } kTile[3] = {     // [float32]
        {256, 256, 1, {3000., 15400.}, {3000., 15400.}, 22000.},
        {128, 128, 2, {1000., 4000.}, {1450., 4100.}, 9000.},
        {64, 128, 3, {700., 2050.}, {1150., 2100.}, 5000.}};
    const bool gated = form == LVG_TOKEN_GATED, f32 = es == 4;
    const int64_t steps = std::max<int64_t>(1, lvg_ceil_div(inner * es, 128)), width = cols * (gated ? 2 : 1);
    const int64_t pBytes = layout_p(form) == ALONG ? inner * es : cols * es;       // of an operand's row
    const Work copies = work_of({0, 1, true}, rows, cols, inner, es, form);
    const bool odd = pBytes % 16 != 0 || (layout_q(form) == ALONG && form != LVG_TOKEN_ROW_GRAD && (inner * es) % 16 != 0);
    TokenPlan best = {LVG_TILE_128, 1, false};
    double least = 1e300;
    for (int pack = 0; pack <= (odd && (copies.p + copies.q) / 4096 < kPackBlocks ? 1 : 0); pack++)
    {
        // (bytes of the operands, read and written; bytes a cycle)
        const double packing = pack ? 12000. + 2. * es * (double)inner * ((double)width + (layout_q(form) == ALONG && form != LVG_TOKEN_ROW_GRAD ? (double)rows : 0.)) / 1500. : 0.;
        const double slow = odd && !pack ? (f32 ? 1.25 : 1.8) : 1.;
        for (int t = 0; t < 3; t++)
        {
            if (es == 1 && odd && !pack && t == LVG_TILE_256) continue;
            const int64_t tiles = lvg_ceil_div(rows, kTile[t].bm) * lvg_ceil_div(cols, kTile[t].bn / (gated ? 2 : 1));
            if (tiles > kGridBlocks) continue;
            for (int64_t splits = 1; splits <= 64 && splits <= steps; splits = splits < 4 ? splits + 1 : splits * 3 / 2)
            {
                if (splits > 1 && (tiles * splits > 2048 || (double)rows * (double)width > 1e9)) break;
                const int64_t each = lvg_ceil_div(steps, splits);
                if (lvg_ceil_div(steps, each) != splits) continue;
                const int64_t perCu = lvg_ceil_div(tiles * splits, 256), rounds = lvg_ceil_div(perCu, kTile[t].held);
                const double held = (double)std::min<int64_t>(perCu, kTile[t].held);
                double cost = packing + (double)rounds * ((double)each * slow * std::max(kTile[t].alone[f32], held * kTile[t].cycles[f32]) + kTile[t].more);
                if (splits > 1) cost += 8000. + (double)splits * (double)rows * (double)width * 8. / 3000.;
                if (cost < least) { least = cost; best = {t, (int)splits, pack != 0}; }
            }
        }
    }
    return best;
}

int64_t work_bytes(int64_t rows, int64_t cols, int64_t inner, int dtype, int form)
{
    const int es = esize_of(dtype);
    if (!streams(rows, cols, form)) return work_of(token_plan(rows, cols, inner, es, form), rows, cols, inner, es, form).all;
    const bool gated = form == LVG_TOKEN_GATED;
    const int splits = token_stream_splits(rows, cols, inner * es, gated);
    return splits > 1 ? (int64_t)splits * rows * part_pitch(cols, gated) * 4 : 0;
}

// ---------------------------------------------------------------------------------------------------------------------
// Repacking: rows of n bytes to rows that start at multiples of 16 bytes, zeros behind them. Two matrices in one launch, a thread a 16-byte chunk.

struct PackArgs { const char* src[2]; char* dst[2]; int64_t ld[2], bytes[2], chunks[2]; };    // chunks: of the whole matrix

template <class T>
__global__ __launch_bounds__(256) void token_pack_kernel(PackArgs p)
{
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int which = i >= p.chunks[0] ? 1 : 0;
    i -= which ? p.chunks[0] : 0;
    if (i >= p.chunks[which]) return;
    const int64_t per = (p.bytes[which] + 15) / 16, row = i / per, at = (i - row * per) * 16;
    const char* src = p.src[which] + row * p.ld[which] + at;
    const int64_t n = (p.bytes[which] - at) / (int64_t)sizeof(T);
    constexpr int kE = 16 / (int)sizeof(T);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n >= kE) __builtin_memcpy(&v, src, 16);
    else
    {
        T e[kE];
        #pragma unroll
        for (int j = 0; j < kE; j++)
        {
            if (j < n) e[j] = reinterpret_cast<const T*>(src)[j];
            else __builtin_memset(&e[j], 0, sizeof(T));
        }
        __builtin_memcpy(&v, e, 16);
    }
    *reinterpret_cast<uint4*>(p.dst[which] + i * 16) = v;
}

int launch_pack(const PackArgs& p, int es, hipStream_t s)
{
    const int64_t blocks = lvg_ceil_div(p.chunks[0] + p.chunks[1], 256);
    if (blocks == 0) return LVG_OK;
    if (blocks > kPackBlocks) { lvg_set_error("token product: operands of %lld bytes to repack", (long long)blocks * 4096); return LVG_ERR_INVALID; }
    const dim3 grid((unsigned)blocks), block(256);
    if (es == 4) hipLaunchKernelGGL(token_pack_kernel<float>, grid, block, 0, s, p);
    else if (es == 2) hipLaunchKernelGGL(token_pack_kernel<bf16_t>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(token_pack_kernel<e4m3_t>, grid, block, 0, s, p);
    return lvg_check_launch("token product, repacking its operands");
}

// Offsets inside an operand's tile fit 32 bits.
bool near_ok(int64_t ld, int64_t count, int layout, int es, bool gated)
{
    return (layout == ALONG ? 256 * ld + (gated ? count * ld : 0) : (128 / es) * ld + 1024) < ((int64_t)1 << 32);
}

// Operands that can travel to LDS without registers: 16-byte aligned rows, whole chunks of columns.
bool direct_ok(const void* base, int64_t ld, int64_t stored, int layout, int es)
{
    if (!lvg_aligned16(base) || ld % 16 != 0) return false;
    return layout == ALONG || ((stored * es) % 16 == 0 && stored * es >= 16);
}

// The product itself: rows x cols results over `inner`, args with operands and finish filled in.
int run_product(TokenArgs& a, int form, int dtype, int out_dtype, void* work, int64_t work_size, hipStream_t s, const char* what)
{
    const int es = esize_of(dtype), os = esize_of(out_dtype);
    const bool gated = form == LVG_TOKEN_GATED;
    const int64_t rows = a.qRows, cols = a.pRows, need = work_bytes(rows, cols, a.inner, dtype, form);
    LVG_REQUIRE(need == 0 || (work && lvg_aligned16(work) && work_size >= need), "%s: the workspace must be 16-byte aligned and hold %lld bytes", what, (long long)need);
    a.ldpart = part_pitch(cols, gated);
    Finish& f = a.fin;
    auto whole = [&](const void* p, int64_t ld) { return !p || (((uintptr_t)p) % (4 * os) == 0 && ld % 4 == 0); };
    f.vec = cols % 4 == 0 && whole(f.bias, 0) && whole(f.residual, f.ldr) && whole(f.out, f.ldo) && (!f.slopes || lvg_aligned16(f.slopes));
    f.past = gated && os == 2 && rows * cols * os + slope_bytes(rows, cols, 2, f.slopeKind, out_dtype) >= (int64_t)64 << 20;
    int rc, splits;
    if (streams(rows, cols, form))
    {
        splits = token_stream_splits(rows, cols, a.inner * es, gated);
        a.part = splits > 1 ? static_cast<float*>(work) : nullptr;
        StreamArgs t = {a.p, a.q, a.ldp, a.ldq, a.inner * es, rows, cols, 0, 0, a.part, a.ldpart, f};
        t.spans = (int)lvg_ceil_div(t.bytes, 256);
        t.spansPerSplit = (int)lvg_ceil_div(t.spans, splits);
        rc = token_stream_launch(t, dtype, out_dtype, gated, splits, s);
    }
    else
    {
        TokenPlan k = token_plan(rows, cols, a.inner, es, form);
        const Work w = work_of(k, rows, cols, a.inner, es, form);
        const int pl = layout_p(form), ql = layout_q(form);
        splits = k.splits;
        a.part = splits > 1 ? static_cast<float*>(work) : nullptr;
        if (!a.pStored) a.pStored = cols;
        if (!a.qStored) a.qStored = rows;
        if (k.pack && a.inner > 0)
        {
            PackArgs g;
            memset(&g, 0, sizeof(g));
            char* at = static_cast<char*>(work) + w.part;
            if (w.p && !direct_ok(a.p, a.ldp, a.pStored, pl, es))
            {
                const int64_t n = pl == ALONG ? a.inner * es : cols * es, ld = pad16(n);
                g.src[0] = static_cast<const char*>(a.p); g.dst[0] = at; g.ld[0] = a.ldp; g.bytes[0] = n; g.chunks[0] = w.p / 16;
                a.p = at; a.ldp = ld;
                if (pl == DOWN) a.pStored = ld / es;
            }
            if (w.q && !direct_ok(a.q, a.ldq, a.qStored, ql, es))
            {
                at += w.p;
                g.src[1] = static_cast<const char*>(a.q); g.dst[1] = at; g.ld[1] = a.ldq; g.bytes[1] = a.inner * es; g.chunks[1] = w.q / 16;
                a.q = at; a.ldq = pad16(a.inner * es);
            }
            rc = launch_pack(g, es, s);
            if (rc != LVG_OK) return rc;
        }
        a.near = near_ok(a.ldp, cols, pl, es, gated) && near_ok(a.ldq, rows, ql, es, false);
        const bool direct = a.near && direct_ok(a.p, a.ldp, a.pStored, pl, es) && direct_ok(a.q, a.ldq, a.qStored, ql, es);
        // (8-bit steps through registers hold twice the fragments: the largest tile would not fit)
        if (es == 1 && !direct && k.tile == LVG_TILE_256) k.tile = LVG_TILE_128;
        const int bm = k.tile == LVG_TILE_256 ? 256 : k.tile == LVG_TILE_128 ? 128 : 64, bn = (k.tile == LVG_TILE_256 ? 256 : 128) / (gated ? 2 : 1);
        a.steps = (int)lvg_ceil_div(a.inner * es, 128);
        a.stepsPerSplit = (int)lvg_ceil_div(a.steps, splits);
        a.splits = splits;
        a.tilesM = (int)lvg_ceil_div(rows, bm);
        a.tilesN = (int)lvg_ceil_div(cols, bn);
        LVG_REQUIRE((int64_t)a.tilesM * a.tilesN <= kGridBlocks, "%s: a result of %lld x %lld", what, (long long)rows, (long long)cols);
        a.tiles = a.tilesM * a.tilesN;
        if (dtype == LVG_E4M3)      rc = token_launch_8bit(form, k.tile, direct, out_dtype, a, s);
        else if (dtype == LVG_F32)  rc = token_launch_f32(form, k.tile, direct, a, s);
        else if (dtype == LVG_F16)  rc = token_launch_f16(form, k.tile, direct, a, s);
        else                        rc = token_launch_bf16(form, k.tile, direct, a, s);
    }
    if (rc != LVG_OK || splits <= 1) return rc;
    return launch_finish(a.part, splits, a.ldpart, f, out_dtype, gated, s);
}

} // namespace

extern "C" int64_t lvg_linear_act_work(int64_t rows, int64_t outer, int64_t inner, int dtype, int gated)
{
    if (!(float_type(dtype) || dtype == LVG_E4M3) || !size_ok(rows) || !size_ok(outer) || !size_ok(inner)) return LVG_ERR_INVALID;
    return rows && outer ? work_bytes(rows, outer, inner, dtype, gated ? LVG_TOKEN_GATED : LVG_TOKEN_FORWARD) : 0;
}

extern "C" int64_t lvg_linear_slope_bytes(int64_t rows, int64_t outer, int halves, int slope_kind, int dtype)
{
    if (!float_type(dtype) || !size_ok(rows) || !size_ok(outer) || (halves != 1 && halves != 2) || slope_kind < LVG_SLOPE_NONE || slope_kind > LVG_SLOPE_CODE) return LVG_ERR_INVALID;
    return slope_bytes(rows, outer, halves, slope_kind, dtype);
}

extern "C" int lvg_linear_act(const void* x, const void* w, const void* b, const void* residual, const float* x_scale, const float* w_scale,
                              void* y, void* slopes, void* work, int64_t work_size, int64_t rows, int64_t outer, int64_t inner,
                              int64_t x_stride, int64_t w_stride, int64_t residual_stride, int64_t y_stride,
                              int dtype, int out_dtype, int gated, int act, int slope_kind, float alpha, float gain, float clamp, void* stream)
{
    LVG_REQUIRE(float_type(dtype) || dtype == LVG_E4M3, "lvg_linear_act: operands must be float32 / float16 / bfloat16 / e4m3 (dtype %d)", dtype);
    if (dtype == LVG_E4M3)
        LVG_REQUIRE((out_dtype == LVG_BF16 || out_dtype == LVG_F16) && x_scale && w_scale, "lvg_linear_act: 8-bit operands need both scales and a float16 / bfloat16 result");
    else
        LVG_REQUIRE(out_dtype == dtype && !x_scale && !w_scale, "lvg_linear_act: the result has the operands' type, scales belong to 8-bit operands");
    LVG_REQUIRE(size_ok(rows) && size_ok(outer) && size_ok(inner) && (!gated || size_ok(2 * outer)), "lvg_linear_act: bad size");
    LVG_REQUIRE(act >= LVG_ACT_LINEAR && act <= LVG_ACT_SWISH, "lvg_linear_act: unknown activation %d", act);
    if (rows == 0 || outer == 0) return LVG_OK;
    LVG_REQUIRE(y && (inner == 0 || (x && w)), "lvg_linear_act: missing pointer");
    LVG_REQUIRE(x_stride >= 0 && w_stride >= 0 && residual_stride >= 0 && y_stride >= outer, "lvg_linear_act: bad row stride");
    LVG_REQUIRE(!gated || (!residual && clamp < 0.f), "lvg_linear_act: a gated unit has neither residual nor clamp");
    LVG_REQUIRE(slope_kind == LVG_SLOPE_NONE || (slopes && (slope_kind == LVG_SLOPE_SMOOTH || (slope_kind == LVG_SLOPE_CODE && !gated &&
                (act == LVG_ACT_LINEAR || act == LVG_ACT_RELU || act == LVG_ACT_LRELU)))), "lvg_linear_act: bad slopes");
    TokenArgs a;
    memset(&a, 0, sizeof(a));
    const int es = esize_of(dtype);
    a.p = w; a.q = x;
    a.ldp = w_stride * es; a.ldq = x_stride * es;
    a.inner = inner; a.pRows = outer; a.qRows = rows;
    Finish& f = a.fin;
    f.qs = x_scale; f.ps = w_scale; f.bias = b; f.residual = residual; f.out = y; f.slopes = slope_kind ? slopes : nullptr;
    f.ldr = residual_stride; f.ldo = y_stride; f.rows = rows; f.cols = outer;
    f.act = act; f.slopeKind = slope_kind; f.alpha = alpha; f.gain = gain; f.clamp = clamp;
    return run_product(a, gated ? LVG_TOKEN_GATED : LVG_TOKEN_FORWARD, dtype, out_dtype, work, work_size, static_cast<hipStream_t>(stream), "lvg_linear_act");
}

namespace {

// One of the two products of the backward pass: grad = gain * dz . w (weight false) or gain * dz^T . x. dz_whole: dz's rows are readable up to
// their stride.
int grad_product(const void* dz, int64_t dz_stride, bool dz_whole, const void* other, int64_t other_stride, void* grad, void* work, int64_t work_size,
                 int64_t rows, int64_t outer, int64_t inner, bool weight, float gain, int dtype, hipStream_t s)
{
    if (inner == 0) return LVG_OK;
    TokenArgs a;
    memset(&a, 0, sizeof(a));
    const int es = esize_of(dtype);
    a.p = other; a.q = dz;
    a.ldp = other_stride * es; a.ldq = dz_stride * es;
    a.inner = weight ? rows : outer; a.pRows = inner; a.qRows = weight ? outer : rows;
    if (weight && dz_whole) a.qStored = dz_stride;
    Finish& f = a.fin;
    f.out = grad; f.ldo = inner; f.rows = a.qRows; f.cols = inner;
    f.act = LVG_ACT_LINEAR; f.gain = gain; f.clamp = -1.f;
    return run_product(a, weight ? LVG_TOKEN_WEIGHT_GRAD : LVG_TOKEN_ROW_GRAD, dtype, dtype, work, work_size, s, "lvg_linear_backward");
}

// Workspace of a backward pass: dz (rows that start at multiples of 16 bytes whatever the width: both products read them as they like it best),
// the column sums by row ranges, and what the larger of the two products needs (they follow one another on the stream).
struct BackWork { int64_t dz, dzStride, part, product, all; int slots; };

BackWork back_work(int64_t rows, int64_t outer, int64_t inner, int halves, int kind, bool dx, bool dw, bool db, int dtype)
{
    const int es = esize_of(dtype);
    BackWork w = {0, pad16(outer * halves * es) / es, 0, 0, 0, 0};
    if (rows == 0 || outer == 0) return w;
    w.slots = slope_slots(rows, outer, es);
    if (kind != LVG_SLOPE_NONE && (dx || dw)) w.dz = rows * w.dzStride * es;
    if (db) w.part = pad16((int64_t)w.slots * halves * outer * 4);
    if (dx && inner) w.product = work_bytes(rows, inner, outer * halves, dtype, LVG_TOKEN_ROW_GRAD);
    if (dw && inner) w.product = std::max(w.product, work_bytes(outer * halves, inner, rows, dtype, LVG_TOKEN_WEIGHT_GRAD));
    w.all = w.dz + w.part + w.product;
    return w;
}

bool back_sizes(int64_t rows, int64_t outer, int64_t inner, int halves, int kind, int dtype)
{
    return float_type(dtype) && size_ok(rows) && size_ok(outer) && size_ok(inner) && (halves == 1 || halves == 2) && size_ok(outer * halves) &&
           (kind == LVG_SLOPE_NONE || kind == LVG_SLOPE_SMOOTH || kind == LVG_SLOPE_CODE) && (halves == 1 || kind == LVG_SLOPE_SMOOTH);
}

} // namespace

extern "C" int64_t lvg_linear_backward_work(int64_t rows, int64_t outer, int64_t inner, int halves, int slope_kind, int grads, int dtype)
{
    if (!back_sizes(rows, outer, inner, halves, slope_kind, dtype)) return LVG_ERR_INVALID;
    return back_work(rows, outer, inner, halves, slope_kind, grads & 1, grads & 2, grads & 4, dtype).all;
}

extern "C" int lvg_linear_backward(const void* dy, const void* slopes, const void* x, const void* w, void* dx, void* dw, void* db, void* work, int64_t work_size,
                                   int64_t rows, int64_t outer, int64_t inner, int64_t dy_stride, int64_t x_stride, int64_t w_stride,
                                   int halves, int slope_kind, float alpha, float gain, int dtype, void* stream)
{
    LVG_REQUIRE(back_sizes(rows, outer, inner, halves, slope_kind, dtype), "lvg_linear_backward: bad size, type or slopes");
    // (nothing to sum over: the gradients that have values are zeros)
    const bool none = rows == 0 || outer == 0;
    LVG_REQUIRE((none || (dy && (slope_kind == LVG_SLOPE_NONE || slopes))) && (!dx || inner == 0 || none || w) && (!dw || inner == 0 || none || x), "lvg_linear_backward: missing pointer");
    LVG_REQUIRE(dy_stride >= 0 && x_stride >= 0 && w_stride >= 0, "lvg_linear_backward: negative row stride");
    const BackWork k = back_work(rows, outer, inner, halves, slope_kind, dx != nullptr, dw != nullptr, db != nullptr, dtype);
    LVG_REQUIRE(k.all == 0 || (work && lvg_aligned16(work) && work_size >= k.all), "lvg_linear_backward: the workspace must be 16-byte aligned and hold %lld bytes", (long long)k.all);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool plain = slope_kind == LVG_SLOPE_NONE;               // dy times the gain is the gradient of the sums
    char* const mem = static_cast<char*>(work);
    const void* dz = plain ? dy : mem;                             // (the column sums alone leave none)
    const int64_t dzStride = plain ? dy_stride : k.dzStride, total = outer * halves;
    if (none && db && outer) row_column_sum(nullptr, db, 0, total, 0.f, dtype, s);
    if (!none && (!plain || db))
    {
        float* part = db ? reinterpret_cast<float*>(mem + k.dz) : nullptr;
        SlopeArgs a = {dy, slopes, k.dz ? mem : nullptr, part, rows, outer, dy_stride, k.dzStride, slope_kind, slope_lanes(outer, esize_of(dtype)), alpha, plain ? 1.f : gain, false};
        const int es = esize_of(dtype);
        a.once = rows * total * es >= (int64_t)64 << 20 && lvg_aligned16(dy) && (dy_stride * es) % 16 == 0 && (outer * es) % 16 == 0 && (!slopes || lvg_aligned16(slopes));
        const dim3 grid((unsigned)lvg_ceil_div(lvg_ceil_div(outer, 16 / esize_of(dtype)), a.lanes), (unsigned)k.slots), block(256);
        #define LVG_TYPE(T) { \
            if (halves == 2) hipLaunchKernelGGL((token_slope_kernel<T, 2>), grid, block, 0, s, a); \
            else             hipLaunchKernelGGL((token_slope_kernel<T, 1>), grid, block, 0, s, a); }
        if (dtype == LVG_F32) LVG_TYPE(float) else if (dtype == LVG_F16) LVG_TYPE(f16_t) else LVG_TYPE(bf16_t)
        #undef LVG_TYPE
        if (db) row_column_sum(part, db, k.slots, total, plain ? gain : 1.f, dtype, s);
        const int rc = lvg_check_launch("lvg_linear_backward");
        if (rc != LVG_OK) return rc;
    }
    void* const pw = mem + k.dz + k.part;
    if (dx && rows)
    {
        const int rc = grad_product(dz, dzStride, !plain, w, w_stride, dx, pw, k.product, rows, total, inner, false, plain ? gain : 1.f, dtype, s);
        if (rc != LVG_OK) return rc;
    }
    if (dw && outer) return grad_product(dz, dzStride, !plain, x, x_stride, dw, pw, k.product, rows, total, inner, true, plain ? gain : 1.f, dtype, s);
    return LVG_OK;
}
