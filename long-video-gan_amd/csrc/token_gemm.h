// token_gemm.h -- the matrix products of token rows on the gfx950 matrix cores, one K loop for the three of them:
//
//   forward      y[m][n]  = sum_k x[m][k] w[n][k]            rows x, columns w, both with k along their rows
//   row gradient dx[m][k] = sum_n dz[m][n] w[n][k]           columns w with the summed index DOWN its rows
//   weight       dw[n][k] = sum_m dz[m][n] x[m][k]           both operands with the summed index down their rows
//
// A workgroup owns a BM x BN tile of the result and steps over the summed index 128 bytes at a time (64 16-bit, 32 float32 or 128 8-bit values):
// the two operand tiles of a step lie in one of two LDS buffers while the next step's travel to the other. The tile of an operand whose rows run
// along the summed index ("along") is [row][128 bytes]; of the other kind ("down") [index][BX values], exactly as in memory, and is read
// through the transposing LDS read, so neither gradient needs a transposed copy of its operands. 16-byte chunks are exchanged inside a tile so
// that the reads of a wave meet every LDS bank once (along: chunk ^ (row / 2) & 7; down: 64-byte groups ^ index & 3).
//
// The column operand is the matrix instruction's first one: a lane then holds four neighbouring columns of one row, and what is done with the
// sums (token_act.h) moves whole vectors. The tile leaves through LDS, wave by wave without a barrier, in rows of 64 columns.
//
// Aligned operands go from memory to LDS without registers; rows that start at odd places are loaded (unaligned 16-byte accesses), held over the
// step's products and written to LDS behind them. Steps past the operand's last whole 128 bytes are loaded under masks, zeros beyond the end.
//
// A result too small for the chip is split over the summed index: every part writes its float32 sums, token_finish.hip adds them in order.
#pragma once
#include "wgrad_common.h"
#include "token_act.h"

struct e4m3_t { uint8_t bits; };

struct TokenArgs
{
    const void* p;             // column operand
    const void* q;             // row operand
    int64_t     ldp, ldq;      // bytes between stored rows
    int64_t     inner;         // summed index
    int64_t     pRows, qRows;  // columns / rows of the result (gated: pRows of each half)
    int64_t     steps, stepsPerSplit;
    int64_t     tiles, tilesN;
    int         tilesM;
    int         splits;
    float*      part;          // [splits][rows][ldpart] or NULL
    int64_t     ldpart;        // gated: the up half lies ldpart / 2 behind the gate half
    Finish      fin;
};

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) u32x4* lds_vec_ptr;
typedef __attribute__((address_space(3))) uint32_t* lds_word_ptr;

enum { ALONG = 0, DOWN = 1 };

template <class T, int BX, int LAYOUT> struct Fragments;

// One 16-byte fragment: this lane's column (lane & 31 of a block of 32) at 16 / size values of the summed index. Which ones is the same for both
// operands; the matrix instruction sums over all of them.
template <class T, int BX> struct Fragments<T, BX, ALONG>
{
    uint32_t off[4];
    __device__ __forceinline__ void init(int lane, int base)
    {
        #pragma unroll
        for (int ks = 0; ks < 4; ks++)
            off[ks] = (uint32_t)(base + (lane & 31)) * 128u + (uint32_t)(((2 * ks + (lane >> 5)) ^ ((lane >> 1) & 7)) << 4);
    }
    __device__ __forceinline__ uint4 read(uint32_t tile, int j, int ks) const
    {
        const u32x4 v = *(lds_vec_ptr)(uintptr_t)(tile + off[ks] + (uint32_t)j * 4096u);
        uint4 r;
        __builtin_memcpy(&r, &v, 16);
        return r;
    }
};

template <class T, int BX> struct Fragments<T, BX, DOWN>
{
    static constexpr int kPitch = BX * (int)sizeof(T);
    uint32_t off[4];           // one per block of 32 columns
    __device__ __forceinline__ void init(int lane, int base)
    {
        if (sizeof(T) == 4)
        {
            #pragma unroll
            for (int j = 0; j < 4; j++) off[j] = (uint32_t)(4 * (lane >> 5)) * kPitch + (uint32_t)(base + 32 * j + (lane & 31)) * 4u;
            return;
        }
        const uint32_t row = (uint32_t)(8 * (lane >> 5) + ((lane & 15) >> 2));
        const uint32_t sw = kPitch >= 256 ? (row & 3u) : ((row >> 1) & 1u);
        #pragma unroll
        for (int j = 0; j < 4; j++)
            off[j] = row * kPitch + (((uint32_t)(base / 32 + j) ^ sw) << 6) + 32u * ((lane >> 4) & 1) + 8u * (lane & 3);
    }
    __device__ __forceinline__ uint4 read(uint32_t tile, int j, int ks) const
    {
        uint4 r;
        if (sizeof(T) == 4)
        {
            uint32_t w[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) w[i] = *(lds_word_ptr)(uintptr_t)(tile + off[j] + (uint32_t)((8 * ks + i) * kPitch));
            __builtin_memcpy(&r, w, 16);
            return r;
        }
        const uint32_t at = tile + off[j] + (uint32_t)(16 * ks * kPitch);
        const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(uintptr_t)at);
        const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(uintptr_t)(at + 4u * kPitch));
        __builtin_memcpy(&r, &lo, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
        return r;
    }
};

// Moves one operand's tiles from memory to LDS. The tile is BX * 8 chunks of 16 bytes, thread t takes chunks t, t + NTHR, ...
template <class T, int BX, int LAYOUT, int NTHR, bool GATED, bool DIRECT> struct Loader
{
    static constexpr int kE = 16 / (int)sizeof(T);                 // values a chunk
    static constexpr int kDepth = 128 / (int)sizeof(T);            // summed index a step
    static constexpr int kNum = BX * 8 / NTHR;
    static constexpr int kPitchChunks = BX * (int)sizeof(T) / 16;  // down
    const char* base;          // operand at the tile's first row (along) / column (down)
    int64_t     ld, inner, left;   // left: rows / columns of the operand from the tile's first on
    int64_t     upOff;         // gated: bytes from a gate row to its up row
    int         tid;
    uint32_t    off[DIRECT ? kNum : 1];
    uint4       hold[DIRECT ? 1 : kNum];

    // row of the tile -> row of the operand behind the tile's first one; gated tiles alternate 32 gate rows and 32 up rows
    __device__ __forceinline__ int64_t place(int row, bool& up) const
    {
        up = GATED && (row & 32);
        const int64_t r = GATED ? (row >> 6) * 32 + (row & 31) : row;
        return r < left ? r : left - 1;            // past the end: the last row again, its products are not stored
    }
    __device__ __forceinline__ void chunk_of(int i, int& row, int& chunk) const
    {
        const int c = i * NTHR + tid;
        if (LAYOUT == ALONG)
        {
            row = c >> 3;
            chunk = (c & 7) ^ ((row >> 1) & 7);
        }
        else
        {
            row = c / kPitchChunks;
            chunk = c % kPitchChunks;
            if (sizeof(T) == 2) chunk ^= kPitchChunks >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
        }
    }
    __device__ __forceinline__ void init(const void* operand, int64_t ld_, int64_t inner_, int64_t first, int64_t count, int tid_)
    {
        ld = ld_; inner = inner_; left = count - first; tid = tid_;
        base = static_cast<const char*>(operand) + (LAYOUT == ALONG ? first * ld : first * (int64_t)sizeof(T));
        upOff = GATED ? count * ld : 0;
        if (DIRECT)
        {
            #pragma unroll
            for (int i = 0; i < kNum; i++)
            {
                int row, chunk;
                chunk_of(i, row, chunk);
                if (LAYOUT == ALONG)
                {
                    bool up;
                    const int64_t r = place(row, up);
                    off[i] = (uint32_t)(r * ld + (up ? upOff : 0) + chunk * 16);
                }
                else
                {
                    int64_t col = (int64_t)chunk * kE;
                    if (col > left - kE) col = left - kE;
                    off[i] = (uint32_t)(row * ld + col * (int64_t)sizeof(T));
                }
            }
        }
    }
    __device__ __forceinline__ uint4 masked(int64_t step, int i) const
    {
        int row, chunk;
        chunk_of(i, row, chunk);
        const char* at;
        int64_t n;                                 // valid values of the chunk
        if (LAYOUT == ALONG)
        {
            bool up;
            const int64_t r = place(row, up);
            const int64_t k = step * kDepth + chunk * kE;
            at = base + r * ld + (up ? upOff : 0) + k * (int64_t)sizeof(T);
            n = inner - k;
        }
        else
        {
            const int64_t k = step * kDepth + row;
            at = base + k * ld + (int64_t)chunk * 16;
            n = k < inner ? left - (int64_t)chunk * kE : 0;
        }
        uint4 r = make_uint4(0, 0, 0, 0);
        if (n >= kE) __builtin_memcpy(&r, at, 16);
        else if (n > 0)
        {
            T e[kE];
            #pragma unroll
            for (int j = 0; j < kE; j++)
            {
                if (j < n) e[j] = reinterpret_cast<const T*>(at)[j];
                else __builtin_memset(&e[j], 0, sizeof(T));
            }
            __builtin_memcpy(&r, e, 16);
        }
        return r;
    }
    __device__ __forceinline__ void put(uint32_t tile, int i, const uint4& v) const
    {
        u32x4 w;
        __builtin_memcpy(&w, &v, 16);
        *(lds_vec_ptr)(uintptr_t)(tile + (uint32_t)(i * NTHR + tid) * 16u) = w;
    }
    // before a step's products: start what the next step needs
    __device__ __forceinline__ void begin(int64_t step, uint32_t tile)
    {
        if (DIRECT)
        {
            if ((step + 1) * kDepth <= inner)
            {
                const char* b = base + (LAYOUT == ALONG ? step * 128 : step * kDepth * ld);
                #pragma unroll
                for (int i = 0; i < kNum; i++)
                    wdma16(reinterpret_cast<const unsigned char*>(b), off[i], tile + (uint32_t)(i * NTHR + (tid & ~63)) * 16u);
            }
            else
            {
                #pragma unroll 1
                for (int i = 0; i < kNum; i++) put(tile, i, masked(step, i));
            }
        }
        else
        {
            #pragma unroll
            for (int i = 0; i < kNum; i++) hold[i] = masked(step, i);
        }
    }
    // behind them
    __device__ __forceinline__ void end(uint32_t tile)
    {
        if (DIRECT) return;
        #pragma unroll
        for (int i = 0; i < kNum; i++) put(tile, i, hold[i]);
    }
};

template <class T> struct Product
{
    // 32 x 32 block += fragments of the 128-byte step's quarter
    static __device__ __forceinline__ f32x16 run(const uint4& a, const uint4& b, const f32x16& c) { return MmaW<T>::run(a, b, c); }
};
template <> struct Product<float>
{
    static __device__ __forceinline__ f32x16 run(const uint4& a, const uint4& b, f32x16 c)
    {
        const float av[4] = {__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w)};
        const float bv[4] = {__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w)};
        #pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(av[i], bv[i], c, 0, 0, 0);
        return c;
    }
};

// Two quarters of a step of 8-bit values: 32 bytes a lane, 64 values of the summed index (twice the 16-bit rate). Both scale operands are 2^0.
__device__ __forceinline__ f32x16 product8(const uint4& a0, const uint4& a1, const uint4& b0, const uint4& b1, const f32x16& c)
{
    i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
    i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

// LDS written by the lanes of a wave, read by others of the same wave: the hardware keeps their order, this makes the compiler keep it.
__device__ __forceinline__ void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// T operands, O results; WR x WC waves, each with a (BM / WR) x 64 part of the tile.
template <class T, class O, int BM, int BN, int WR, int WC, int PL, int QL, bool GATED, bool DIRECT>
__global__ __launch_bounds__(WR * WC * 64) void token_gemm_kernel(TokenArgs a)
{
    constexpr int kThreads = WR * WC * 64, MT = BM / WR / 32, NT = BN / WC / 32;
    static_assert(NT == 2 && MT >= 1 && MT <= 4, "a wave owns two blocks of 32 columns");
    constexpr uint32_t kBufBytes = (uint32_t)(BM + BN) * 128u;
    constexpr int kOutPitch = 64 * 4 + 16;                         // bytes of a row of a wave's results on their way out
    static_assert(WR * WC * 32 * kOutPitch <= 2 * (int)kBufBytes, "the results leave through the operands' LDS");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * kBufBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WC, wc = wave % WC;

    // Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, in bands of four tile rows, so that the tiles its 32 compute
    // units work on at a time share operand rows in its L2.
    const int64_t total = gridDim.x;
    int64_t id = blockIdx.x;
    {
        const int64_t each = total / 8, more = total % 8, x = id % 8;
        id = x * each + (x < more ? x : more) + id / 8;
    }
    const int split = (int)(id / a.tiles);
    id -= (int64_t)split * a.tiles;
    const int64_t band = 4 * a.tilesN, g = id / band;
    const int64_t high = min((int64_t)4, (int64_t)a.tilesM - g * 4);
    const int64_t tm = g * 4 + (id - g * band) % high, tn = (id - g * band) / high;
    const int64_t m0 = tm * BM, n0 = tn * (GATED ? BN / 2 : BN);

    Loader<T, BN, PL, kThreads, GATED, DIRECT> pl;
    Loader<T, BM, QL, kThreads, false, DIRECT> ql;
    pl.init(a.p, a.ldp, a.inner, n0, a.pRows, tid);
    ql.init(a.q, a.ldq, a.inner, m0, a.qRows, tid);
    Fragments<T, BN, PL> pf;
    Fragments<T, BM, QL> qf;
    pf.init(lane, wc * 64);
    qf.init(lane, wr * MT * 32);

    f32x16 acc[MT][NT];
    #pragma unroll
    for (int i = 0; i < MT; i++)
        #pragma unroll
        for (int j = 0; j < NT; j++)
            #pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    const uint32_t lds = (uint32_t)(uintptr_t)smem;
    const int64_t s0 = split * a.stepsPerSplit, s1 = min(s0 + a.stepsPerSplit, a.steps);
    if (s0 < s1)
    {
        pl.begin(s0, lds);
        ql.begin(s0, lds + BN * 128);
        pl.end(lds);
        ql.end(lds + BN * 128);
    }
    for (int64_t s = s0; s < s1; s++)
    {
        const uint32_t pt = lds + (uint32_t)((s - s0) & 1) * kBufBytes, qt = pt + BN * 128;
        const uint32_t pn = lds + (uint32_t)((s - s0 + 1) & 1) * kBufBytes, qn = pn + BN * 128;
        // this step's tiles have arrived, and every wave is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < s1)
        {
            pl.begin(s + 1, pn);
            ql.begin(s + 1, qn);
        }
        if constexpr (sizeof(T) == 1)
        {
            #pragma unroll
            for (int ks = 0; ks < 4; ks += 2)
            {
                uint4 pv[NT][2], qv[MT][2];
                #pragma unroll
                for (int j = 0; j < NT; j++) { pv[j][0] = pf.read(pt, j, ks); pv[j][1] = pf.read(pt, j, ks + 1); }
                #pragma unroll
                for (int i = 0; i < MT; i++) { qv[i][0] = qf.read(qt, i, ks); qv[i][1] = qf.read(qt, i, ks + 1); }
                #pragma unroll
                for (int i = 0; i < MT; i++)
                    #pragma unroll
                    for (int j = 0; j < NT; j++) acc[i][j] = product8(pv[j][0], pv[j][1], qv[i][0], qv[i][1], acc[i][j]);
            }
        }
        else
        {
            #pragma unroll
            for (int ks = 0; ks < 4; ks++)
            {
                uint4 pv[NT], qv[MT];
                #pragma unroll
                for (int j = 0; j < NT; j++) pv[j] = pf.read(pt, j, ks);
                #pragma unroll
                for (int i = 0; i < MT; i++) qv[i] = qf.read(qt, i, ks);
                #pragma unroll
                for (int i = 0; i < MT; i++)
                    #pragma unroll
                    for (int j = 0; j < NT; j++) acc[i][j] = Product<T>::run(pv[j], qv[i], acc[i][j]);
            }
        }
        if (s + 1 < s1)
        {
            pl.end(pn);
            ql.end(qn);
        }
    }
    __syncthreads();

    // A block's lane holds row lane & 31, columns 8 (r / 4) + 4 (lane / 32) + r % 4.
    unsigned char* const out = smem + wave * 32 * kOutPitch;
    #pragma unroll
    for (int i = 0; i < MT; i++)
    {
        #pragma unroll
        for (int j = 0; j < NT; j++)
            #pragma unroll
            for (int c = 0; c < 4; c++)
                *reinterpret_cast<float4*>(out + (lane & 31) * kOutPitch + (32 * j + 8 * c + 4 * (lane >> 5)) * 4) =
                    make_float4(acc[i][j][4 * c], acc[i][j][4 * c + 1], acc[i][j][4 * c + 2], acc[i][j][4 * c + 3]);
        wave_lds_order();
        const int64_t mBase = m0 + wr * MT * 32 + i * 32;
        constexpr int kLanes = GATED ? 8 : 16;                     // lanes a row, four columns each
        #pragma unroll 1
        for (int r = 0; r < 32; r += 64 / kLanes)
        {
            const int row = r + lane / kLanes, c = (lane % kLanes) * 4;
            const int64_t m = mBase + row, n = n0 + wc * (GATED ? 32 : 64) + c;
            const float4 v4 = *reinterpret_cast<const float4*>(out + row * kOutPitch + c * 4);
            float v[4] = {v4.x, v4.y, v4.z, v4.w}, u[4] = {0.f, 0.f, 0.f, 0.f};
            if (GATED)
            {
                const float4 u4 = *reinterpret_cast<const float4*>(out + row * kOutPitch + (32 + c) * 4);
                u[0] = u4.x; u[1] = u4.y; u[2] = u4.z; u[3] = u4.w;
            }
            if (a.part)
            {
                if (m >= a.qRows || n >= a.pRows) continue;
                float* at = a.part + ((int64_t)split * a.qRows + m) * a.ldpart + n;      // (ldpart, or each half of it, is a multiple of four)
                *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
                if (GATED) *reinterpret_cast<float4*>(at + a.ldpart / 2) = make_float4(u[0], u[1], u[2], u[3]);
            }
            else finish4<O, GATED>(a.fin, m, n, v, u);
        }
        wave_lds_order();
    }
}

} // namespace

// How a product is laid out over the chip (token_finish.hip); the same answer sizes the workspace and launches.
struct TokenPlan { int tile, splits; };
enum { LVG_TILE_256 = 0, LVG_TILE_128 = 1, LVG_TILE_64 = 2 };
TokenPlan token_plan(int64_t rows, int64_t cols, int64_t inner, int esize, bool gated);

// One launcher per operand type and kind of product, each in a file of its own (they are compiled side by side).
enum { LVG_TOKEN_FORWARD = 0, LVG_TOKEN_GATED = 1, LVG_TOKEN_ROW_GRAD = 2, LVG_TOKEN_WEIGHT_GRAD = 3 };
int token_launch_bf16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_f16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_f32(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_8bit(int form, int tile, bool direct, int out_dtype, const TokenArgs& a, hipStream_t s);

namespace {

template <class T, class O, int PL, int QL, bool GATED> int token_launch_form(int tile, bool direct, const TokenArgs& a, hipStream_t s)
{
    const int64_t blocks = a.tiles * a.splits;
    if (blocks > ((int64_t)1 << 22)) { lvg_set_error("token product: %lld workgroups", (long long)blocks); return LVG_ERR_INVALID; }
    const dim3 grid((unsigned)blocks);
    #define LVG_TILE(ID, BM, BN, WR, WC) if (tile == ID) { \
        if (direct) hipLaunchKernelGGL((token_gemm_kernel<T, O, BM, BN, WR, WC, PL, QL, GATED, true>), grid, dim3(WR * WC * 64), 0, s, a); \
        else        hipLaunchKernelGGL((token_gemm_kernel<T, O, BM, BN, WR, WC, PL, QL, GATED, false>), grid, dim3(WR * WC * 64), 0, s, a); }
    LVG_TILE(LVG_TILE_256, 256, 256, 2, 4)
    LVG_TILE(LVG_TILE_128, 128, 128, 2, 2)
    LVG_TILE(LVG_TILE_64, 64, 128, 2, 2)
    #undef LVG_TILE
    return lvg_check_launch("token product");
}

} // namespace
