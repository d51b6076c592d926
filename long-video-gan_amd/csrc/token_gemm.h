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
// A wave of the largest tile owns 128 x 128 results (256 accumulator registers, one wave a SIMD): 32 fragment reads feed 64 products a step, where
// eight waves of 128 x 64 would read 48.
//
// Aligned operands go from memory to LDS without registers; rows that start at odd places are loaded (unaligned 16-byte accesses), held over the
// step's products and written to LDS behind them. Steps past the operand's last whole 128 bytes are loaded under masks, zeros beyond the end.
//
// A result too small for the chip is split over the summed index: every part writes its float32 sums, token_finish.hip adds them in order.
#pragma once
#include "wgrad_common.h"
#include "token_act.h"
#include "token_stream.h"

struct TokenArgs
{
    const void* p;             // column operand
    const void* q;             // row operand
    int64_t     ldp, ldq;      // bytes between stored rows
    int64_t     inner;         // summed index
    int64_t     pRows, qRows;  // columns / rows of the result (gated: pRows of each half)
    int64_t     pStored, qStored;   // columns / rows of them that the operands hold: more where their rows are padded
    int         steps, stepsPerSplit;
    int         tiles, tilesM, tilesN, splits;
    bool        near;          // offsets inside a tile fit 32 bits
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
    // at: the operand's place in the tile buffer
    __device__ __forceinline__ uint4 read(uint32_t tile, int at, int j, int ks) const
    {
        const u32x4 v = ((lds_vec_ptr)(uintptr_t)(tile + off[ks]))[at / 16 + j * 256];
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
    __device__ __forceinline__ uint4 read(uint32_t tile, int at, int j, int ks) const
    {
        uint4 r;
        if (sizeof(T) == 4)
        {
            uint32_t w[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) w[i] = ((lds_word_ptr)(uintptr_t)(tile + off[j]))[(at + (8 * ks + i) * kPitch) / 4];
            __builtin_memcpy(&r, w, 16);
            return r;
        }
        const lds_tr_ptr from = (lds_tr_ptr)(uintptr_t)(tile + off[j]);
        const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(from + (at + 16 * ks * kPitch) / 8);
        const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(from + (at + (16 * ks + 4) * kPitch) / 8);
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
    static constexpr int kFirst = sizeof(T) == 1 ? kNum : kNum / 2;    // chunks a step's first sends are for (see spread)
    const char* base;          // operand at the tile's first row (along) / column (down)
    int64_t     ld, inner, left;   // left: rows / columns of the operand from the tile's first on
    int64_t     upOff;         // gated: bytes from a gate row to its up row
    int         tid;
    uint32_t    off[kNum];     // of the chunks, from the tile's place in the operand on
    uint4       hold[DIRECT ? 1 : kNum];
    uint32_t    edge;          // through registers: chunks that are never whole (bits); all of them where offsets pass 32 bits

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
    __device__ __forceinline__ void init(const void* operand, int64_t ld_, int64_t inner_, int64_t first, int64_t count, int tid_, bool near)
    {
        ld = ld_; inner = inner_; left = count - first; tid = tid_;
        base = static_cast<const char*>(operand) + (LAYOUT == ALONG ? first * ld : first * (int64_t)sizeof(T));
        upOff = GATED ? count * ld : 0;
        edge = near ? 0u : ~0u;
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
                if (col > left - kE)
                {
                    if (!DIRECT) edge |= 1u << i;
                    col = left - kE;
                }
                off[i] = (uint32_t)(row * ld + col * (int64_t)sizeof(T));
            }
        }
    }
    __device__ __forceinline__ uint4 masked(int step, int i) const
    {
        int row, chunk;
        chunk_of(i, row, chunk);
        const char* at;
        int64_t n;                                 // valid values of the chunk
        if (LAYOUT == ALONG)
        {
            bool up;
            const int64_t r = place(row, up);
            const int64_t k = (int64_t)step * kDepth + chunk * kE;
            at = base + r * ld + (up ? upOff : 0) + k * (int64_t)sizeof(T);
            n = inner - k;
        }
        else
        {
            const int64_t k = (int64_t)step * kDepth + row;
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
    // a whole step's tile straight to LDS, this thread's chunk i of it
    __device__ __forceinline__ void send(int i, int step, uint32_t tile, int wave) const
    {
        const char* b = base + (int64_t)step * (LAYOUT == ALONG ? 128 : kDepth * ld);
        wdma16(reinterpret_cast<const unsigned char*>(b), off[i], tile + (uint32_t)(i * NTHR + wave * 64) * 16u);
    }
    // A step's tile is started in two halves (0, 1). Rows that go through registers are all loaded in the first, masked steps of direct ones are
    // written in the second.
    __device__ __forceinline__ void begin(int half, int step, uint32_t tile, int wave)
    {
        if (!DIRECT)
        {
            if (half) return;
            if ((int64_t)(step + 1) * kDepth <= inner)
            {
                const char* b = base + (int64_t)step * (LAYOUT == ALONG ? 128 : kDepth * ld);
                if (edge == 0)
                {
                    #pragma unroll
                    for (int i = 0; i < kNum; i++) __builtin_memcpy(&hold[i], b + off[i], 16);
                    return;
                }
                #pragma unroll
                for (int i = 0; i < kNum; i++)
                {
                    if (edge >> i & 1) hold[i] = masked(step, i);
                    else __builtin_memcpy(&hold[i], b + off[i], 16);
                }
            }
            else
            {
                #pragma unroll
                for (int i = 0; i < kNum; i++) hold[i] = masked(step, i);
            }
        }
        else if ((int64_t)(step + 1) * kDepth <= inner)
        {
            #pragma unroll
            for (int i = 0; i < kNum; i++) if ((i < kFirst) == (half == 0)) send(i, step, tile, wave);
        }
        else if (half)
        {
            #pragma unroll 1
            for (int i = 0; i < kNum; i++) put(tile, i, masked(step, i));
        }
    }
    // registers to LDS
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
// The unit adds the products of eight neighbouring values at the largest one's exponent, cut 13 bits below it, and these sums to the accumulators in
// float32. Float16 results of unit normals (inner 64 to 4096) are 2.08e-4 from the exact ones in the 2-norm, which is their own rounding; exact products
// would take the 16-bit instruction, at half the rate.
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

// Values that are the same for the whole workgroup, kept in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <int N> struct Const { static constexpr int value = N; };

// The sums' way out: four columns of a row a lane, the same four for all rows, so what belongs to columns is loaded once.
template <class O, bool GATED> struct Columns
{
    float bias[4], biasUp[4], scale[4], scaleUp[4];
    __device__ __forceinline__ void init(const Finish& f, int64_t n)
    {
        const int64_t left = f.cols - n;
        #pragma unroll
        for (int i = 0; i < 4; i++) { bias[i] = biasUp[i] = 0.f; scale[i] = scaleUp[i] = 1.f; }
        if (left <= 0) return;
        if (f.bias)
        {
            quad_load(static_cast<const O*>(f.bias) + n, left, f.vec, bias);
            if (GATED) quad_load(static_cast<const O*>(f.bias) + f.cols + n, left, f.vec, biasUp);
        }
        if (f.qs)
        {
            quad_load(f.ps + n, left, false, scale);
            if (GATED) quad_load(f.ps + f.cols + n, left, false, scaleUp);
        }
    }
    __device__ __forceinline__ void apply(const Finish& f, int64_t m, float* v, float* u) const
    {
        if (f.qs)
        {
            const RowScale s(f.qs[m]);
            #pragma unroll
            for (int i = 0; i < 4; i++)
            {
                v[i] = s.of(v[i], scale[i]);
                if (GATED) u[i] = s.of(u[i], scaleUp[i]);
            }
        }
        #pragma unroll
        for (int i = 0; i < 4; i++)
        {
            v[i] += bias[i];
            if (GATED) u[i] += biasUp[i];
        }
    }
};

// T operands, O results; WR x WC waves, each with a (BM / WR) x (BN / WC) part of the tile.
template <class T, class O, int BM, int BN, int WR, int WC, int PL, int QL, bool GATED, bool DIRECT>
__global__ __launch_bounds__(WR * WC * 64) void token_gemm_kernel(TokenArgs a)
{
    constexpr int kThreads = WR * WC * 64, MT = BM / WR / 32, NT = BN / WC / 32;
    static_assert((NT == 2 || NT == 4) && MT >= 1 && MT <= 4, "a wave owns 64 or 128 columns");
    constexpr int kFrags = sizeof(T) == 1 ? 2 : 1, kGroups = 4 / kFrags;    // 16-byte fragments a product takes; groups of products a step
    constexpr uint32_t kBufBytes = (uint32_t)(BM + BN) * 128u;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * kBufBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WC, wc = wave % WC;

    // Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, in bands of four tile rows, so that the tiles its 32 compute
    // units work on at a time share operand rows in its L2.
    const uint32_t total = gridDim.x;
    uint32_t id = blockIdx.x;
    {
        const uint32_t each = total / 8, more = total % 8, x = id % 8;
        id = x * each + (x < more ? x : more) + id / 8;
    }
    const int split = uniform((int)(id / (uint32_t)a.tiles));
    id -= (uint32_t)split * (uint32_t)a.tiles;
    const uint32_t band = 4 * (uint32_t)a.tilesN, g = id / band, inBand = id - g * band;
    const uint32_t high = min(4u, (uint32_t)a.tilesM - g * 4), across = inBand / high;
    const int64_t m0 = (int64_t)uniform((int)(g * 4 + inBand - across * high)) * BM, n0 = (int64_t)uniform((int)across) * (GATED ? BN / 2 : BN);

    Loader<T, BN, PL, kThreads, GATED, DIRECT> pl;
    Loader<T, BM, QL, kThreads, false, DIRECT> ql;
    pl.init(a.p, a.ldp, a.inner, n0, a.pStored, tid, a.near);
    ql.init(a.q, a.ldq, a.inner, m0, a.qStored, tid, a.near);
    Fragments<T, BN, PL> pf;
    Fragments<T, BM, QL> qf;
    pf.init(lane, wc * NT * 32);
    qf.init(lane, wr * MT * 32);

    f32x16 acc[MT][NT];
    #pragma unroll
    for (int i = 0; i < MT; i++)
        #pragma unroll
        for (int j = 0; j < NT; j++)
            #pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    const uint32_t lds = (uint32_t)(uintptr_t)smem;
    const int s0 = split * a.stepsPerSplit, s1 = min(s0 + a.stepsPerSplit, a.steps);

    // The fragments of a group of products are read while the group before it is multiplied, over the step's end too: once the last group's
    // fragments are in registers the step's buffer is free, every wave meets at the barrier, the next step's tiles (on their way for a whole
    // step) are there, and the tiles of the step after that start into the freed buffer.
    uint4 pv[2][kFrags][NT], qv[2][kFrags][MT];
    auto fetch = [&](uint32_t pt, int group, int set)
    {
        #pragma unroll
        for (int f = 0; f < kFrags; f++)
        {
            #pragma unroll
            for (int j = 0; j < NT; j++) pv[set][f][j] = pf.read(pt, 0, j, group * kFrags + f);
            #pragma unroll
            for (int i = 0; i < MT; i++) qv[set][f][i] = qf.read(pt, BN * 128, i, group * kFrags + f);
        }
    };
    // between: called behind every product with its number, for work that the matrix unit's time covers
    auto multiply = [&](int set, auto between)
    {
        #pragma unroll
        for (int i = 0; i < MT; i++)
            #pragma unroll
            for (int j = 0; j < NT; j++)
            {
                if constexpr (kFrags == 2) acc[i][j] = product8(pv[set][0][j], pv[set][1][j], qv[set][0][i], qv[set][1][i], acc[i][j]);
                else acc[i][j] = Product<T>::run(pv[set][0][j], qv[set][0][i], acc[i][j]);
                between(i * NT + j);
            }
    };
    auto start = [&](int half, int step, uint32_t pt) { pl.begin(half, step, pt, wave); ql.begin(half, step, pt + BN * 128, wave); };
    auto meet = [&] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (s0 < s1)
    {
        start(0, s0, lds);
        start(1, s0, lds);
    }
    // 8 bit: whether the plain product of two scales will do for all of this wave's results; asked for here, while the first step's tiles travel. The results'
    // quick ways out take it then (norm, gated unit, 8-bit rows, projection, 8192 x 4096 -> 8192: two factors there cost 16 us of 786, this test 10 of 792).
    bool plainScales = true;
    if (sizeof(T) == 1 && !a.part)
    {
        constexpr int kCols = NT * 32 / (GATED ? 2 : 1);
        bool plain = true;
        #pragma unroll
        for (int i = 0; i < MT * 32; i += 64)
        {
            const int64_t m = m0 + wr * MT * 32 + i + lane;
            if (i + lane < MT * 32 && m < a.fin.rows) plain = plain && plain_scale(a.fin.qs[m]);
        }
        #pragma unroll
        for (int i = 0; i < kCols; i += 64)
        {
            const int64_t n = n0 + wc * kCols + i + lane;
            if (i + lane >= kCols || n >= a.fin.cols) continue;
            plain = plain && plain_scale(a.fin.ps[n]);
            if (GATED) plain = plain && plain_scale(a.fin.ps[a.fin.cols + n]);
        }
        plainScales = __all(plain);
    }
    if (s0 < s1)
    {
        pl.end(lds);
        ql.end(lds + BN * 128);
        meet();
        if (s0 + 1 < s1) start(0, s0 + 1, lds + kBufBytes);
        fetch(lds, 0, 0);
    }
    int s = s0;
    if (DIRECT)
    {
        // Steps whose second next one is whole: no branches. The sends for a step lie between the products of the group behind the barrier that
        // frees its buffer and of the group after that, one for two products: one for each costs 16-bit products 11 % (8192^3: 805 -> 893 us). The
        // 8-bit step has two groups of products twice as long, all its sends lie in the first of them and have a whole step to arrive (8192 x 4096
        // -> 4096: 133 -> 121 us).
        auto spread = [&](int k, int half, int step, uint32_t pt)
        {
            constexpr int kPF = decltype(pl)::kFirst, kQF = decltype(ql)::kFirst, kMma = MT * NT;
            const int np = half ? decltype(pl)::kNum - kPF : kPF, all = np + (half ? decltype(ql)::kNum - kQF : kQF);
            #pragma unroll
            for (int i = 0; i < all; i++)
                if (i * kMma / all == k)
                {
                    if (i < np) pl.send(half * kPF + i, step, pt, wave);
                    else ql.send(half * kQF + i - np, step, pt + BN * 128, wave);
                }
            __builtin_amdgcn_sched_barrier(0);
        };
        const int whole = min(s1, (int)(a.inner / (128 / (int)sizeof(T))));
        for (; s + 2 < whole; s++)
        {
            const uint32_t pt = lds + (uint32_t)((s - s0) & 1) * kBufBytes, pn = lds + (uint32_t)((s - s0 + 1) & 1) * kBufBytes;
            __builtin_amdgcn_s_waitcnt(0xc07f);        // lgkmcnt(0): the first group's fragments, asked for a group of products ago
            #pragma unroll
            for (int group = 0; group < kGroups; group++)
            {
                if (group + 1 < kGroups) fetch(pt, group + 1, (group + 1) & 1);
                else
                {
                    meet();
                    fetch(pn, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (group == 0) multiply(0, [&](int k) { spread(k, 1, s + 1, pn); });
                else if (group + 1 == kGroups) multiply(group & 1, [&](int k) { spread(k, 0, s + 2, pt); });
                else multiply(group & 1, [](int) {});
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    for (; s < s1; s++)
    {
        const uint32_t pt = lds + (uint32_t)((s - s0) & 1) * kBufBytes, pn = lds + (uint32_t)((s - s0 + 1) & 1) * kBufBytes;
        if (s + 1 < s1) start(1, s + 1, pn);
        #pragma unroll
        for (int group = 0; group < kGroups; group++)
        {
            if (group + 1 < kGroups) fetch(pt, group + 1, (group + 1) & 1);
            else if (s + 1 < s1)
            {
                pl.end(pn);
                ql.end(pn + BN * 128);
                meet();
                fetch(pn, 0, 0);
                if (s + 2 < s1) start(0, s + 2, pt);
            }
            multiply(group & 1, [](int) {});
        }
    }
    __syncthreads();

    // 64 columns of a wave's sums at a time. A block's lane holds row lane & 31, columns 8 (r / 4) + 4 (lane / 32) + r % 4; read back from LDS
    // (256 bytes a row, 16-byte chunks exchanged by row & 15 against bank conflicts), neighbouring lanes hold neighbouring columns, and whole rows go
    // to memory.
    constexpr uint32_t kOutBytes = MT * 32 * 256;
    static_assert(WR * WC * kOutBytes <= 2 * kBufBytes, "the results leave through the operands' LDS");
    unsigned char* const out = smem + wave * kOutBytes;
    constexpr int kLanes = GATED ? 8 : 16, kRows = 64 / kLanes, kTurns = 32 / kRows;   // lanes a row (four columns each), rows a turn
    const int chunk = lane % kLanes, c = chunk * 4, rowIn = lane / kLanes;
    const Finish& f = a.fin;
    auto exchange = [&](auto half)
    {
        constexpr int h = decltype(half)::value;           // (known at compile time: an index would put the accumulators in memory)
        wave_lds_order();
        #pragma unroll
        for (int i = 0; i < MT; i++)
            #pragma unroll
            for (int j = 0; j < 2; j++)
                #pragma unroll
                for (int k = 0; k < 4; k++)
                    *reinterpret_cast<float4*>(out + (i * 32 + (lane & 31)) * 256 + (((8 * j + 2 * k + (lane >> 5)) ^ (lane & 15)) << 4)) =
                        make_float4(acc[i][2 * h + j][4 * k], acc[i][2 * h + j][4 * k + 1], acc[i][2 * h + j][4 * k + 2], acc[i][2 * h + j][4 * k + 3]);
        wave_lds_order();
    };
    auto sumsOf = [&](int pass, int t, float* v, float* u)
    {
        const int row = t * kRows + rowIn;
        const unsigned char* from = out + (pass * 32 + row) * 256;
        const float4 v4 = *reinterpret_cast<const float4*>(from + ((chunk ^ (row & 15)) << 4));
        v[0] = v4.x; v[1] = v4.y; v[2] = v4.z; v[3] = v4.w;
        if (GATED)
        {
            const float4 u4 = *reinterpret_cast<const float4*>(from + (((chunk + 8) ^ (row & 15)) << 4));
            u[0] = u4.x; u[1] = u4.y; u[2] = u4.z; u[3] = u4.w;
        }
    };
    auto halves = [&](auto work)
    {
        work(Const<0>());
        if constexpr (NT == 4) work(Const<1>());
    };
    auto rowOf = [&](int pass) { return m0 + wr * MT * 32 + pass * 32 + rowIn; };
    auto colOf = [&](int h) { return n0 + (wc * NT / 2 + h) * (GATED ? 32 : 64) + c; };
    Columns<O, GATED> cols;

    if (a.part)
    {
        halves([&](auto h)
        {
            exchange(h);
            #pragma unroll 1
            for (int pass = 0; pass < MT; pass++)
            {
            const int64_t m = rowOf(pass), n = colOf(h.value);
            float* at = a.part + ((int64_t)split * a.qRows + m) * a.ldpart + n;      // (ldpart, or each half of it, is a multiple of four)
            #pragma unroll
            for (int t = 0; t < kTurns; t++)
            {
                float v[4], u[4];
                sumsOf(pass, t, v, u);
                if (m + t * kRows < a.qRows && n < a.pRows)
                {
                    *reinterpret_cast<float4*>(at + t * kRows * a.ldpart) = make_float4(v[0], v[1], v[2], v[3]);
                    if (GATED) *reinterpret_cast<float4*>(at + t * kRows * a.ldpart + a.ldpart / 2) = make_float4(u[0], u[1], u[2], u[3]);
                }
            }
            }
        });
        return;
    }

    // What is used most: nothing in a turn waits for memory, since that would wait for the turn's own stores too (the residual of a pass is asked
    // for before the stores of the pass ahead of it), and little code: each workgroup runs through it once, from a cold instruction cache. Tiles
    // inside the result know no bounds.
    const bool inside = f.vec && m0 + BM <= f.rows && n0 + (GATED ? BN / 2 : BN) <= f.cols;
    auto straight = [&](auto withResidual, auto atEdge)
    {
        constexpr bool kRes = decltype(withResidual)::value != 0, kEdge = decltype(atEdge)::value != 0;
        Quad<O> res[kTurns];
        auto ask = [&](int h, int pass)
        {
            const int64_t m = rowOf(pass), n = colOf(h), left = f.cols - n;
            const O* r = static_cast<const O*>(f.residual) + m * f.ldr + n;
            #pragma unroll
            for (int t = 0; t < kTurns; t++)
            {
                if (!kEdge) res[t] = *reinterpret_cast<const Quad<O>*>(r + t * kRows * f.ldr);
                else if (m + t * kRows < f.rows)
                {
                    if (f.vec && left >= 4) res[t] = *reinterpret_cast<const Quad<O>*>(r + t * kRows * f.ldr);
                    else
                    {
                        #pragma unroll
                        for (int k = 0; k < 4; k++) if (k < left) res[t].v[k] = r[t * kRows * f.ldr + k];
                    }
                }
            }
        };
        if (kRes) ask(0, 0);
        halves([&](auto h)
        {
            const int64_t n = colOf(h.value), left = f.cols - n;
            cols.init(f, n);
            exchange(h);
            #pragma unroll 1
            for (int pass = 0; pass < MT; pass++)
            {
                const int64_t m = rowOf(pass);
                float scale[kTurns];
                if (sizeof(T) == 1)
                {
                    #pragma unroll
                    for (int t = 0; t < kTurns; t++) scale[t] = !kEdge || m + t * kRows < f.rows ? f.qs[m + t * kRows] : 0.f;
                }
                float v[kTurns][4], u[4];
                #pragma unroll
                for (int t = 0; t < kTurns; t++)
                {
                    sumsOf(pass, t, v[t], u);
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                    {
                        if (sizeof(T) == 1) v[t][k] *= scale[t] * cols.scale[k];
                        v[t][k] = (v[t][k] + cols.bias[k]) * f.gain + (kRes ? row_load(res[t].v[k]) : 0.f);
                    }
                }
                if (kRes)
                {
                    if (pass + 1 < MT) ask(h.value, pass + 1);
                    else if (h.value + 1 < NT / 2) ask(h.value + 1, 0);
                }
                O* to = static_cast<O*>(f.out) + m * f.ldo + n;
                #pragma unroll
                for (int t = 0; t < kTurns; t++)
                    if (!kEdge || (m + t * kRows < f.rows && left > 0)) quad_store(to + t * kRows * f.ldo, kEdge ? left : 4, kEdge ? f.vec : true, v[t]);
            }
        });
    };
    auto gate = [&](auto withSlopes, auto atEdge)
    {
        constexpr bool kSlopes = decltype(withSlopes)::value != 0, kEdge = decltype(atEdge)::value != 0;
        halves([&](auto h)
        {
            const int64_t n = colOf(h.value), left = f.cols - n;
            cols.init(f, n);
            exchange(h);
            #pragma unroll 1
            for (int pass = 0; pass < MT; pass++)
            {
                const int64_t m = rowOf(pass);
                float scale[kTurns];
                if (sizeof(T) == 1)
                {
                    #pragma unroll
                    for (int t = 0; t < kTurns; t++) scale[t] = !kEdge || m + t * kRows < f.rows ? f.qs[m + t * kRows] : 0.f;
                }
                const Place<O, 2> at(f, m, n);
                float v[kTurns][4], u[kTurns][4];
                #pragma unroll
                for (int t = 0; t < kTurns; t++) sumsOf(pass, t, v[t], u[t]);
                #pragma unroll
                for (int t = 0; t < kTurns; t++)
                {
                    float act[4], d[4];
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                    {
                        if (sizeof(T) == 1) { v[t][k] *= scale[t] * cols.scale[k]; u[t][k] *= scale[t] * cols.scaleUp[k]; }
                        v[t][k] += cols.bias[k];
                        u[t][k] += cols.biasUp[k];
                    }
                    act4<LVG_ACT_SWISH, sizeof(O) == 2>(LVG_ACT_SWISH, 0.f, v[t], kSlopes, act, d);
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                    {
                        act[k] *= f.gain;               // dh/du
                        d[k] *= u[t][k] * f.gain;       // dh/dg
                        v[t][k] = act[k] * u[t][k];
                    }
                    if (kEdge && (m + t * kRows >= f.rows || left <= 0)) continue;
                    const Place<O, 2> here = at.down(f, t * kRows);
                    if (kSlopes)
                    {
                        here.keep(f, 0, kEdge ? f.vec : true, d);
                        here.keep(f, 1, kEdge ? f.vec : true, act);
                    }
                    if (!kEdge && sizeof(O) == 2 && f.past)
                    {
                        Quad<O> q;
                        #pragma unroll
                        for (int k = 0; k < 4; k++) q.v[k] = from_acc<O>(v[t][k]);
                        quad_past(here.out, q);
                    }
                    else quad_store(here.out, kEdge ? left : 4, kEdge ? f.vec : true, v[t]);
                }
            }
        });
    };
    if constexpr (GATED)
    {
        if (f.act == LVG_ACT_SWISH && plainScales)
        {
            if (f.slopeKind == LVG_SLOPE_SMOOTH) { if (inside) gate(Const<1>(), Const<0>()); else gate(Const<1>(), Const<1>()); }
            else                              { if (inside) gate(Const<0>(), Const<0>()); else gate(Const<0>(), Const<1>()); }
            return;
        }
    }
    else if (f.act == LVG_ACT_LINEAR && f.slopeKind == LVG_SLOPE_NONE && f.clamp < 0.f && plainScales)
    {
        if (f.residual) { if (inside) straight(Const<1>(), Const<0>()); else straight(Const<1>(), Const<1>()); }
        else            { if (inside) straight(Const<0>(), Const<0>()); else straight(Const<0>(), Const<1>()); }
        return;
    }

    // Every other activation (and scales far from one), one turn at a time; a turn's residual is asked for before the turn ahead of it stores.
    halves([&](auto h)
    {
        const int64_t n = colOf(h.value), left = f.cols - n;
        cols.init(f, n);
        exchange(h);
        #pragma unroll 1
        for (int pass = 0; pass < MT; pass++)
        {
            const int64_t m = rowOf(pass);
            const Place<O, GATED ? 2 : 1> at(f, m, n);
            float next[4] = {0.f, 0.f, 0.f, 0.f};
            auto ask = [&](int t)
            {
                if (!GATED && f.residual && m + t * kRows < f.rows && left > 0)
                    quad_load(static_cast<const O*>(f.residual) + (m + t * kRows) * f.ldr + n, left, f.vec, next);
            };
            ask(0);
            #pragma unroll 1
            for (int t = 0; t < kTurns; t++)
            {
                float v[4], u[4], res[4];
                sumsOf(pass, t, v, u);
                #pragma unroll
                for (int k = 0; k < 4; k++) res[k] = next[k];
                if (t + 1 < kTurns) ask(t + 1);
                if (m + t * kRows >= f.rows || left <= 0) continue;
                cols.apply(f, m + t * kRows, v, u);
                finish4<O, GATED>(f, at.down(f, t * kRows), v, u, res);
            }
        }
    });
}

} // namespace

enum { LVG_TILE_256 = 0, LVG_TILE_128 = 1, LVG_TILE_64 = 2 };

// One launcher per operand type and kind of product, each in a file of its own (they are compiled side by side).
enum { LVG_TOKEN_FORWARD = 0, LVG_TOKEN_GATED = 1, LVG_TOKEN_ROW_GRAD = 2, LVG_TOKEN_WEIGHT_GRAD = 3 };
int token_launch_bf16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_f16(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_f32(int form, int tile, bool direct, const TokenArgs& a, hipStream_t s);
int token_launch_8bit(int form, int tile, bool direct, int out_dtype, const TokenArgs& a, hipStream_t s);

namespace {

template <class T, class O, int PL, int QL, bool GATED> int token_launch_form(int tile, bool direct, const TokenArgs& a, hipStream_t s)
{
    const int64_t blocks = (int64_t)a.tiles * a.splits;
    if (blocks > kGridBlocks) { lvg_set_error("token product: %lld workgroups", (long long)blocks); return LVG_ERR_INVALID; }
    const dim3 grid((unsigned)blocks);
    #define LVG_TILE(ID, BM, BN, WR, WC, STAGED) if (tile == ID) { \
        if (direct) hipLaunchKernelGGL((token_gemm_kernel<T, O, BM, BN, WR, WC, PL, QL, GATED, true>), grid, dim3(WR * WC * 64), 0, s, a); \
        else if constexpr (STAGED) hipLaunchKernelGGL((token_gemm_kernel<T, O, BM, BN, WR, WC, PL, QL, GATED, false>), grid, dim3(WR * WC * 64), 0, s, a); \
        else { lvg_set_error("token product: no such kernel"); return LVG_ERR_INVALID; } }
    LVG_TILE(LVG_TILE_256, 256, 256, 2, 2, sizeof(T) != 1)
    LVG_TILE(LVG_TILE_128, 128, 128, 2, 2, true)
    LVG_TILE(LVG_TILE_64, 64, 128, 2, 2, true)
    #undef LVG_TILE
    return lvg_check_launch("token product");
}

} // namespace
