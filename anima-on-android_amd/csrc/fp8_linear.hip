// Linear layer on 8-bit rows: C[M,N] = A[M,K] . W[N,K]^T, A and W in FP8 rows
// (fp8.h), C f32 or bf16.  Rows are padded to whole groups of 128, so K is
// always a multiple of 128 here.
//
// Arithmetic, by the type of C:
//   * bf16: products on the fp8 MFMA with its e8m0 scales (16x16x128 and
//     32x32x64).  Its adder takes eight products at a time, cuts each off at
//     2^-13 of the largest one's power of two, and adds the eights in f32:
//     measured 1.5e-5 of the result on normal values, whatever K, where bf16 itself
//     rounds by 1.7e-3;
//   * f32: elements are decoded to bf16, scale included, which holds them exactly,
//     and multiplied on the bf16 MFMA, half as fast, whose sums are f32 throughout.
#include "fp8.h"
#include "fp8_plan.h"

#include <algorithm>
#include <type_traits>

namespace anima_hip {
namespace {

using namespace fp8;
using namespace fp8_plan;
using flash_tile::acc_row;
using flash_tile::dma16s;
using flash_tile::dma4s;
using flash_tile::f32x16;
using flash_tile::mfma_bf16;
using flash_tile::ring_barrier;
using flash_tile::u16;

struct LinArgs {
    const uint8_t *a, *as, *w, *ws;
    void *c;
    float *part;  // split K: f32 planes [splits][M][N]
    int64_t ldc;
    int M, N, groups, sg;  // sg: scale bytes of a row
    int tiles_m, tiles_n, splits, per_split;  // staged: tiles, and splits of K by groups
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Waits until the fp8 MFMAs before it have written their results.  The compiler's
// own wait before a vector instruction reads them is that of shorter MFMAs (a
// 32x32x64 product of fp8 takes 16 passes, and it waits for 8: the last registers were
// read before they were written), so every reader comes behind one of these, 32 wait
// states, in the block of the MFMAs.
__device__ __forceinline__ void mfma_drain()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight codes as bf16, times their scale.
__device__ __forceinline__ bf16x8 decode8(unsigned lo, unsigned hi, float scale)
{
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
    return __builtin_bit_cast(bf16x8, v);
}

// Two 16-byte pieces of a row as one operand of the fp8 MFMA.
__device__ __forceinline__ i32x8 whole(const u32x4 &x, const u32x4 &y)
{
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Four consecutive columns of C from nn on.
__device__ __forceinline__ void store4(float *row, int nn, int N, f32x4 v)
{
    if (nn + 4 <= N) {
        *reinterpret_cast<any_f32x4 *>(row + nn) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (nn + r < N)
            row[nn + r] = v[r];
}

__device__ __forceinline__ void store4(uint16_t *row, int nn, int N, f32x4 v)
{
    const u32x2 b = {bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    if (nn + 4 <= N) {
        *reinterpret_cast<any_u32x2 *>(row + nn) = b;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (nn + r < N)
            row[nn + r] = uint16_t(b[r >> 1] >> (16 * (r & 1)));
}

// ------------------------------------------------------------- few rows

// A workgroup takes 16 weight rows and 16 rows of A; its waves share the groups of K,
// kDepth of them on their way at once, and both operands go from memory to registers to the
// MFMA.  Lane (n, g) holds bytes 16 g and 64 + 16 g on of row n's 128: the products' order
// within a group is free as long as both operands have the same.
// For small products, bound by latency: 1 x 2048 x 2048 takes 4.1 us.  Its loads, 64 bytes
// of each of 16 rows, keep less on its way than whole lines by DMA do, so long sums and
// large weights go through the tiles whatever the rows (1 x 2048 x 8192: 9.9 us here, 8.3
// there; 1 x 131072 x 2048: 50 and 47).

constexpr int kDepth = 4;

template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fp8_few_kernel(LinArgs p)
{
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ f32x4 red[WAVES > 1 ? WAVES * 64 : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const unsigned blocks_m = (unsigned(p.M) + 15) / 16;
    const unsigned strip = blockIdx.x / blocks_m;
    const int row0 = int(strip) * 16, m0 = int(blockIdx.x - strip * blocks_m) * 16;
    const int wrow = min(row0 + n, p.N - 1), arow = min(m0 + n, p.M - 1);

    struct Piece {
        u32x4 w[2], a[2];
        unsigned ws, as;
    };
    auto load = [&](int grp, Piece &x) {
        const uint8_t *w = p.w + (int64_t(wrow) * p.groups + grp) * kGroup + 16 * g;
        const uint8_t *a = p.a + (int64_t(arow) * p.groups + grp) * kGroup + 16 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x.w[h] = *reinterpret_cast<const u32x4 *>(w + 64 * h);
            x.a[h] = *reinterpret_cast<const u32x4 *>(a + 64 * h);
        }
        x.ws = p.ws[int64_t(wrow) * p.sg + grp];
        x.as = p.as[int64_t(arow) * p.sg + grp];
    };
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Piece &x) {
        if constexpr (EXACT) {
            const float ws = scale_of(x.ws), as = scale_of(x.as);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc = mfma16(decode8(x.w[j >> 1][2 * (j & 1)], x.w[j >> 1][2 * (j & 1) + 1], ws),
                             decode8(x.a[j >> 1][2 * (j & 1)], x.a[j >> 1][2 * (j & 1) + 1], as),
                             acc);
        } else {
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                whole(x.w[0], x.w[1]), whole(x.a[0], x.a[1]), acc, 0, 0, 0, int(x.ws), 0,
                int(x.as));
        }
    };
    Piece ring[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (wave + d * WAVES < p.groups)
            load(wave + d * WAVES, ring[d]);
    for (int grp = wave; grp < p.groups; grp += kDepth * WAVES) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int at = grp + d * WAVES;
            if (at >= p.groups)
                break;
            multiply(ring[d]);
            if (at + kDepth * WAVES < p.groups)
                load(at + kDepth * WAVES, ring[d]);
        }
        if constexpr (!EXACT)
            mfma_drain();
    }
    if constexpr (WAVES > 1) {
        // The waves' sums in wave order.
        red[wave * 64 + lane] = acc;
        __syncthreads();
        if (wave > 0)
            return;
        acc = red[lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            acc += red[w * 64 + lane];
    }
    // Lane (n, g): columns 4g .. 4g+3 of row n.
    if (m0 + n < p.M)
        store4(static_cast<T *>(p.c) + int64_t(m0 + n) * p.ldc, row0 + 4 * g, p.N, acc);
}

// --------------------------------------------------------- staged tiles

// Tiles of 32 MB WM rows of A by 32 NB WN rows of W; waves as WM x WN x KS, each 32 MB
// x 32 NB of C on the K steps of its share (KS > 1: the shares are added through
// LDS at the end).  C^T on 32x32 MFMAs, W the first operand, so that a lane's four
// consecutive accumulators are four columns of one row.
//
// Rows of both operands reach LDS by DMA, KC bytes at a time through S stages; 16-byte
// pieces are placed by piece ^ swizzle(row) against bank conflicts.  Their scales
// come in sections of 16 groups, two at a time.  Fragments of a step are read
// while the MFMAs of the step before run; a chunk's first ones under the last step of
// the chunk before, behind the barrier that ends it.
//
// With KS = 1 a workgroup takes several tiles in turn, the next one's first chunks coming
// in while this one's results go out (4608 x 8192 x 2048 in bf16: 82 us, so 76).
//
// Large products are bound by the MFMA at the clock that its power allows: 4608 x 8192 x 2048
// takes 71 to 74 us in bf16, 2.1 PFLOP/s at 1.8 GHz with the MFMA busy 57 % of the cycles, 142
// in f32; 8192 x 8192 x 8192 408, 2.7 PFLOP/s.  A few hundred rows are bound by the copies from
// L2, 64 to 100 bytes a ns and CU (256 x 2048 x 8192: 15 us).
template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int KC>
struct Staged {
    static constexpr bool TURN = KS == 1;
    static constexpr int WAVES = WM * WN * KS, THREADS = WAVES * 64;
    static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
    static constexpr int STEP = sizeof(T) == 4 ? 32 : 64;  // elements of K
    static constexpr int STEPS = KC / STEP, SHARE = STEPS / KS;
    // LDS in bytes: S stages of A and W, then two sections of scales, 16 bytes a row.
    static constexpr int A_BY = BM * KC, STAGE = A_BY + BN * KC;
    static constexpr int ROWS = BM + BN, SCALES = S * STAGE, SECTION = ROWS * 16;
    // 1 KiB windows per chunk, and per wave; a wave without one copies the last again,
    // so that all count the same.
    static constexpr int A_WIN = A_BY / 1024, WIN = STAGE / 1024;
    static constexpr int OPS = (WIN + WAVES - 1) / WAVES;
    // The epilogue's rows, in the last stage: 32 of them by the columns of JB blocks (128
    // bytes or more) per wave at a time.  The shares' sums take all of LDS.
    static constexpr int JB = sizeof(T) == 4 ? 1 : NB;
    static constexpr int OUT_ROW = 32 * JB * int(sizeof(T));
    static constexpr int OUT = TURN ? (S - 1) * STAGE : 0;
    static constexpr int OUT_BY = WAVES / KS * 32 * OUT_ROW;
    static constexpr int RED_BY = (KS - 1) * (WAVES / KS) * MB * NB * 4096;
    static constexpr int USED = SCALES + 2 * SECTION;
    static constexpr int LDS = USED > RED_BY ? USED : RED_BY;
    // Workgroups that a CU holds at once.
    static constexpr int ROOM = LDS <= 81920 && THREADS <= 256 ? 2 : 1;
    static_assert(STEPS % KS == 0 && LDS <= 163840, "160 KiB of LDS");
    static_assert(OUT + OUT_BY <= SCALES, "the epilogue's rows fit the stages");
    static_assert((OUT_ROW & (OUT_ROW - 1)) == 0, "and their pieces are placed by xor");
    static_assert(S >= 2 && (S - 2) * OPS < 64, "counted by vmcnt");
};

// Place of a 16-byte piece of a row of ROW bytes in LDS, so that the 16 rows of a
// ds_read_b128 quarter touch distinct banks.
template <int ROW>
__device__ __forceinline__ int swizzle(int row)
{
    return ROW == 64 ? row >> 2 & 3 : ROW == 128 ? (row & 7) ^ (row >> 3 & 1) : row & 15;
}

// The compiler gives up inlining bodies used several times, and with them the scalar
// registers that the copies' addresses need.
#define INLINED __attribute__((always_inline))

// s_waitcnt vmcnt(N), N < 64.
template <int N>
__device__ __forceinline__ void wait_copies()
{
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
}

template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int KC>
__global__ __launch_bounds__(WM *WN *KS * 64) void fp8_staged_kernel(LinArgs p)
{
    using G = Staged<T, MB, NB, WM, WN, KS, S, KC>;
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int CG = KC / kGroup;  // groups of a chunk
    __shared__ __attribute__((aligned(16))) uint8_t smem[G::LDS];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM % WN, share = wave / (WM * WN);
    const int col = lane & 31, half = lane >> 5;
    constexpr int WROWS = 1024 / KC, PIECES = KC / 16;  // of a window, of a row
    const int64_t pitch = int64_t(p.groups) * kGroup;

    // The tile and split in work, its chunks, and this lane's part of each copy in bytes from the
    // tile's first row; rows past M or N read the last one again (their results are not
    // stored).
    int row0, col0, split, c0, c1;
    const uint8_t *a0, *w0, *as0, *ws0;
    unsigned doff[G::OPS];
    int ddst[G::OPS];
    bool dw[G::OPS];
    auto take = [&](int item) INLINED {
        const int tiles = p.tiles_m * p.tiles_n;
        split = item / tiles;
        const int t = item - split * tiles;
        // Four M tiles by all N tiles at a time, M inside: the 32 CUs of an XCD work
        // on about 4 x 8 tiles.
        const int band = t / (4 * p.tiles_n), in_band = t - band * 4 * p.tiles_n;
        const int bm = min(4, p.tiles_m - 4 * band);
        const int tn = in_band / bm, tm = 4 * band + in_band - tn * bm;
        row0 = tm * G::BM;
        col0 = tn * G::BN;
        c0 = split * p.per_split / CG;
        c1 = min((split + 1) * p.per_split, p.groups) / CG;
        a0 = p.a + row0 * pitch;
        w0 = p.w + col0 * pitch;
        as0 = p.as + int64_t(row0) * p.sg;
        ws0 = p.ws + int64_t(col0) * p.sg;
#pragma unroll
        for (int i = 0; i < G::OPS; ++i) {
            const int w = min(i * G::WAVES + wave, G::WIN - 1);
            dw[i] = w >= G::A_WIN;
            const int r = (dw[i] ? w - G::A_WIN : w) * WROWS + lane / PIECES;
            const int at = dw[i] ? min(col0 + r, p.N - 1) - col0 : min(row0 + r, p.M - 1) - row0;
            doff[i] = unsigned(at * pitch + 16 * (lane % PIECES ^ swizzle<KC>(r)));
            ddst[i] = w * 1024;
        }
    };
    // Part i of `parts` of chunk c's copies.
    auto copies = [&](int c, unsigned stage, int i, int parts) INLINED {
#pragma unroll
        for (int k = G::OPS * i / parts; k < G::OPS * (i + 1) / parts; ++k)
            dma16s((dw[k] ? w0 : a0) + int64_t(c) * KC, doff[k],
                   reinterpret_cast<u16 *>(
                       smem + __builtin_amdgcn_readfirstlane(int(stage) + ddst[k])));
    };
    // Section s of the scales, groups 16 s on: windows of 16 rows by four dwords, so that a
    // row is one request (a dword of each of 64 rows costs 64), past a row's end its
    // last dword again.
    auto scales = [&](int section) INLINED {
        const int s = __builtin_amdgcn_readfirstlane(section);
#pragma unroll
        for (int i = 0; i < (G::ROWS / 16 + G::WAVES - 1) / G::WAVES; ++i) {
            const int w = min(i * G::WAVES + wave, G::ROWS / 16 - 1);
            const bool is_w = w * 16 >= G::BM;
            const int r = w * 16 + lane / 4 - (is_w ? G::BM : 0);
            const int at = is_w ? min(col0 + r, p.N - 1) - col0 : min(row0 + r, p.M - 1) - row0;
            dma4s(is_w ? ws0 : as0, unsigned(at * p.sg + min(16 * s + lane % 4 * 4, p.sg - 4)),
                  reinterpret_cast<u16 *>(smem + __builtin_amdgcn_readfirstlane(
                                                     G::SCALES + (s & 1) * G::SECTION + w * 256)));
        }
    };
    // The first copies of the tile.
    auto start = [&]() INLINED {
        if (c0 >= c1)
            return;
        const int s = c0 * CG / 16;
        scales(s);
        if (16 * (s + 1) < p.groups)
            scales(s + 1);
#pragma unroll
        for (int i = 0; i < S - 1; ++i)
            if (c0 + i < c1)
                copies(c0 + i, i * G::STAGE, 0, 1);
    };
    auto after = [&](unsigned stage) INLINED {
        return stage == (S - 1) * G::STAGE ? 0u : stage + G::STAGE;
    };

    f32x16 acc[MB][NB];
    unsigned sa[MB], sw[NB];  // scales of a chunk from its first group's on
    unsigned ao = 0, wo = 0;  // rows (wm MB) 32 + col and (wn NB) 32 + col of a chunk
    unsigned stage = 0;       // of the chunk in work
    // Chunk c is there, at `stage`, and its scales in na and nw; every wave has left the
    // stage before it.
    auto enter = [&](int c, unsigned (&na)[MB], unsigned (&nw)[NB]) INLINED {
        ring_barrier();
        ao = stage + (wm * 32 * MB + col) * KC;
        wo = stage + G::A_BY + (wn * 32 * NB + col) * KC;
        asm volatile("" : "+v"(ao), "+v"(wo));
        const int g = c * CG, shift = g % 4 * 8;
        const uint8_t *s = smem + G::SCALES + (g / 16 & 1) * G::SECTION + (g % 16 & ~3) + col * 16;
#pragma unroll
        for (int i = 0; i < MB; ++i)
            na[i] = *reinterpret_cast<const unsigned *>(s + (wm * MB + i) * 512) >> shift;
#pragma unroll
        for (int j = 0; j < NB; ++j)
            nw[j] = *reinterpret_cast<const unsigned *>(s + G::BM * 16 + (wn * NB + j) * 512) >>
                    shift;
    };
    // 16 bytes of row col of block b; the swizzle depends on col alone.
    auto piece = [&](unsigned row, int b, int i) INLINED {
        return *reinterpret_cast<const u32x4 *>(smem + row + 32 * b * KC +
                                                16 * (i ^ swizzle<KC>(col)));
    };
    // This wave's steps of a chunk: share * SHARE .. .
    auto step_of = [&](int i) INLINED { return KS == 1 ? i : share * G::SHARE + i; };
    constexpr int LAST = G::SHARE - 1;

    // What follows a chunk: nothing, another, or another and the copies for S chunks on.
    enum { kEnd, kMore, kCopy };
    using End = std::integral_constant<int, kEnd>;
    using More = std::integral_constant<int, kMore>;
    using Copy = std::integral_constant<int, kCopy>;
    // To the next chunk, c: it has landed when at most the S - 2 behind it are on their
    // way.
    auto turn = [&](int c, auto follows, unsigned (&na)[MB], unsigned (&nw)[NB]) INLINED {
        wait_copies<decltype(follows)::value == kCopy ? (S - 2) * G::OPS : 0>();
        stage = after(stage);
        enter(c, na, nw);
    };
    // The stage that copies for S chunks on go to, behind the turn: that of the chunk before.
    auto fill = [&]() INLINED { return stage == 0 ? (S - 1) * G::STAGE : stage - G::STAGE; };

    // All chunks of a tile, chunk c by work(c, what follows); its first copies are on
    // their way, and the stores of the tile before behind them.
    auto product = [&](auto &&begin, auto &&work) INLINED {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[i][j][r] = 0.0f;
        if (c0 >= c1)
            return;
        stage = 0;
        if (!G::TURN && c0 + S - 1 < c1)
            wait_copies<(S - 2) * G::OPS>();
        else
            wait_copies<0>();
        enter(c0, sa, sw);
        if (c0 + S - 1 < c1)
            copies(c0 + S - 1, (S - 1) * G::STAGE, 0, 1);
        begin();
        int c = c0;
        int section = c0 * CG / 16;
        while (c + S < c1) {
            // To the end of the section; the one after next takes its place then.
            const int e = min((section + 1) * 16 / CG, c1 - S);
            for (; c < e; ++c)
                work(c, Copy{});
            ++section;
            if (c + S < c1 && 16 * (section + 1) < p.groups)
                scales(section + 1);
        }
        for (; c + 1 < c1; ++c)
            work(c, More{});
        work(c, End{});
    };

    // A tile's results.
    auto finish = [&](int m0, int n0, int plane_of) INLINED {
        if constexpr (KS > 1) {
            // The shares' sums, in their order.
            f32x4 *red = reinterpret_cast<f32x4 *>(smem);
            constexpr int BLOCKS = WM * WN * MB * NB;
            const int w0i = wave % (WM * WN);
            if (share > 0)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            red[(((share - 1) * BLOCKS + (w0i * MB + i) * NB + j) * 4 + q) * 64 +
                                lane] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                              acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            __syncthreads();
            if (share == 0)
#pragma unroll
                for (int k = 0; k < KS - 1; ++k)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int j = 0; j < NB; ++j)
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const f32x4 v =
                                    red[((k * BLOCKS + (w0i * MB + i) * NB + j) * 4 + q) * 64 +
                                        lane];
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    acc[i][j][4 * q + e] += v[e];
                            }
            __syncthreads();
            if (share > 0)
                return;
        }
        // Lane (col, half): row col of its blocks, columns acc_row(r, half).
        m0 += wm * MB * 32;
        n0 += wn * NB * 32;
        if (p.part) {
            float *plane = p.part + int64_t(plane_of) * p.M * p.N;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int m = m0 + i * 32 + col;
                if (m >= p.M)
                    continue;
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        store4(plane + int64_t(m) * p.N, n0 + 32 * j + acc_row(r, half), p.N,
                               f32x4{acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2],
                                     acc[i][j][r + 3]});
            }
            return;
        }
        // Through LDS, so that rows go out in runs of 32 JB columns; pieces of 16 bytes are
        // placed as in the stages.
        constexpr int JB = G::JB, ROW = G::OUT_ROW;
        // Rows that begin anywhere share cache lines, which must stay for the next store.
        const bool aligned = (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 &&
                             p.ldc % (16 / int(sizeof(T))) == 0;
        constexpr int RUN = ROW / 16, E = 16 / int(sizeof(T));  // pieces of a row, their elements
        uint8_t *so = smem + G::OUT + wave % (WM * WN) * (32 * ROW);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int jb = 0; jb < NB; jb += JB) {
#pragma unroll
                for (int j = 0; j < JB; ++j)
#pragma unroll
                    for (int q = 0; q < 16; q += 4) {
                        const f32x16 &v = acc[i][jb + j];
                        const int at = (32 * j + acc_row(q, half)) * int(sizeof(T));
                        uint8_t *dst = so + col * ROW +
                                       ((at / 16) ^ swizzle<ROW>(col)) * 16 + at % 16;
                        if constexpr (sizeof(T) == 4)
                            *reinterpret_cast<f32x4 *>(dst) =
                                f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
                        else
                            *reinterpret_cast<u32x2 *>(dst) =
                                u32x2{bf16_pair(v[q], v[q + 1]), bf16_pair(v[q + 2], v[q + 3])};
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int q = 0; q < RUN / 2; ++q) {
                    const int f = q * 64 + lane, r = f / RUN, pc = f % RUN;
                    const u32x4 v =
                        *reinterpret_cast<const u32x4 *>(so + r * ROW + (pc ^ swizzle<ROW>(r)) * 16);
                    const int m = m0 + i * 32 + r, nn = n0 + 32 * jb + E * pc;
                    if (m >= p.M)
                        continue;
                    T *dst = static_cast<T *>(p.c) + int64_t(m) * p.ldc + nn;
                    if (nn + E <= p.N) {
                        if (aligned)
                            __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(dst));
                        else
                            *reinterpret_cast<any_u32x4 *>(dst) = v;
                    } else
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (nn + e < p.N) {
                                if constexpr (EXACT)
                                    dst[e] = __uint_as_float(v[e]);
                                else
                                    dst[e] = u16(v[e >> 1] >> (16 * (e & 1)));
                            }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
    };
    // The tiles of this workgroup: XCD x = blockIdx % 8 has a contiguous range of them, and
    // its workgroups take every so many-th.
    auto tiles = [&](auto &&begin, auto &&work) INLINED {
        const unsigned items = unsigned(p.tiles_m * p.tiles_n) * p.splits;
        const unsigned x = blockIdx.x % kXcds, q = items / kXcds, r = items % kXcds;
        const unsigned to = x * q + min(x, r) + q + (x < r ? 1 : 0);
        const unsigned step = (gridDim.x - x + kXcds - 1) / kXcds;
        unsigned item = x * q + min(x, r) + blockIdx.x / kXcds;
        take(__builtin_amdgcn_readfirstlane(int(item)));
        start();
        for (;;) {
            product(begin, work);
            const int m0 = row0, n0 = col0, plane_of = split;
            item += step;
            const bool more = G::TURN && item < to;
            __syncthreads();  // every wave has left the stages
            if (more) {
                take(__builtin_amdgcn_readfirstlane(int(item)));
                start();
            }
            finish(m0, n0, plane_of);
            if (!more)
                return;
        }
    };

    if constexpr (EXACT) {
        // A step is 32 elements: 16 of each half, two bf16 MFMAs.  A fragment's
        // registers are free once it is decoded, and take the next step's then.
        u32x4 ra[MB], rw[NB];
        auto decode2 = [&](const u32x4 &x, unsigned scale, bf16x8 (&v)[2]) INLINED {
            const float f = scale_of(scale & 255u);
            v[0] = decode8(x[0], x[1], f);
            v[1] = decode8(x[2], x[3], f);
        };
        auto begin = [&]() INLINED {
#pragma unroll
            for (int j = 0; j < NB; ++j)
                rw[j] = piece(wo, j, 2 * step_of(0) + half);
#pragma unroll
            for (int i = 0; i < MB; ++i)
                ra[i] = piece(ao, i, 2 * step_of(0) + half);
        };
        tiles(begin, [&](int c, auto follows) INLINED {
            constexpr int F = decltype(follows)::value;
#pragma unroll
            for (int st = 0; st < G::SHARE; ++st) {
                const int byte = step_of(st) / 4 * 8;  // of the step's group
                const int next = step_of(st < LAST ? st + 1 : 0);
                const bool last = st == LAST;
                bf16x8 wv[NB][2], av[MB][2];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    decode2(rw[j], sw[j] >> byte, wv[j]);
                if (last) {
                    // Decoded whole, so that the next chunk's first fragments can come in
                    // under the products.
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        decode2(ra[i], sa[i] >> byte, av[i]);
                    if constexpr (F > kEnd)
                        turn(c + 1, follows, sa, sw);
                }
                if (!last || F > kEnd) {
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        rw[j] = piece(wo, j, 2 * next + half);
                    if (last)
#pragma unroll
                        for (int i = 0; i < MB; ++i)
                            ra[i] = piece(ao, i, 2 * next + half);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    if (!last) {
                        decode2(ra[i], sa[i] >> byte, av[i]);
                        ra[i] = piece(ao, i, 2 * next + half);
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int j = 0; j < NB; ++j)
                            acc[i][j] = mfma_bf16(wv[j][q], av[i][q], acc[i][j]);
                    if (last && F >= kCopy) {
                        copies(c + S, fill(), i, MB);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        });
    } else {
        // A step is 64 elements, 32 of each half, one fp8 MFMA.  The fragments of W
        // have two sets of registers; those of A too in small blocks, and in large ones
        // one, a block of rows' next fragment read behind its last product.
        constexpr bool ONE = MB * NB >= 6;
        constexpr int SETS = ONE ? 1 : 2;
        i32x8 fa[SETS][MB], fw[2][NB];
        auto read = [&](unsigned row, int b, int st) INLINED {
            return whole(piece(row, b, 4 * st + 2 * half), piece(row, b, 4 * st + 2 * half + 1));
        };
        auto begin = [&]() INLINED {
#pragma unroll
            for (int j = 0; j < NB; ++j)
                fw[0][j] = read(wo, j, step_of(0));
#pragma unroll
            for (int i = 0; i < MB; ++i)
                fa[0][i] = read(ao, i, step_of(0));
        };
        tiles(begin, [&](int c, auto follows) INLINED {
            constexpr int F = decltype(follows)::value;
            unsigned na[MB], nw[NB];
#pragma unroll
            for (int st = 0; st < G::SHARE; ++st) {
                const int now = G::SHARE == 1 ? 0 : st & 1, nxt = now ^ 1;
                const int byte = step_of(st) / 2 * 8;  // of the step's group
                const int next = step_of(st < LAST ? st + 1 : 0);
                const bool last = st == LAST, go = !last || F > kEnd;
                auto mfma = [&](int i, int j) INLINED {
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        fw[now][j], fa[ONE ? 0 : now][i], acc[i][j], 0, 0, 0, int(sw[j] >> byte),
                        0, int(sa[i] >> byte));
                };
                if constexpr (ONE) {
                    // Between the products: the turn to the next chunk behind the first one,
                    // then the next fragments, those of A behind their last product, and the
                    // copies, one or two each (in lumps the products wait for them: 192 x
                    // 256 by four waves 88 us, so 76).
                    constexpr int N = MB * NB;
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const int i = k / NB, j = k % NB;
                        mfma(i, j);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (F > kEnd)
                            if (last && k == 0)
                                turn(c + 1, follows, na, nw);
                        if (go && k < NB)
                            fw[nxt][k] = read(wo, k, next);
                        if (last && F >= kCopy)
                            copies(c + S, fill(), k, N);
                        if (go && j == NB - 1)
                            fa[0][i] = read(ao, i, next);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
                    // Small blocks: all of the next step's fragments before its products.
                    if constexpr (F > kEnd)
                        if (last)
                            turn(c + 1, follows, na, nw);
                    if (go) {
#pragma unroll
                        for (int j = 0; j < NB; ++j)
                            fw[nxt][j] = read(wo, j, next);
#pragma unroll
                        for (int i = 0; i < MB; ++i)
                            fa[nxt][i] = read(ao, i, next);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < MB; ++i) {
#pragma unroll
                        for (int j = 0; j < NB; ++j)
                            mfma(i, j);
                        __builtin_amdgcn_sched_barrier(0);
                        if (last && F >= kCopy)
                            copies(c + S, fill(), i, MB);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            if constexpr (F == kEnd)
                mfma_drain();
            else {
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    sa[i] = na[i];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    sw[j] = nw[j];
                if constexpr (G::SHARE % 2 == 1) {
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        fw[0][j] = fw[1][j];
                    if constexpr (!ONE) {
#pragma unroll
                        for (int i = 0; i < MB; ++i)
                            fa[0][i] = fa[1][i];
                    }
                }
            }
        });
    }
}

// C = the planes' sum, in split order (at most kMaxSplits), all loads in flight.
template <typename T>
__global__ __launch_bounds__(256) void fp8_sum_kernel(const float *part, T *c, int64_t ldc, int M,
                                                      int N, int splits)
{
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t plane = int64_t(M) * N;
    if (i >= plane)
        return;
    float x[kMaxSplits];
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s)
        if (s < splits)
            x[s] = part[s * plane + i];
    float sum = x[0];
#pragma unroll
    for (int s = 1; s < kMaxSplits; ++s)
        if (s < splits)
            sum += x[s];
    const int64_t m = i / N;
    T *dst = c + m * ldc + (i - m * N);
    if constexpr (sizeof(T) == 4)
        *dst = sum;
    else
        *dst = __builtin_bit_cast(uint16_t, static_cast<__bf16>(sum));
}

// -------------------------------------------------------------- launches

// Shapes of the staged kernel: MB, NB, WM, WN, KS, S, KC.
#define STAGED_BF16(X) \
    X(0, 4, 4, 2, 2, 1, 2, 128) X(1, 3, 2, 2, 4, 1, 2, 128) X(2, 2, 4, 2, 2, 1, 2, 128) \
    X(3, 2, 2, 2, 2, 1, 2, 128) X(4, 2, 1, 2, 2, 1, 3, 128) X(5, 1, 2, 2, 2, 1, 3, 128) \
    X(6, 1, 1, 2, 2, 1, 4, 128) X(7, 1, 1, 2, 2, 2, 3, 256) X(8, 1, 1, 1, 2, 2, 4, 128) \
    X(9, 1, 1, 1, 2, 4, 3, 256)
#define STAGED_F32(X) \
    X(0, 2, 4, 4, 2, 1, 2, 128) X(1, 3, 2, 2, 4, 1, 2, 128) X(2, 2, 2, 2, 4, 1, 2, 128) \
    X(3, 2, 2, 2, 2, 1, 2, 128) X(4, 1, 2, 2, 2, 1, 3, 128) X(5, 1, 2, 2, 2, 2, 2, 256) \
    X(6, 1, 1, 2, 2, 1, 4, 128) X(7, 1, 1, 2, 2, 2, 3, 256) X(8, 1, 1, 1, 2, 2, 4, 128) \
    X(9, 1, 1, 1, 2, 4, 3, 256)

#define SHAPE_CHECK(table, T, i, mb, nb, wm, wn, ks, s, kc) \
    static_assert(table[i].bm == 32 * mb * wm && table[i].bn == 32 * nb * wn && \
                  table[i].groups == kc / kGroup && \
                  table[i].room == Staged<T, mb, nb, wm, wn, ks, s, kc>::ROOM, "shape table");
#define CHECK_BF16(...) SHAPE_CHECK(kBf16Shapes, uint16_t, __VA_ARGS__)
#define CHECK_F32(...) SHAPE_CHECK(kF32Shapes, float, __VA_ARGS__)
STAGED_BF16(CHECK_BF16)
STAGED_F32(CHECK_F32)

#define STAGED_CASE(i, mb, nb, wm, wn, ks, s, kc)                   \
    case i:                                                         \
        launch_staged<T, mb, nb, wm, wn, ks, s, kc>(p, items, st);  \
        break;

template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int KC>
void launch_staged(const LinArgs &p, int64_t items, hipStream_t st)
{
    using G = Staged<T, MB, NB, WM, WN, KS, S, KC>;
    // As many workgroups as the CUs hold at once, where they take tiles in turn.
    const dim3 grid(unsigned(G::TURN ? std::min<int64_t>(items, 256 * G::ROOM) : items));
    hipLaunchKernelGGL((fp8_staged_kernel<T, MB, NB, WM, WN, KS, S, KC>), grid,
                       dim3(G::THREADS), 0, st, p);
}

template <typename T>
bool run_staged(LinArgs p, const LinPlan &pl, hipStream_t st)
{
    p.tiles_m = pl.tiles_m;
    p.tiles_n = pl.tiles_n;
    p.splits = pl.splits;
    p.per_split = pl.per_split;
    const int64_t items = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;
    if (!launch_fits(items, 512))
        return fail("linear_fp8_dev: too many tiles for one launch");
    if constexpr (sizeof(T) == 2)
        switch (pl.shape) {
            STAGED_BF16(STAGED_CASE)
        }
    else
        switch (pl.shape) {
            STAGED_F32(STAGED_CASE)
        }
    if (!hip_ok(hipGetLastError(), "fp8_staged_kernel launch"))
        return false;
    if (pl.splits == 1)
        return true;
    const int64_t n = int64_t(p.M) * p.N;
    hipLaunchKernelGGL(fp8_sum_kernel<T>, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st,
                       p.part, static_cast<T *>(p.c), p.ldc, p.M, p.N, pl.splits);
    return hip_ok(hipGetLastError(), "fp8_sum_kernel launch");
}

template <typename T>
bool run_few(const LinArgs &p, int waves, hipStream_t st)
{
    const int64_t blocks = (int64_t(p.N) + 15) / 16 * ((int64_t(p.M) + 15) / 16);
    if (!launch_fits(blocks, waves * 64))
        return fail("linear_fp8_dev: too many rows for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    switch (waves) {
    case 1: hipLaunchKernelGGL((fp8_few_kernel<T, 1>), grid, dim3(64), 0, st, p); break;
    case 2: hipLaunchKernelGGL((fp8_few_kernel<T, 2>), grid, dim3(128), 0, st, p); break;
    case 4: hipLaunchKernelGGL((fp8_few_kernel<T, 4>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((fp8_few_kernel<T, 8>), grid, dim3(512), 0, st, p); break;
    }
    return hip_ok(hipGetLastError(), "fp8_few_kernel launch");
}

template <typename T>
bool run_linear(const LinArgs &p, const LinPlan &pl, hipStream_t st)
{
    return pl.staged ? run_staged<T>(p, pl, st) : run_few<T>(p, pl.waves, st);
}

}  // namespace

size_t linear_fp8_scratch_bytes(int M, int N, int K, Mx4Type type)
{
    if (M <= 0 || N <= 0 || K <= 0)
        return 0;
    return size_t(lin_scratch(lin_plan(M, N, int(fp8_groups(K)), type == kMx4F32), M, N));
}

bool launch_linear_fp8(const Fp8Linear &a, void *scratch, size_t scratch_bytes, hipStream_t st)
{
    if (a.M <= 0 || a.N <= 0)
        return true;
    LinArgs p{};
    p.a = a.a;
    p.as = a.a_scales;
    p.w = a.w;
    p.ws = a.w_scales;
    p.c = a.c;
    p.ldc = a.ldc;
    p.M = a.M;
    p.N = a.N;
    p.groups = int(fp8_groups(a.K));
    p.sg = int(fp8_scale_bytes(a.K));
    const LinPlan pl = lin_plan(a.M, a.N, p.groups, a.type == kMx4F32);
    const size_t need = size_t(lin_scratch(pl, a.M, a.N));
    if (need > 0) {
        if (scratch_bytes < need || !scratch)
            return fail("linear_fp8_dev: scratch smaller than anima_hip_linear_fp8_scratch_bytes");
        if (!flash_tile::aligned(scratch, 16))
            return fail("linear_fp8_dev: scratch must be 16-byte aligned");
        p.part = static_cast<float *>(scratch);
    }
    return a.type == kMx4F32 ? run_linear<float>(p, pl, st) : run_linear<uint16_t>(p, pl, st);
}

}  // namespace anima_hip
