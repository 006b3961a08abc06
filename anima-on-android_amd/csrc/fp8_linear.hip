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
using flash_tile::wait_vmcnt;
using flash_tile::xcd_major_block;

struct LinArgs {
    const uint8_t *a, *as, *w, *ws;
    void *c;
    float *part;  // split K: f32 planes [splits][M][N]
    int64_t ldc;
    int M, N, groups, sg;  // sg: scale bytes of a row
    int tiles_m, tiles_n, per_split;  // staged: tiles, and groups of one split
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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

// Four consecutive columns of C from nn on.
__device__ __forceinline__ void store4(float *row, int nn, int N, bool wide, f32x4 v)
{
    if (wide && nn + 4 <= N) {
        *reinterpret_cast<f32x4 *>(row + nn) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (nn + r < N)
            row[nn + r] = v[r];
}

__device__ __forceinline__ void store4(uint16_t *row, int nn, int N, bool wide, f32x4 v)
{
    const u32x2 b = {bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    if (wide && nn + 4 <= N) {
        *reinterpret_cast<u32x2 *>(row + nn) = b;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (nn + r < N)
            row[nn + r] = uint16_t(b[r >> 1] >> (16 * (r & 1)));
}

// ------------------------------------------------------------- few rows

// A workgroup takes 16 weight rows and up to 16 MB rows of A; its waves share the
// groups of K, and both operands go from memory to registers to the MFMA.  Lane (n, g)
// holds bytes 16 g and 64 + 16 g on of row n's 128: the products' order within
// a group is free as long as both operands have the same.
template <typename T, int MB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fp8_few_kernel(LinArgs p)
{
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ f32x4 red[WAVES > 1 ? WAVES * MB * 64 : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const unsigned blocks_m = (unsigned(p.M) + 16 * MB - 1) / (16 * MB);
    const unsigned strip = blockIdx.x / blocks_m;
    const int row0 = int(strip) * 16, m0 = int(blockIdx.x - strip * blocks_m) * (16 * MB);
    const int wrow = min(row0 + n, p.N - 1);
    int arow[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
        arow[i] = min(m0 + 16 * i + n, p.M - 1);

    struct Piece {
        u32x4 w[2], a[MB][2];
        unsigned ws, as[MB];
    };
    auto load = [&](int grp, Piece &x) {
        const uint8_t *w = p.w + (int64_t(wrow) * p.groups + grp) * kGroup + 16 * g;
        x.w[0] = *reinterpret_cast<const u32x4 *>(w);
        x.w[1] = *reinterpret_cast<const u32x4 *>(w + 64);
        x.ws = p.ws[int64_t(wrow) * p.sg + grp];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const uint8_t *a = p.a + (int64_t(arow[i]) * p.groups + grp) * kGroup + 16 * g;
            x.a[i][0] = *reinterpret_cast<const u32x4 *>(a);
            x.a[i][1] = *reinterpret_cast<const u32x4 *>(a + 64);
            x.as[i] = p.as[int64_t(arow[i]) * p.sg + grp];
        }
    };
    f32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
        acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Piece &x) {
        if constexpr (EXACT) {
            const float ws = scale_of(x.ws);
            bf16x8 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = decode8(x.w[j >> 1][2 * (j & 1)], x.w[j >> 1][2 * (j & 1) + 1], ws);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const float as = scale_of(x.as[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i] = mfma16(w[j],
                                    decode8(x.a[i][j >> 1][2 * (j & 1)],
                                            x.a[i][j >> 1][2 * (j & 1) + 1], as),
                                    acc[i]);
            }
        } else {
            i32x8 w;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = int(x.w[j >> 2][j & 3]);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                i32x8 a;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    a[j] = int(x.a[i][j >> 2][j & 3]);
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    w, a, acc[i], 0, 0, 0, int(x.ws), 0, int(x.as[i]));
            }
        }
    };
    Piece cur, next;
    if (wave < p.groups)
        load(wave, cur);
    for (int grp = wave; grp < p.groups; grp += WAVES) {
        if (grp + WAVES < p.groups)
            load(grp + WAVES, next);
        multiply(cur);
        cur = next;
    }
    if constexpr (WAVES > 1) {
        // The waves' sums in wave order.
#pragma unroll
        for (int i = 0; i < MB; ++i)
            red[(wave * MB + i) * 64 + lane] = acc[i];
        __syncthreads();
    }
    const bool wide = (reinterpret_cast<uintptr_t>(p.c) & (4 * sizeof(T) - 1)) == 0 &&
                      p.ldc % 4 == 0;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        if (wave != i % WAVES)
            continue;
        f32x4 sum = acc[i];
        if constexpr (WAVES > 1) {
            sum = red[i * 64 + lane];
#pragma unroll
            for (int w = 1; w < WAVES; ++w)
                sum += red[(w * MB + i) * 64 + lane];
        }
        // Lane (n, g): columns 4g .. 4g+3 of row n.
        const int m = m0 + 16 * i + n;
        if (m < p.M)
            store4(static_cast<T *>(p.c) + int64_t(m) * p.ldc, row0 + 4 * g, p.N, wide, sum);
    }
}

// --------------------------------------------------------- staged tiles

// Tiles of 32 MB WM rows of A by 32 NB WN rows of W; waves as WM x WN x KS, each 32 MB
// x 32 NB of C on the K steps of its share (KS > 1: the shares are added through
// LDS at the end).  C^T on 32x32 MFMAs, W the first operand, so that a lane's four
// consecutive accumulators are four columns of one row.
//
// Rows of both operands, 128 CM bytes at a time, and the dwords of their scales reach
// LDS by DMA through S stages; 16-byte pieces are placed by piece ^ swizzle(row) against
// bank conflicts.  Fragments of a step are read while the MFMAs of the step before run; a
// chunk's first ones under the last step of the chunk before, behind the barrier that
// ends it.
template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int CM>
struct Staged {
    static constexpr int WAVES = WM * WN * KS, THREADS = WAVES * 64;
    static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
    static constexpr int KC = 128 * CM;  // bytes of a row in a chunk
    static constexpr int STEP = sizeof(T) == 4 ? 32 : 64;  // elements of K
    static constexpr int STEPS = KC / STEP, SHARE = STEPS / KS;
    // LDS in bytes: A, W, a dword of scales for each row of both.
    static constexpr int A_BY = BM * KC, W_BY = BN * KC;
    static constexpr int AS_WIN = (BM + 63) / 64, WS_WIN = (BN + 63) / 64;
    static constexpr int STAGE = A_BY + W_BY + (AS_WIN + WS_WIN) * 256;
    // 1 KiB windows (scales: 256 bytes) per chunk, and per wave; a wave without
    // one copies the last again, so that all count the same.
    static constexpr int A_WIN = A_BY / 1024, W_WIN = W_BY / 1024, S_WIN = AS_WIN + WS_WIN;
    static constexpr int A_OPS = (A_WIN + WAVES - 1) / WAVES;
    static constexpr int W_OPS = (W_WIN + WAVES - 1) / WAVES;
    static constexpr int S_OPS = (S_WIN + WAVES - 1) / WAVES;
    static constexpr int OPS = A_OPS + W_OPS + S_OPS;
    // The epilogue's rows of one 32-row block per wave, and the shares' sums.
    static constexpr int PITCH = 32 * NB + 16 / int(sizeof(T));
    static constexpr int OUT_BY = WAVES / KS * 32 * PITCH * int(sizeof(T));
    static constexpr int RED_BY = (KS - 1) * (WAVES / KS) * MB * NB * 4096;
    static constexpr int MAX2 = RED_BY > OUT_BY ? RED_BY : OUT_BY;
    static constexpr int LDS = S * STAGE > MAX2 ? S * STAGE : MAX2;
    static_assert(STEPS % KS == 0 && LDS <= 163840, "160 KiB of LDS");
    static_assert(S >= 2 && (S - 2) * OPS < 16, "counted by vmcnt");
};

// Place of piece `i` of a staged row, so that the 16 rows of a ds_read_b128 quarter
// touch distinct banks.
template <int CM>
__device__ __forceinline__ int swizzle(int row)
{
    return CM == 1 ? (row & 7) ^ (row >> 3 & 1) : row & 15;
}

template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int CM>
__global__ __launch_bounds__(WM *WN *KS * 64) void fp8_staged_kernel(LinArgs p)
{
    using G = Staged<T, MB, NB, WM, WN, KS, S, CM>;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[G::LDS];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM % WN, share = wave / (WM * WN);
    const int col = lane & 31, half = lane >> 5;
    const int tiles = p.tiles_m * p.tiles_n;
    const int blk = xcd_major_block();
    const int split = blk / tiles, t = blk - split * tiles;
    // Four M tiles by all N tiles at a time, M inside: the 32 CUs of an XCD work
    // on about 4 x 8 tiles.
    const int band = t / (4 * p.tiles_n), in_band = t - band * 4 * p.tiles_n;
    const int bm = min(4, p.tiles_m - 4 * band);
    const int tn = in_band / bm, tm = 4 * band + in_band - tn * bm;
    const int row0 = tm * G::BM, col0 = tn * G::BN;
    // Chunks of this split.
    const int c0 = split * (p.per_split / CM), c1 = min(c0 + p.per_split / CM, p.groups / CM);

    // This lane's part of each copy, in bytes from the tile's first row; rows past
    // M or N read the last one again (their results are not stored).
    constexpr int ROWS = 8 / CM, PIECES = 8 * CM;  // of a window, of a row
    const int64_t pitch = int64_t(p.groups) * kGroup;
    unsigned aoff[G::A_OPS], woff[G::W_OPS], soff[G::S_OPS];
    int adst[G::A_OPS], wdst[G::W_OPS], sdst[G::S_OPS];
    bool swin[G::S_OPS];  // scales of W
#pragma unroll
    for (int i = 0; i < G::A_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::A_WIN - 1);
        const int r = w * ROWS + lane / PIECES;
        aoff[i] = unsigned((min(row0 + r, p.M - 1) - row0) * pitch +
                           16 * (lane % PIECES ^ swizzle<CM>(r)));
        adst[i] = w * 1024;
    }
#pragma unroll
    for (int i = 0; i < G::W_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::W_WIN - 1);
        const int r = w * ROWS + lane / PIECES;
        woff[i] = unsigned((min(col0 + r, p.N - 1) - col0) * pitch +
                           16 * (lane % PIECES ^ swizzle<CM>(r)));
        wdst[i] = G::A_BY + w * 1024;
    }
#pragma unroll
    for (int i = 0; i < G::S_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::S_WIN - 1);
        swin[i] = w >= G::AS_WIN;
        const int r = (swin[i] ? w - G::AS_WIN : w) * 64 + lane;
        soff[i] = unsigned((swin[i] ? min(col0 + r, p.N - 1) - col0 : min(row0 + r, p.M - 1) - row0) *
                           p.sg);
        sdst[i] = G::A_BY + G::W_BY + w * 256;
    }
    const uint8_t *a0 = p.a + row0 * pitch, *w0 = p.w + col0 * pitch;
    const uint8_t *as0 = p.as + int64_t(row0) * p.sg, *ws0 = p.ws + int64_t(col0) * p.sg;
    auto dma = [&](int c, int stage) {
        uint8_t *dst = smem + stage * G::STAGE;
#pragma unroll
        for (int i = 0; i < G::A_OPS; ++i)
            dma16s(a0 + int64_t(c) * G::KC, aoff[i], reinterpret_cast<u16 *>(dst + adst[i]));
#pragma unroll
        for (int i = 0; i < G::W_OPS; ++i)
            dma16s(w0 + int64_t(c) * G::KC, woff[i], reinterpret_cast<u16 *>(dst + wdst[i]));
        // The scales of the four groups that the chunk is among.
#pragma unroll
        for (int i = 0; i < G::S_OPS; ++i)
            dma4s((swin[i] ? ws0 : as0) + (c * CM & ~3), soff[i],
                  reinterpret_cast<u16 *>(dst + sdst[i]));
    };

    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[i][j][r] = 0.0f;

    unsigned sa[MB], sw[NB];  // scales of a chunk from its first group's on
    unsigned ao = 0, wo = 0;  // rows (wm MB) 32 + col and (wn NB) 32 + col of a chunk
    // Chunk c's scales go to na and nw.
    auto enter = [&](int c, unsigned (&na)[MB], unsigned (&nw)[NB]) {
        // Chunk c has landed when at most the S - 2 behind it are on their way.
        if (c + S - 2 < c1)
            wait_vmcnt<(S - 2) * G::OPS>();
        else
            wait_vmcnt<0>();
        ring_barrier();  // for every wave; and all have left the stage before it
        if (c + S - 1 < c1)
            dma(c + S - 1, (c + S - 1 - c0) % S);
        const unsigned base = (c - c0) % S * G::STAGE;
        ao = base + (wm * 32 * MB + col) * G::KC;
        wo = base + G::A_BY + (wn * 32 * NB + col) * G::KC;
        asm volatile("" : "+v"(ao), "+v"(wo));
        const unsigned *s = reinterpret_cast<const unsigned *>(smem + base + G::A_BY + G::W_BY);
        const int shift = c * CM % 4 * 8;
#pragma unroll
        for (int i = 0; i < MB; ++i)
            na[i] = s[(wm * MB + i) * 32 + col] >> shift;
#pragma unroll
        for (int j = 0; j < NB; ++j)
            nw[j] = s[G::AS_WIN * 64 + (wn * NB + j) * 32 + col] >> shift;
    };
    // 16 bytes of row col of block b; the swizzle depends on col alone.
    auto piece = [&](unsigned row, int b, int i) {
        return *reinterpret_cast<const u32x4 *>(smem + row + 32 * b * G::KC +
                                                16 * (i ^ swizzle<CM>(col)));
    };
    // This wave's steps of a chunk: share * SHARE .. .
    auto step_of = [&](int i) { return KS == 1 ? i : share * G::SHARE + i; };
    constexpr int LAST = G::SHARE - 1;
    if (c0 < c1) {
#pragma unroll
        for (int i = 0; i < S - 1; ++i)
            if (c0 + i < c1)
                dma(c0 + i, i);
        enter(c0, sa, sw);
    }

    if constexpr (EXACT) {
        // A step is 32 elements: 16 of each half, two bf16 MFMAs.  A fragment's
        // registers are free once it is decoded, and take the next step's then.
        u32x4 ra[MB], rw[NB];
        auto decode2 = [&](const u32x4 &x, unsigned scale, bf16x8 (&v)[2]) {
            const float f = scale_of(scale & 255u);
            v[0] = decode8(x[0], x[1], f);
            v[1] = decode8(x[2], x[3], f);
        };
        if (c0 < c1) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
                rw[j] = piece(wo, j, 2 * step_of(0) + half);
#pragma unroll
            for (int i = 0; i < MB; ++i)
                ra[i] = piece(ao, i, 2 * step_of(0) + half);
        }
        for (int c = c0; c < c1; ++c) {
#pragma unroll
            for (int st = 0; st < G::SHARE; ++st) {
                const int byte = step_of(st) / 4 * 8;  // of the step's group
                const int next = step_of(st < LAST ? st + 1 : 0);
                bf16x8 wv[NB][2];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    decode2(rw[j], sw[j] >> byte, wv[j]);
                if (st < LAST) {
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        rw[j] = piece(wo, j, 2 * next + half);
#pragma unroll
                    for (int i = 0; i < MB; ++i) {
                        bf16x8 av[2];
                        decode2(ra[i], sa[i] >> byte, av);
                        ra[i] = piece(ao, i, 2 * next + half);
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int j = 0; j < NB; ++j)
                                acc[i][j] = mfma_bf16(wv[j][q], av[q], acc[i][j]);
                    }
                    continue;
                }
                // The chunk's last step is decoded whole, so that the next chunk's first
                // fragments can come in under its products (past the last chunk: its own
                // first ones again, which nothing uses).
                bf16x8 av[MB][2];
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    decode2(ra[i], sa[i] >> byte, av[i]);
                if (c + 1 < c1)
                    enter(c + 1, sa, sw);
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    rw[j] = piece(wo, j, 2 * next + half);
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    ra[i] = piece(ao, i, 2 * next + half);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int j = 0; j < NB; ++j)
                            acc[i][j] = mfma_bf16(wv[j][q], av[i][q], acc[i][j]);
            }
        }
    } else {
        // A step is 64 elements, 32 of each half, one fp8 MFMA.  The fragments of W
        // have two sets of registers; those of A too in small blocks, and in large ones
        // one, a block of rows' next fragment read behind its last product.
        constexpr bool ONE = MB * NB >= 8;
        constexpr int SETS = ONE ? 1 : 2;
        i32x8 fa[SETS][MB], fw[2][NB];
        auto read = [&](unsigned row, int b, int st) {
            const u32x4 x = piece(row, b, 4 * st + 2 * half);
            const u32x4 y = piece(row, b, 4 * st + 2 * half + 1);
            return __builtin_bit_cast(i32x8,
                                      __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        if (c0 < c1) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
                fw[0][j] = read(wo, j, step_of(0));
#pragma unroll
            for (int i = 0; i < MB; ++i)
                fa[0][i] = read(ao, i, step_of(0));
        }
        for (int c = c0; c < c1; ++c) {
#pragma unroll
            for (int st = 0; st < G::SHARE; ++st) {
                const int now = G::SHARE == 1 ? 0 : st & 1, nxt = now ^ 1;
                const int na_set = ONE ? 0 : nxt, a_set = ONE ? 0 : now;
                const int byte = step_of(st) / 2 * 8;  // of the step's group
                const int next = step_of(st < LAST ? st + 1 : 0);
                // Past the last chunk: its own first step again, which nothing uses.
                unsigned na[MB], nw[NB];
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    na[i] = sa[i];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    nw[j] = sw[j];
                if (st == LAST && c + 1 < c1)
                    enter(c + 1, na, nw);
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    fw[nxt][j] = read(wo, j, next);
                if constexpr (!ONE) {
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        fa[na_set][i] = read(ao, i, next);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MB; ++i) {
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                            fw[now][j], fa[a_set][i], acc[i][j], 0, 0, 0, int(sw[j] >> byte), 0,
                            int(sa[i] >> byte));
                    if constexpr (ONE) {
                        fa[0][i] = read(ao, i, next);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (st == LAST) {
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        sa[i] = na[i];
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        sw[j] = nw[j];
                }
                if (G::SHARE % 2 == 1 && st == LAST) {
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        fw[0][j] = fw[nxt][j];
                    if constexpr (!ONE) {
#pragma unroll
                        for (int i = 0; i < MB; ++i)
                            fa[0][i] = fa[na_set][i];
                    }
                }
            }
        }
    }

    __syncthreads();
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
                        red[(((share - 1) * BLOCKS + (w0i * MB + i) * NB + j) * 4 + q) * 64 + lane] =
                            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                                  acc[i][j][4 * q + 3]};
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
                                red[((k * BLOCKS + (w0i * MB + i) * NB + j) * 4 + q) * 64 + lane];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[i][j][4 * q + e] += v[e];
                        }
        __syncthreads();
        if (share > 0)
            return;
    }

    // Lane (col, half): row col of its blocks, columns acc_row(r, half).
    const int n0 = col0 + wn * 32 * NB;
    if (p.part) {
        float *plane = p.part + int64_t(split) * p.M * p.N;
        const bool wide = p.N % 4 == 0;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int m = row0 + (wm * MB + i) * 32 + col;
            if (m >= p.M)
                continue;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    store4(plane + int64_t(m) * p.N, n0 + 32 * j + acc_row(r, half), p.N, wide,
                           f32x4{acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2],
                                 acc[i][j][r + 3]});
        }
        return;
    }
    // Through LDS, so that rows go out in runs of 32 NB columns.
    T *so = reinterpret_cast<T *>(smem) + (wave % (WM * WN)) * 32 * G::PITCH;
    constexpr int E = 16 / int(sizeof(T));  // elements of a 16-byte piece
    constexpr int OUT = 32 * NB / E;        // pieces of a row
    const bool wide = (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.ldc % E == 0 &&
                      n0 + 32 * NB <= p.N;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                store4(so + col * G::PITCH, 32 * j + acc_row(r, half), 32 * NB, true,
                       f32x4{acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]});
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < OUT / 2; ++q) {
            const int f = q * 64 + lane, r = f / OUT, piece = f % OUT;
            const int m = row0 + (wm * MB + i) * 32 + r;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(so + r * G::PITCH + E * piece);
            if (m >= p.M)
                continue;
            const int nn = n0 + E * piece;
            T *dst = static_cast<T *>(p.c) + int64_t(m) * p.ldc + nn;
            if (wide)
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(dst));
            else
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

// Shapes of the staged kernel, MB, NB, WM, WN, KS, S, and of the same with two groups
// at once.
#define STAGED_BF16(X, cm) \
    X(cm, 0, 4, 4, 2, 2, 1, 2) X(cm, 1, 3, 4, 2, 2, 1, 2) X(cm, 2, 2, 4, 2, 2, 1, 3) \
    X(cm, 3, 2, 2, 2, 2, 1, 3) X(cm, 4, 1, 2, 2, 2, 1, 3) X(cm, 5, 1, 1, 2, 2, 1, 4) \
    X(cm, 6, 1, 1, 1, 2, 2, 4)
#define PAIRED_BF16(X, cm) \
    X(cm, 4, 1, 2, 2, 2, 2, 2) X(cm, 5, 1, 1, 2, 2, 2, 3) X(cm, 6, 1, 1, 1, 2, 4, 3)
#define STAGED_F32(X, cm) \
    X(cm, 0, 2, 4, 4, 2, 1, 2) X(cm, 1, 1, 4, 4, 2, 1, 3) X(cm, 2, 2, 2, 2, 2, 1, 3) \
    X(cm, 3, 1, 2, 2, 2, 1, 3) X(cm, 4, 1, 1, 2, 2, 1, 4) X(cm, 5, 1, 1, 1, 2, 2, 4)
#define PAIRED_F32(X, cm) \
    X(cm, 3, 1, 2, 2, 2, 2, 2) X(cm, 4, 1, 1, 2, 2, 2, 3) X(cm, 5, 1, 1, 1, 2, 4, 3)

#define SHAPE_CHECK(table, i, mb, nb, wm, wn, cm) \
    static_assert(table[i].bm == 32 * mb * wm && table[i].bn == 32 * nb * wn && \
                  (cm == 1 || table[i].pairs), "shape table");
#define CHECK_BF16(cm, i, mb, nb, wm, wn, ks, s) SHAPE_CHECK(kBf16Shapes, i, mb, nb, wm, wn, cm)
#define CHECK_F32(cm, i, mb, nb, wm, wn, ks, s) SHAPE_CHECK(kF32Shapes, i, mb, nb, wm, wn, cm)
STAGED_BF16(CHECK_BF16, 1)
PAIRED_BF16(CHECK_BF16, 2)
STAGED_F32(CHECK_F32, 1)
PAIRED_F32(CHECK_F32, 2)

constexpr int kPairs = 16;  // beside a shape's number: two groups at once
#define STAGED_CASE(cm, i, mb, nb, wm, wn, ks, s)                                                \
    case i + (cm == 2 ? kPairs : 0):                                                             \
        if (!launch_fits(blocks, wm * wn * ks * 64))                                             \
            return fail("linear_fp8_dev: too many tiles for one launch");                        \
        hipLaunchKernelGGL((fp8_staged_kernel<T, mb, nb, wm, wn, ks, s, cm>),                    \
                           dim3(unsigned(blocks)), dim3(wm * wn * ks * 64), 0, st, p);           \
        break;

template <typename T>
bool run_staged(LinArgs p, const LinPlan &pl, hipStream_t st)
{
    p.tiles_m = pl.tiles_m;
    p.tiles_n = pl.tiles_n;
    p.per_split = pl.per_split;
    const int64_t blocks = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;
    const int shape = pl.shape + (pl.pairs ? kPairs : 0);
    if constexpr (sizeof(T) == 2) {
        switch (shape) {
            STAGED_BF16(STAGED_CASE, 1)
            PAIRED_BF16(STAGED_CASE, 2)
        }
    } else {
        switch (shape) {
            STAGED_F32(STAGED_CASE, 1)
            PAIRED_F32(STAGED_CASE, 2)
        }
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

template <typename T, int MB>
bool run_few(const LinArgs &p, int waves, hipStream_t st)
{
    const int64_t strips = (p.N + 15) / 16, blocks_m = (p.M + 16 * MB - 1) / (16 * MB);
    if (!launch_fits(strips * blocks_m, waves * 64))
        return fail("linear_fp8_dev: too many rows for one launch");
    // Blocks of A rows inside: those of one strip read its weights at about the same time.
    const dim3 grid(unsigned(strips * blocks_m));
    switch (waves) {
    case 1: hipLaunchKernelGGL((fp8_few_kernel<T, MB, 1>), grid, dim3(64), 0, st, p); break;
    case 2: hipLaunchKernelGGL((fp8_few_kernel<T, MB, 2>), grid, dim3(128), 0, st, p); break;
    case 4: hipLaunchKernelGGL((fp8_few_kernel<T, MB, 4>), grid, dim3(256), 0, st, p); break;
    case 8: hipLaunchKernelGGL((fp8_few_kernel<T, MB, 8>), grid, dim3(512), 0, st, p); break;
    default: hipLaunchKernelGGL((fp8_few_kernel<T, MB, 16>), grid, dim3(1024), 0, st, p); break;
    }
    return hip_ok(hipGetLastError(), "fp8_few_kernel launch");
}

template <typename T>
bool run_linear(const LinArgs &p, const LinPlan &pl, hipStream_t st)
{
    if (pl.staged)
        return run_staged<T>(p, pl, st);
    return pl.blocks == 1   ? run_few<T, 1>(p, pl.waves, st)
           : pl.blocks == 2 ? run_few<T, 2>(p, pl.waves, st)
                            : run_few<T, 4>(p, pl.waves, st);
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
