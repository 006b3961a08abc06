// Linear layer with 4-bit weights: C[M,N] = A[M,K] . W[N,K]^T, W in MX4 rows
// (mx4.h), A and C both f32 or both bf16.
//
// Arithmetic: every MX4 weight is a bf16 number, so W enters the bf16 MFMA
// unrounded.  bf16 activations enter as they are; f32 activations as three
// bf16 terms whose sum is the f32 value (terms2), three MFMAs per product.
// Sums are f32, and C is rounded once, to its own type.
//
// Two kernels:
//   * few rows (M <= 16), bound by the one pass over the codes (17/32 byte per
//     weight) or, below about 8 MiB of codes, by latency: a workgroup takes 16
//     weight rows, its waves share K in blocks of 128, and the weights go from
//     memory to registers to the MFMA without touching LDS;
//   * tiles (M > 16), bound by the MFMA at large M: A (as terms) and the decoded
//     weights staged in LDS, two stages, split over K across workgroups where
//     the tiles alone would leave CUs idle.
#include "mx4.h"

#include <algorithm>

namespace anima_hip {
namespace {

using namespace flash_tile;
using mx4::decode8;
using mx4::mfma16;
using mx4::scale_of;
using mx4::terms2;
using mx4::u32x2;

// bf16 terms of an activation: f32 takes three, bf16 is its own.
template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;

// Eight elements of a row from k0 as packed bf16 terms; zero past K.
template <bool VEC>
__device__ __forceinline__ void load_terms8(const uint16_t *row, int k0, int K, u32x4 (&t)[1])
{
    if (VEC) {  // K % 8 == 0 and 16-byte aligned rows
        t[0] = k0 < K ? *reinterpret_cast<const u32x4 *>(row + k0) : u32x4{0, 0, 0, 0};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned lo = k0 + 2 * i < K ? row[k0 + 2 * i] : 0u;
        const unsigned hi = k0 + 2 * i + 1 < K ? row[k0 + 2 * i + 1] : 0u;
        t[0][i] = lo | hi << 16;
    }
}

template <bool VEC>
__device__ __forceinline__ void load_f8(const float *row, int k0, int K, f32x4 (&x)[2])
{
    if (VEC) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            x[i] = k0 < K ? *reinterpret_cast<const f32x4 *>(row + k0 + 4 * i)
                          : f32x4{0.f, 0.f, 0.f, 0.f};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i >> 2][i & 3] = k0 + i < K ? row[k0 + i] : 0.0f;
}

__device__ __forceinline__ void split_terms8(const f32x4 (&x)[2], u32x4 (&t)[3])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned p[3];
        terms2<3>(x[i >> 1][2 * (i & 1)], x[i >> 1][2 * (i & 1) + 1], p);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            t[j][i] = p[j];
    }
}

template <bool VEC>
__device__ __forceinline__ void load_terms8(const float *row, int k0, int K, u32x4 (&t)[3])
{
    f32x4 x[2];
    load_f8<VEC>(row, k0, K, x);
    split_terms8(x, t);
}

__device__ __forceinline__ void store_c(float *c, float v) { *c = v; }
__device__ __forceinline__ void store_c(uint16_t *c, float v)
{
    const __bf16 b = static_cast<__bf16>(v);  // round to nearest even
    *c = __builtin_bit_cast(uint16_t, b);
}

struct LinArgs {
    const void *a;
    const uint8_t *codes, *scales;
    void *c;
    float *part;  // split K: f32 planes [splits][M][N]
    int64_t lda, ldc;
    int M, N, K, groups;
    int chunk;               // few rows: elements of K staged at once
    int tiles_m, tiles_n;    // tiles
    int chunks, per_split;   // tiles: K chunks, and of one split
};

// ------------------------------------------------------------- few rows

constexpr int kFewRows = 16;             // batch rows of a workgroup
constexpr int kFewLds = 32768;           // staged bf16 elements (64 KiB)
constexpr int kFewBlock = 128;           // K elements a wave takes at a time
constexpr int kFewPad = 8;               // elements between staged rows (16 bytes)

template <typename T, int WAVES, bool VEC>
__global__ __launch_bounds__(WAVES * 64) void linear_few_kernel(LinArgs p)
{
    constexpr int NT = kTerms<T>;
    __shared__ __attribute__((aligned(16))) uint16_t smem[kFewLds];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16;
    const int ld = p.chunk + kFewPad;
    // This lane's weight row and, as the other operand, its batch row.
    const int64_t wrow = int64_t(min(row0 + n, p.N - 1)) * p.groups;
    const int xoff = min(n, p.M - 1) * ld + 32 * g;

    auto load = [&](int blk, u32x4 &codes, unsigned &scale) {
        const int kg = blk * 4 + g;
        codes = u32x4{0, 0, 0, 0};
        scale = 127;
        if (kg < p.groups) {
            codes = *reinterpret_cast<const u32x4 *>(p.codes + (wrow + kg) * 16);
            scale = p.scales[wrow + kg];
        }
    };
    const int blocks = (p.K + kFewBlock - 1) / kFewBlock;
    const int chunk_blocks = p.chunk / kFewBlock;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    u32x4 codes;
    unsigned scale;
    load(wave, codes, scale);
    for (int b0 = 0; b0 < blocks; b0 += chunk_blocks) {
        const int nb = min(chunk_blocks, blocks - b0);
        // Stage rows [M][nb * 128] as terms, eight elements per thread and step.
        const int pieces = nb * (kFewBlock / 8);
        if (b0)
            __syncthreads();
        for (int i = tid; i < pieces * p.M; i += WAVES * 64) {
            const int m = i / pieces, k8 = (i - m * pieces) * 8;
            u32x4 t[NT];
            load_terms8<VEC>(static_cast<const T *>(p.a) + m * p.lda, b0 * kFewBlock + k8, p.K, t);
#pragma unroll
            for (int j = 0; j < NT; ++j)
                *reinterpret_cast<u32x4 *>(smem + (j * p.M + m) * ld + k8) = t[j];
        }
        __syncthreads();
        if (wave >= nb)  // no block of this chunk: look to the next
            load(b0 + chunk_blocks + wave, codes, scale);
        for (int b = wave; b < nb; b += WAVES) {
            const u32x4 w = codes;
            const float s = scale_of(scale);
            // The next block of this wave: of this chunk, or its first of the next.
            const int nxt = b + WAVES < nb ? b0 + b + WAVES : b0 + chunk_blocks + wave;
            load(nxt, codes, scale);
            const uint16_t *x = smem + xoff + b * kFewBlock;
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const bf16x8 wf = decode8(w[st], s);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc = mfma16(wf, *reinterpret_cast<const bf16x8 *>(x + j * p.M * ld + 8 * st),
                                 acc);
            }
        }
    }
    // Waves' sums in wave order: lane (n, g) holds weight rows 4g .. 4g+3 of batch row n.
    __syncthreads();
    f32x4 *red = reinterpret_cast<f32x4 *>(smem);
    red[tid] = acc;
    __syncthreads();
    if (tid < 64 && n < p.M) {
        f32x4 sum = red[lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            sum += red[w * 64 + lane];
        T *c = static_cast<T *>(p.c) + n * p.ldc + row0 + 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row0 + 4 * g + r < p.N)
                store_c(c + r, sum[r]);
    }
}

// ---------------------------------------------------------------- tiles

constexpr int kTileK = 64;  // K elements per chunk: 128-byte rows of bf16

// 16-byte pieces of a staged 128-byte row, so that the 16 rows of a
// ds_read_b128 quarter touch distinct banks.
__device__ __forceinline__ int swizzle(int row, int piece)
{
    return piece ^ ((row & 7) ^ ((row >> 3) & 1));
}

template <typename T, int BM, int BN, int WM, int WN, bool VEC>
__global__ __launch_bounds__(WM *WN * 64) void linear_tile_kernel(LinArgs p)
{
    constexpr int NT = kTerms<T>;
    constexpr int THREADS = WM * WN * 64;
    constexpr int MB = BM / WM / 32, NB = BN / WN / 32;
    constexpr int A_EL = NT * BM * kTileK, STAGE = A_EL + BN * kTileK;
    constexpr int AT = BM * 8 / THREADS;      // 8-element pieces of A per thread
    constexpr int CPT = BN * kTileK / THREADS;  // codes per thread
    static_assert(AT >= 1 && (CPT == 16 || CPT == 32), "tile too small for its threads");
    __shared__ __attribute__((aligned(16))) uint16_t smem[2 * STAGE];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int col = lane & 31, half = lane >> 5;
    const int tiles = p.tiles_m * p.tiles_n;
    const int blk = xcd_major_block();
    const int split = blk / tiles, t = blk - split * tiles;
    const int tm = t / p.tiles_n, tn = t - tm * p.tiles_n;
    const int row0 = tm * BM, col0 = tn * BN;
    const int c0 = split * p.per_split, c1 = min(c0 + p.per_split, p.chunks);

    // What this thread stages: AT pieces of A, CPT codes of one weight row.
    const T *arow[AT];
    int apiece[AT], ar[AT];
#pragma unroll
    for (int i = 0; i < AT; ++i) {
        const int f = i * THREADS + tid;
        ar[i] = f >> 3;
        apiece[i] = f & 7;
        arow[i] = static_cast<const T *>(p.a) + int64_t(min(row0 + ar[i], p.M - 1)) * p.lda;
    }
    constexpr int PER_ROW = kTileK / CPT;  // threads per weight row
    const int br = tid / PER_ROW, bpart = tid % PER_ROW;
    const int64_t brow = int64_t(min(col0 + br, p.N - 1)) * p.groups;

    f32x4 af[AT][2];
    u32x4 ab[AT];
    u32x4 codes;
    unsigned scale;
    auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            const int k0 = c * kTileK + apiece[i] * 8;
            if constexpr (NT == 3)
                load_f8<VEC>(arow[i], k0, p.K, af[i]);
            else {
                u32x4 t1[1];
                load_terms8<VEC>(arow[i], k0, p.K, t1);
                ab[i] = t1[0];
            }
        }
        const int kg = c * 2 + bpart * CPT / 32;
        codes = u32x4{0, 0, 0, 0};
        scale = 127;
        if (kg < p.groups) {
            const uint8_t *src = p.codes + (brow + kg) * 16 + (CPT == 16 ? (bpart & 1) * 8 : 0);
            if constexpr (CPT == 32)
                codes = *reinterpret_cast<const u32x4 *>(src);
            else {
                const u32x2 h = *reinterpret_cast<const u32x2 *>(src);
                codes = u32x4{h[0], h[1], 0, 0};
            }
            scale = p.scales[brow + kg];
        }
    };
    auto store = [&](int stage) {
        uint16_t *sa = smem + stage * STAGE;
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            uint16_t *dst = sa + ar[i] * kTileK + swizzle(ar[i], apiece[i]) * 8;
            if constexpr (NT == 3) {
                u32x4 t3[3];
                split_terms8(af[i], t3);
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    *reinterpret_cast<u32x4 *>(dst + j * BM * kTileK) = t3[j];
            } else
                *reinterpret_cast<u32x4 *>(dst) = ab[i];
        }
        const float s = scale_of(scale);
        uint16_t *sb = sa + A_EL + br * kTileK;
#pragma unroll
        for (int i = 0; i < CPT / 8; ++i)
            *reinterpret_cast<bf16x8 *>(sb + swizzle(br, bpart * (CPT / 8) + i) * 8) =
                decode8(codes[i], s);
    };

    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[i][j][r] = 0.0f;

    load(c0);
    store(0);
    if (c0 + 1 < c1)
        load(c0 + 1);
    __syncthreads();
    for (int c = c0; c < c1; ++c) {
        const int stage = (c - c0) & 1;
        const uint16_t *sa = smem + stage * STAGE;
        const uint16_t *sb = sa + A_EL;
#pragma unroll
        for (int ks = 0; ks < kTileK / 16; ++ks) {
            bf16x8 bw[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int r = (wn * NB + j) * 32 + col;
                bw[j] = *reinterpret_cast<const bf16x8 *>(sb + r * kTileK +
                                                          swizzle(r, 2 * ks + half) * 8);
            }
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int r = (wm * MB + i) * 32 + col;
#pragma unroll
                for (int q = 0; q < NT; ++q) {
                    const bf16x8 av = *reinterpret_cast<const bf16x8 *>(
                        sa + (q * BM + r) * kTileK + swizzle(r, 2 * ks + half) * 8);
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        acc[i][j] = mfma_bf16(av, bw[j], acc[i][j]);
                }
            }
        }
        if (c + 1 < c1) {
            store(stage ^ 1);
            if (c + 2 < c1)
                load(c + 2);
            __syncthreads();
        }
    }

    // Lane (col, half) holds column col of rows acc_row(r, half) of its blocks.
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int nn = col0 + (wn * NB + j) * 32 + col;
        if (nn >= p.N)
            continue;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = row0 + (wm * MB + i) * 32 + acc_row(r, half);
                if (m < p.M) {
                    if (p.part)
                        p.part[(int64_t(split) * p.M + m) * p.N + nn] = acc[i][j][r];
                    else
                        store_c(static_cast<T *>(p.c) + int64_t(m) * p.ldc + nn, acc[i][j][r]);
                }
            }
    }
}

// ----------------------------------------------------------- wide tiles

constexpr int kWideK = 128;   // K elements per chunk: 256-byte rows of A, 64 bytes of codes
constexpr int kWideN = 256;   // weight rows of a tile

// bf16 activations, K a multiple of 128, 16-byte aligned rows.  Tiles of
// 64 MB x 256: 8 waves as 2 (M) x 4 (N), each 32 MB rows and 64 columns, C^T
// on 32x32x16 MFMAs (W the first operand), so that a lane's four consecutive
// accumulators are four columns of one row.
// A's rows and W's codes reach LDS by DMA, two stages of 128 elements of K; 16-byte
// pieces are placed by piece ^ (row & 15) (A) and piece ^ (row / 4 & 3) (codes).
// A lane takes 64 contiguous codes of a weight row from there, two scale groups,
// and decodes them as the MFMA's k index wants them, k = 64 half + 8 step + j,
// the order A is read in: the decoded weights never pass through LDS, whose reads
// would take as long as the MFMAs with them (256 x 256 tiles with both operands
// decoded to LDS: 200 us at 4608 x 8192 x 2048, this kernel 124 us).  Codes read
// by each wave from memory instead, 16 bytes of 64 rows per instruction, kept
// the address unit as busy as the MFMAs (146 us).
// Bound by the MFMA at the clock that power allows: 1.25 PFLOP/s at that
// size, where a library product of bf16 operands of 8192 x 8192 x 8192 runs 1.4.
template <int MB>
__global__ __launch_bounds__(512, 2) void linear_wide_kernel(LinArgs p)
{
    constexpr int BM = 64 * MB;
    constexpr int STAGE = BM * kWideK;
    constexpr int WINDOWS = 2 * MB;  // 1 KiB DMA windows (4 rows) per wave and chunk
    constexpr int NB = 2;
    constexpr int CODES = kWideN * 64;  // bytes of a stage's codes
    __shared__ __attribute__((aligned(16))) u16 smem[2 * STAGE + CODES];  // two stages of codes

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1;
    const int col = lane & 31, half = lane >> 5;
    const int blk = xcd_major_block();
    // Four M tiles by all N tiles at a time, M inside: the 32 CUs of an XCD work
    // on about 4 x 8 tiles.
    const int band = blk / (4 * p.tiles_n), in_band = blk - band * 4 * p.tiles_n;
    const int bm = min(4, p.tiles_m - 4 * band);
    const int tn = in_band / bm, tm = 4 * band + in_band - tn * bm;
    const int row0 = tm * BM, col0 = tn * kWideN;
    const int chunks = p.K / kWideK;

    unsigned off[WINDOWS];
#pragma unroll
    for (int i = 0; i < WINDOWS; ++i) {
        const int r = (wave * WINDOWS + i) * 4 + (lane >> 4);
        const int rr = min(row0 + r, p.M - 1) - row0;  // rows past M: not stored
        off[i] = unsigned(int64_t(rr) * p.lda * 2 + 16 * ((lane & 15) ^ (r & 15)));
    }
    const char *a0 = reinterpret_cast<const char *>(static_cast<const u16 *>(p.a) +
                                                    int64_t(row0) * p.lda);
    // Codes: 16 windows of 16 rows x 64 bytes, two per wave, 16-byte pieces
    // placed by piece ^ (row / 4 & 3).
    unsigned woff[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (wave * 2 + i) * 16 + (lane >> 2);
        const int rr = min(col0 + r, p.N - 1) - col0;
        woff[i] = unsigned(rr * (p.K / 2) + 16 * ((lane & 3) ^ (r >> 2 & 3)));
    }
    const char *w0 = reinterpret_cast<const char *>(p.codes + int64_t(col0) * (p.K / 2));
    u16 *const smem_w = smem + 2 * STAGE;
    auto dma = [&](int c, int stage) {
        const char *src = a0 + int64_t(c) * (kWideK * 2);
#pragma unroll
        for (int i = 0; i < WINDOWS; ++i)
            dma16s(src, off[i], smem + stage * STAGE + (wave * WINDOWS + i) * 512);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            dma16s(w0 + c * (kWideK / 2), woff[i],
                   smem_w + stage * (CODES / 2) + (wave * 2 + i) * 512);
    };

    // The scales of this wave's 64 rows, one row per lane.
    const uint8_t *ws = p.scales + int64_t(min(col0 + wn * 64 + lane, p.N - 1)) * p.groups;
    unsigned sc[NB], sc_next = 0;
    u32x4 codes[NB][2];
    auto load = [&](int c) { sc_next = *reinterpret_cast<const unsigned *>(ws + c * 4); };
    // Rows wn * 64 + 32 j + col: 64 codes of this half, and their two scales.
    auto fetch = [&](int stage) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int r = wn * 64 + 32 * j + col;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                codes[j][h] = *reinterpret_cast<const u32x4 *>(
                    smem_w + stage * (CODES / 2) + r * 32 + ((2 * half + h) ^ (r >> 2 & 3)) * 8);
            sc[j] = unsigned(__shfl(int(sc_next), 32 * j + col)) >> (16 * half) & 0xFFFFu;
        }
    };

    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[i][j][r] = 0.0f;

    // Fragments of a step are read, and its weights decoded, while the MFMAs of
    // the step before run; a chunk's first ones under the last step of the chunk
    // before it, behind the barrier that ends that chunk.
    bf16x8 af[2][MB], wf[2][NB];
    unsigned ao = 0;
    auto read = [&](int st, bf16x8 (&f)[MB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
            f[i] = *reinterpret_cast<const bf16x8 *>(smem + 32 * i * kWideK + (ao ^ 8 * st));
    };
    auto decode = [&](int st, bf16x8 (&f)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
            f[j] = decode8(codes[j][st >> 2][st & 3],
                           scale_of(st < 4 ? sc[j] & 255u : sc[j] >> 8));
    };
    // Chunk c is staged and its codes are here; the one after next may come.
    auto enter = [&](int c) {
        wait_vmcnt<0>();
        ring_barrier();
        fetch(c & 1);
        if (c + 1 < chunks) {
            load(c + 1);
            dma(c + 1, (c + 1) & 1);
        }
        // Piece 8 half + step of rows wm * 32 MB + 32 i + col.
        ao = (c & 1) * STAGE + (wm * 32 * MB + col) * kWideK + ((8 * half) ^ (col & 15)) * 8;
        asm volatile("" : "+v"(ao));
    };
    load(0);
    dma(0, 0);
    enter(0);
    read(0, af[0]);
    decode(0, wf[0]);
    for (int c = 0; c < chunks; ++c) {
#pragma unroll
        for (int st = 0; st < 8; ++st) {
            if (st < 7)
                read(st + 1, af[(st + 1) & 1]);
            else if (c + 1 < chunks) {
                enter(c + 1);
                read(0, af[0]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    acc[i][j] = mfma_bf16(wf[st & 1][j], af[st & 1][i], acc[i][j]);
            decode((st + 1) & 7, wf[(st + 1) & 1]);
        }
    }

    // Lane (col, half): row col of its blocks, columns acc_row(r, half).  Through
    // LDS, so that rows go out in 128-byte runs.
    __syncthreads();
    constexpr int PITCH = 72;  // bf16 elements of a staged row: 64 and 16 bytes against conflicts
    static_assert(8 * 32 * PITCH <= 2 * STAGE, "the staged rows fit");
    u16 *so = smem + wave * 32 * PITCH;
    const int n0 = col0 + wn * 64;
    const bool wide = (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.ldc % 8 == 0 &&
                      n0 + 64 <= p.N;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                u32x2 v;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    v[e] = __builtin_bit_cast(
                        unsigned, __builtin_convertvector(f32x2{acc[i][j][r + 2 * e],
                                                                acc[i][j][r + 2 * e + 1]},
                                                          bf16x2));
                *reinterpret_cast<u32x2 *>(so + col * PITCH + 32 * j + acc_row(r, half)) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = 8 * q + (lane >> 3), piece = lane & 7;
            const int m = row0 + (wm * MB + i) * 32 + r;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(so + r * PITCH + 8 * piece);
            if (m >= p.M)
                continue;
            u16 *dst = static_cast<u16 *>(p.c) + int64_t(m) * p.ldc + n0 + 8 * piece;
            if (wide)
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(dst));
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n0 + 8 * piece + e < p.N)
                        dst[e] = u16(v[e >> 1] >> (16 * (e & 1)));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// C = the planes' sum, in split order.
template <typename T>
__global__ __launch_bounds__(256) void linear_sum_kernel(const float *part, T *c, int64_t ldc,
                                                         int M, int N, int splits)
{
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t plane = int64_t(M) * N;
    if (i >= plane)
        return;
    float sum = part[i];
    for (int s = 1; s < splits; ++s)
        sum += part[s * plane + i];
    const int64_t m = i / N;
    store_c(c + m * ldc + (i - m * N), sum);
}

// ----------------------------------------------------------------- plans

struct TileShape {
    int bm, bn;
};
// The last three are the wide kernel's.
constexpr TileShape kShapes[] = {{32, 128},  {64, 128},  {128, 128},
                                 {128, 256}, {192, 256}, {256, 256}};

struct Plan {
    int shape;  // -1: few rows
    int tiles_m = 0, tiles_n = 0, splits = 1, per_split = 0, chunks = 0;
};

// What a plan may assume of the pointers and strides (scratch sizes assume the best).
Plan plan_of(int M, int N, int K, Mx4Type type, bool wide = true)
{
    Plan pl;
    if (M <= kFewRows) {
        pl.shape = -1;
        return pl;
    }
    pl.chunks = (K + kTileK - 1) / kTileK;
    pl.shape = M <= 32 ? 0 : M <= 64 ? 1 : 2;
    // The wide tiles where they fill the GPU, of the height whose rounds over the
    // CUs take least.
    if (type == kMx4BF16 && K > 0 && K % kWideK == 0 && wide) {
        int64_t best = INT64_MAX;
        for (int sh = 3; sh < 6; ++sh) {
            const TileShape &t = kShapes[sh];
            const int64_t tiles = int64_t((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
            const int64_t cost = (tiles + 255) / 256 * (t.bm + 32);
            if (tiles >= 192 && cost < best) {
                best = cost;
                pl.shape = sh;
            }
        }
    }
    const TileShape &s = kShapes[pl.shape];
    pl.tiles_m = (M + s.bm - 1) / s.bm;
    pl.tiles_n = (N + s.bn - 1) / s.bn;
    const int64_t tiles = int64_t(pl.tiles_m) * pl.tiles_n;
    int splits = int(std::min<int64_t>(256 / std::max<int64_t>(tiles, 1), pl.chunks / 4));
    splits = pl.shape >= 3 ? 1 : std::max(1, std::min(splits, 16));
    pl.per_split = (pl.chunks + splits - 1) / splits;
    pl.splits = pl.per_split ? (pl.chunks + pl.per_split - 1) / pl.per_split : 1;
    return pl;
}

template <typename T, bool VEC>
bool run_few(LinArgs &p, hipStream_t st)
{
    // Elements of K staged at once, in whole blocks, and as many waves as have
    // a block of it each.
    const int blocks = std::max(1, (p.K + kFewBlock - 1) / kFewBlock);
    const int room = (kFewLds / (kTerms<T> * p.M) - kFewPad) / kFewBlock;
    const int chunk_blocks = std::min(room, blocks);
    p.chunk = chunk_blocks * kFewBlock;
    const dim3 grid((p.N + 15) / 16);
    if (chunk_blocks >= 12)
        hipLaunchKernelGGL((linear_few_kernel<T, 16, VEC>), grid, dim3(1024), 0, st, p);
    else if (chunk_blocks >= 6)
        hipLaunchKernelGGL((linear_few_kernel<T, 8, VEC>), grid, dim3(512), 0, st, p);
    else
        hipLaunchKernelGGL((linear_few_kernel<T, 4, VEC>), grid, dim3(256), 0, st, p);
    return hip_ok(hipGetLastError(), "linear_few_kernel launch");
}

template <typename T, bool VEC>
bool run_tiles(LinArgs &p, const Plan &pl, hipStream_t st)
{
    const int64_t blocks = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;
    if (blocks > INT32_MAX)
        return fail("linear_mx4_dev: too many tiles");
    const dim3 grid(static_cast<unsigned>(blocks));
    switch (pl.shape) {
    case 0:
        hipLaunchKernelGGL((linear_tile_kernel<T, 32, 128, 1, 4, VEC>), grid, dim3(256), 0, st, p);
        break;
    case 1:
        hipLaunchKernelGGL((linear_tile_kernel<T, 64, 128, 2, 2, VEC>), grid, dim3(256), 0, st, p);
        break;
    case 2:
        hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2, 2, VEC>), grid, dim3(256), 0, st,
                           p);
        break;
    case 3:
        hipLaunchKernelGGL((linear_wide_kernel<2>), grid, dim3(512), 0, st, p);
        break;
    case 4:
        hipLaunchKernelGGL((linear_wide_kernel<3>), grid, dim3(512), 0, st, p);
        break;
    default:
        hipLaunchKernelGGL((linear_wide_kernel<4>), grid, dim3(512), 0, st, p);
        break;
    }
    if (!hip_ok(hipGetLastError(), "linear_tile_kernel launch"))
        return false;
    if (pl.splits > 1) {
        const int64_t n = int64_t(p.M) * p.N;
        hipLaunchKernelGGL(linear_sum_kernel<T>, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st,
                           p.part, static_cast<T *>(p.c), p.ldc, p.M, p.N, pl.splits);
        return hip_ok(hipGetLastError(), "linear_sum_kernel launch");
    }
    return true;
}

template <typename T>
bool run_linear(LinArgs &p, const Plan &pl, bool rows16, hipStream_t st)
{
    const bool vec = rows16 && p.K % 8 == 0;
    if (pl.shape < 0)
        return vec ? run_few<T, true>(p, st) : run_few<T, false>(p, st);
    return vec ? run_tiles<T, true>(p, pl, st) : run_tiles<T, false>(p, pl, st);
}

}  // namespace

size_t linear_mx4_scratch_bytes(int M, int N, int K, Mx4Type type)
{
    if (M <= 0 || N <= 0 || K <= 0)
        return 0;
    const Plan pl = plan_of(M, N, K, type);
    return pl.splits > 1 ? size_t(pl.splits) * size_t(M) * size_t(N) * 4 : 0;
}

bool launch_linear_mx4(const void *a, int64_t lda, const uint8_t *codes, const uint8_t *scales,
                       void *c, int64_t ldc, int M, int N, int K, Mx4Type type, void *scratch,
                       size_t scratch_bytes, hipStream_t st)
{
    if (M <= 0 || N <= 0)
        return true;
    const bool rows16 = aligned(a, 16) && lda % (type == kMx4F32 ? 4 : 8) == 0;
    // Row offsets within a wide tile are 32-bit byte counts.
    Plan pl = plan_of(M, N, K, type, rows16 && lda <= (1 << 22));
    LinArgs p{};
    p.a = a;
    p.codes = codes;
    p.scales = scales;
    p.c = c;
    p.lda = lda;
    p.ldc = ldc;
    p.M = M;
    p.N = N;
    p.K = K;
    p.groups = int(mx4_groups(K));
    p.tiles_m = pl.tiles_m;
    p.tiles_n = pl.tiles_n;
    p.chunks = pl.chunks;
    p.per_split = pl.per_split;
    if (pl.splits > 1) {
        if (scratch_bytes < linear_mx4_scratch_bytes(M, N, K, type) || !scratch)
            return fail("linear_mx4_dev: scratch smaller than anima_hip_linear_mx4_scratch_bytes");
        if (!aligned(scratch, 16))
            return fail("linear_mx4_dev: scratch must be 16-byte aligned");
        p.part = static_cast<float *>(scratch);
    }
    return type == kMx4F32 ? run_linear<float>(p, pl, rows16, st)
                           : run_linear<uint16_t>(p, pl, rows16, st);
}

}  // namespace anima_hip
