// Linear layer with 4-bit weights: C[M,N] = A[M,K] . W[N,K]^T, W in MX4 rows
// (mx4.h), A and C both f32 or both bf16.
//
// Arithmetic: every MX4 weight is a bf16 number, so W enters the bf16 MFMA
// unrounded.  bf16 activations enter as they are; f32 activations as three
// bf16 terms whose sum is the f32 value (terms2), three MFMAs per product.
// Sums are f32, and C is rounded once, to its own type.
//
// Three kernels:
//   * few rows (M <= 16), bound by the one pass over the codes (17/32 byte per
//     weight) or, below about 8 MiB of codes, by latency (2048 x 2048 4.0 us): a workgroup takes 16
//     weight rows, its waves share K in blocks of 128, and the weights go from
//     memory to registers to the MFMA without touching LDS; or, of many weight
//     rows, each wave takes 16 through all of K;
//   * staged tiles (K a multiple of 128, 16-byte aligned rows of A), from 32 x 64 at
//     small M to 192 x 256 (bf16) and 256 x 256 (f32): bound by latency and the stream
//     into LDS at the small end, by the MFMA at the large;
//   * plain tiles for every other K and alignment: A (as terms) and the decoded
//     weights staged in LDS, two stages.
// The last two split K across workgroups where the tiles alone would leave CUs idle.
#include "mx4.h"
#include "mx4_plan.h"

#include <algorithm>

namespace anima_hip {
namespace {

using namespace flash_tile;
using mx4::decode8;
using mx4::mfma16;
using mx4::scale_of;
using mx4::terms2;
using mx4::u32x2;
using namespace mx4_plan;

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

// ------------------------------------------ few rows, many weight rows

// The rows of A stay in LDS, and each wave takes 16 weight rows at a time through all
// of K, four blocks (256 bytes of each row) ahead across the ends of the rows:
// no barrier after the first, and no sums between waves.  From 2048 strips of 16
// weight rows on, a workgroup for every CU, if A's terms fit half a CU's LDS.
// bf16, this kernel against the one above: 11.0 and 15.0 us at N x K = 32768 x
// 2048, 10.5 and 7.6 at 16384 x 2048, 6.3 and 14.3 at 65536 x 500, 19.0 and 27.5
// at 65536 x 2048, 146 and 143 at 131072 x 8192, M = 1; 35 (4.1 TB/s) and 54 at
// 131072 x 2048, M = 8, 38 and 82 at M = 16; f32 162 and 173 at 131072 x 8192, M =
// 1.  Blocks loaded one by one leave each row of the memory
// too soon (163), eight at a time take 3 to 5 % more or less.
constexpr int kWideWaves = 8, kWideBlocks = 4;
constexpr int kWideStrips = 256 * kWideWaves;
constexpr int kWideLds = 40960;  // staged bf16 elements (80 KiB)

template <typename T, bool VEC>
__global__ __launch_bounds__(kWideWaves * 64) void linear_wide_kernel(LinArgs p)
{
    constexpr int NT = kTerms<T>;
    __shared__ __attribute__((aligned(16))) uint16_t smem[kWideLds];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int ld = p.chunk + kFewPad;
    const int pieces = p.chunk / 8;
    const int blocks = p.chunk / kFewBlock;
    const int strips = (p.N + 15) / 16, step = int(gridDim.x) * kWideWaves;
    int strip = int(blockIdx.x) * kWideWaves + wave;  // of the products
    int lstrip = strip, lblk = 0;                     // of the next load

    struct Batch {
        u32x4 codes[kWideBlocks];
        unsigned scale[kWideBlocks];
    } cur, next;
    const int batches = (blocks + kWideBlocks - 1) / kWideBlocks;
    auto load = [&](Batch &b) {
        const int64_t row = int64_t(min(lstrip * 16 + n, p.N - 1)) * p.groups;
#pragma unroll
        for (int i = 0; i < kWideBlocks; ++i) {
            const int kg = (lblk * kWideBlocks + i) * 4 + g;
            b.codes[i] = u32x4{0, 0, 0, 0};
            b.scale[i] = 127;
            if (kg < p.groups) {
                b.codes[i] = *reinterpret_cast<const u32x4 *>(p.codes + (row + kg) * 16);
                b.scale[i] = p.scales[row + kg];
            }
        }
        if (++lblk == batches) {
            lblk = 0;
            lstrip += step;
        }
    };
    if (strip < strips)
        load(cur);
    for (int i = tid; i < pieces * p.M; i += kWideWaves * 64) {
        const int m = i / pieces, k8 = (i - m * pieces) * 8;
        u32x4 t[NT];
        load_terms8<VEC>(static_cast<const T *>(p.a) + m * p.lda, k8, p.K, t);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<u32x4 *>(smem + (j * p.M + m) * ld + k8) = t[j];
    }
    __syncthreads();

    const uint16_t *x = smem + min(n, p.M - 1) * ld + 32 * g;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int t = 0; strip < strips;) {
        if (lstrip < strips)
            load(next);
#pragma unroll
        for (int i = 0; i < kWideBlocks; ++i) {
            const int blk = t * kWideBlocks + i;
            if (blk >= blocks)
                break;
            const float s = scale_of(cur.scale[i]);
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const bf16x8 wf = decode8(cur.codes[i][st], s);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc = mfma16(wf,
                                 *reinterpret_cast<const bf16x8 *>(x + j * p.M * ld +
                                                                   blk * kFewBlock + 8 * st),
                                 acc);
            }
        }
        cur = next;
        if (++t < batches)
            continue;
        // Lane (n, g) holds weight rows 4g .. 4g+3 of batch row n.
        const int c0 = strip * 16 + 4 * g;
        if (n < p.M) {
            T *c = static_cast<T *>(p.c) + n * p.ldc + c0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (c0 + r < p.N)
                    store_c(c + r, acc[r]);
        }
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
        t = 0;
        strip += step;
    }
}

// ---------------------------------------------------------------- tiles

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

// --------------------------------------------------------- staged tiles

// K a multiple of 128 and 16-byte aligned rows of A.  Tiles of 32 MB WM rows of
// A by 32 NB WN rows of W; waves as WM x WN x KS, each 32 MB x 32 NB of C on the
// K steps of its share (KS > 1: the shares are added through LDS at the end).
// C^T on 32x32x16 MFMAs, W the first operand, so that a lane's four consecutive
// accumulators are four columns of one row.
//
// A's rows, W's codes and scales reach LDS by DMA through S stages.  A stage is 256
// bytes of each row of A, 128 bf16 or 64 f32 elements, and the codes of as many, or
// twice that (CM = 2: the smaller tiles, whose barrier and addresses take as long as
// their products; 333 x 2048 x 1024 f32 16.1 -> 13.8 us, 160 x 4096 x 4096 bf16 20.5 ->
// 17.5); 16-byte pieces are placed by piece ^ (row & 15) (A) and by code_swizzle
// against bank conflicts.
// A lane takes the contiguous codes of its half of the chunk and decodes them in
// registers, as the MFMA's k index wants them: k = KC / 2 half + 8 step + j, the
// order A is read in.  f32 A is split into its three terms there too, once for
// NB products.  With the decoded weights in LDS its reads take as long as the
// MFMAs (256 x 256 tiles at 4608 x 8192 x 2048, bf16: 200 us, this kernel 124),
// and codes read by each wave from memory, 16 bytes of 64 rows per
// instruction, keep the address unit as busy as the MFMAs (146 us).
// Fragments of a step are read, and its weights decoded, while the MFMAs of the
// step before run; a chunk's first ones under the last step of the chunk before,
// behind the barrier that ends it.
template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int CM>
struct Staged {
    static constexpr int NT = kTerms<T>;
    static constexpr int WAVES = WM * WN * KS, THREADS = WAVES * 64;
    static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
    static constexpr int KC = CM * 256 / int(sizeof(T));  // K elements of a chunk
    static constexpr int STEPS = KC / 16, SHARE = STEPS / KS;
    static constexpr int CP = KC / 32;        // 16-byte pieces of a row's codes, and its scales
    static constexpr int SD = CP > 4 ? 2 : 1;  // dwords of a row's scales
    // LDS in u16: A rows of 128 CM, codes rows of KC / 4, scales SD planes of a dword a row.
    static constexpr int A_ROW = 128 * CM;
    static constexpr int A_EL = BM * A_ROW, C_EL = BN * (KC / 4), STAGE = (A_EL + C_EL + BN * 2 * SD + A_ROW - 1) / A_ROW * A_ROW;
    // 1 KiB windows (scales: 256 bytes) per chunk, and per wave; a wave without
    // one copies the last again, so that all count the same.
    static constexpr int A_WIN = BM * CM / 4, C_WIN = C_EL / 512, S_WIN = SD * BN / 64;
    static constexpr int A_OPS = (A_WIN + WAVES - 1) / WAVES;
    static constexpr int C_OPS = (C_WIN + WAVES - 1) / WAVES;
    static constexpr int S_OPS = (S_WIN + WAVES - 1) / WAVES;
    static constexpr int OPS = A_OPS + C_OPS + S_OPS;
    // The epilogue's rows of one 32-row block per wave, and the shares' sums.
    static constexpr int PITCH = 32 * NB + 16 / int(sizeof(T));
    static constexpr int OUT_EL = WAVES / KS * 32 * PITCH * int(sizeof(T)) / 2;
    static constexpr int RED_EL = (KS - 1) * (WAVES / KS) * MB * NB * 2048;
    static constexpr int LDS =
        S * STAGE > RED_EL ? (S * STAGE > OUT_EL ? S * STAGE : OUT_EL)
                           : (RED_EL > OUT_EL ? RED_EL : OUT_EL);
    static_assert(BN % 64 == 0 && STEPS % KS == 0 && LDS <= 81920, "160 KiB of LDS");
    static_assert((S - 2) * OPS < 16, "counted by vmcnt");
};

// One dword per lane from base + voff to the 256-byte LDS window at `lds`, as
// flash_tile::dma16s copies 16 bytes.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma4s(const void *base, unsigned voff, u16 *lds)
{
    const unsigned m0 = static_cast<unsigned>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(m0), "v"(voff), "s"(base)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename T, int MB, int NB, int WM, int WN, int KS, int S, int CM>
__global__ __launch_bounds__(WM *WN *KS * 64) void linear_staged_kernel(LinArgs p)
{
    using G = Staged<T, MB, NB, WM, WN, KS, S, CM>;
    constexpr int NT = G::NT, CP = G::CP;
    __shared__ __attribute__((aligned(16))) u16 smem[G::LDS];

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
    const int c0 = split * p.per_split, c1 = min(c0 + p.per_split, p.K / G::KC);

    // This lane's part of each copy, in bytes from the tile's first row; rows past
    // M or N read the last one again (their results are not stored).
    unsigned aoff[G::A_OPS], coff[G::C_OPS], soff[G::S_OPS];
    int adst[G::A_OPS], cdst[G::C_OPS], sdst[G::S_OPS];
    constexpr int AROWS = 4 / CM, CROWS = 2048 / G::KC;  // rows of a window
    auto code_swizzle = [](int r) { return CP == 8 ? r & 7 : CP == 4 ? r >> 2 & 3 : r >> 3 & 1; };
#pragma unroll
    for (int i = 0; i < G::A_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::A_WIN - 1);
        const int r = w * AROWS + lane / (16 * CM);
        aoff[i] = unsigned(int64_t(min(row0 + r, p.M - 1) - row0) * p.lda * int(sizeof(T)) +
                           16 * (lane % (16 * CM) ^ (r & 15)));
        adst[i] = w * 512;
    }
#pragma unroll
    for (int i = 0; i < G::C_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::C_WIN - 1);
        const int r = w * CROWS + lane / CP;
        const int piece = lane % CP ^ code_swizzle(r);
        coff[i] = unsigned((min(col0 + r, p.N - 1) - col0) * (p.K / 2) + 16 * piece);
        cdst[i] = G::A_EL + w * 512;
    }
#pragma unroll
    for (int i = 0; i < G::S_OPS; ++i) {
        const int w = min(i * G::WAVES + wave, G::S_WIN - 1);
        const int r = w % (G::BN / 64) * 64 + lane;
        soff[i] = unsigned((min(col0 + r, p.N - 1) - col0) * p.groups + w / (G::BN / 64) * 4);
        sdst[i] = G::A_EL + G::C_EL + w * 128;
    }
    const char *a0 = reinterpret_cast<const char *>(static_cast<const T *>(p.a) +
                                                    int64_t(row0) * p.lda);
    const char *w0 = reinterpret_cast<const char *>(p.codes) + int64_t(col0) * (p.K / 2);
    const char *s0 = reinterpret_cast<const char *>(p.scales) + int64_t(col0) * p.groups;
    auto dma = [&](int c, int stage) {
        u16 *dst = smem + stage * G::STAGE;
#pragma unroll
        for (int i = 0; i < G::A_OPS; ++i)
            dma16s(a0 + int64_t(c) * (256 * CM), aoff[i], dst + adst[i]);
#pragma unroll
        for (int i = 0; i < G::C_OPS; ++i)
            dma16s(w0 + int64_t(c) * (G::KC / 2), coff[i], dst + cdst[i]);
        // Four scales a row: of this chunk, or of the pair of chunks it is in.
#pragma unroll
        for (int i = 0; i < G::S_OPS; ++i)
            dma4s(s0 + (c * (G::KC / 32) & ~3), soff[i], dst + sdst[i]);
    };

    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[i][j][r] = 0.0f;

    constexpr int W = G::KC / 16;  // words of a lane's codes, 64 or 32 of them
    unsigned codes[NB][W], sc[NB];
    unsigned ao = 0;
    typedef u32x4 Raw[NT == 3 ? 2 : 1];  // eight elements of A as they are stored
    Raw raw[2][MB];
    bf16x8 wf[2][NB];
    auto read = [&](int st, Raw(&f)[MB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int h = 0; h < (NT == 3 ? 2 : 1); ++h)
                f[i][h] = *reinterpret_cast<const u32x4 *>(
                    smem + 32 * i * G::A_ROW + (ao ^ (NT == 3 ? 16 * st + 8 * h : 8 * st)));
    };
    auto decode = [&](int st, bf16x8 (&f)[NB]) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
            f[j] = decode8(codes[j][st], scale_of(sc[j] >> (st >> 2) * 8 & 255u));
    };
    auto enter = [&](int c) {
        // Chunk c has landed when at most the S - 2 behind it are on their way.
        if (c + S - 2 < c1)
            wait_vmcnt<(S - 2) * G::OPS>();
        else
            wait_vmcnt<0>();
        ring_barrier();  // for every wave; and all have left the stage before it
        if (c + S - 1 < c1)
            dma(c + S - 1, (c + S - 1 - c0) % S);
        const unsigned base = (c - c0) % S * G::STAGE;
        // Rows (wm MB + i) 32 + col, this half of the chunk.
        ao = base + (wm * 32 * MB + col) * G::A_ROW + ((8 * CM * half) ^ (col & 15)) * 8;
        asm volatile("" : "+v"(ao));
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int r = (wn * NB + j) * 32 + col;
            const u16 *row = smem + base + G::A_EL + r * (G::KC / 4);
#pragma unroll
            for (int h = 0; h < W / 4; ++h) {
                const int piece = (CP / 2 * half + h) ^ code_swizzle(r);
                const u32x4 v = *reinterpret_cast<const u32x4 *>(row + 8 * piece);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    codes[j][4 * h + e] = v[e];
            }
            const unsigned s4 = *reinterpret_cast<const unsigned *>(
                smem + base + G::A_EL + G::C_EL + (CP == 8 ? half * G::BN * 2 : 0) + r * 2);
            sc[j] = s4 >> (CP == 8 ? 0 : CP == 4 ? 16 * half : 16 * (c & 1) + 8 * half);
        }
    };
    auto multiply = [&](const Raw(&f)[MB], const bf16x8 (&w)[NB]) {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            bf16x8 term[NT];
            if constexpr (NT == 3) {
                const f32x4 x[2] = {__builtin_bit_cast(f32x4, f[i][0]),
                                    __builtin_bit_cast(f32x4, f[i][1])};
                u32x4 u[3];
                split_terms8(x, u);
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    term[q] = __builtin_bit_cast(bf16x8, u[q]);
            } else
                term[0] = __builtin_bit_cast(bf16x8, f[i][0]);
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    acc[i][j] = mfma_bf16(w[j], term[q], acc[i][j]);
        }
    };

    // This wave's steps of a chunk: share * SHARE .. .  The step within the
    // share is a constant where codes and scales are picked from registers.
    auto step_of = [&](int i) { return KS == 1 ? i : share * G::SHARE + i; };
    auto pick = [&](int i, bf16x8 (&f)[NB]) {
        if constexpr (KS == 1)
            decode(i, f);
        else
#pragma unroll
            for (int k = 0; k < KS; ++k)
                if (share == k)
                    decode(k * G::SHARE + i, f);
    };
    static_assert(S >= 2, "a stage to fill while one is used");
    if (c0 < c1) {
#pragma unroll
        for (int i = 0; i < S - 1; ++i)
            if (c0 + i < c1)
                dma(c0 + i, i);
        enter(c0);
        read(step_of(0), raw[0]);
        pick(0, wf[0]);
    }
    for (int c = c0; c < c1; ++c) {
#pragma unroll
        for (int st = 0; st < G::SHARE; ++st) {
            constexpr int LAST = G::SHARE - 1;
            const int now = G::SHARE == 1 ? 0 : st & 1, next = G::SHARE == 1 ? 1 : now ^ 1;
            if (st < LAST)
                read(step_of(st + 1), raw[next]);
            else if (c + 1 < c1) {
                enter(c + 1);
                read(step_of(0), raw[next]);
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply(raw[now], wf[now]);
            pick(st < LAST ? st + 1 : 0, wf[next]);
            if (G::SHARE % 2 == 1 && st == LAST) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int h = 0; h < (NT == 3 ? 2 : 1); ++h)
                        raw[0][i][h] = raw[next][i][h];
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    wf[0][j] = wf[next][j];
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
                for (int r = 0; r < 16; r += 4) {
                    const int nn = n0 + 32 * j + acc_row(r, half);
                    float *dst = plane + int64_t(m) * p.N + nn;
                    if (wide && nn < p.N)
                        *reinterpret_cast<f32x4 *>(dst) = f32x4{acc[i][j][r], acc[i][j][r + 1],
                                                                acc[i][j][r + 2], acc[i][j][r + 3]};
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (nn + e < p.N)
                                dst[e] = acc[i][j][r + e];
                }
        }
        return;
    }
    // Through LDS, so that rows go out in runs of 32 NB columns.
    T *so = reinterpret_cast<T *>(smem) + (wave % (WM * WN)) * 32 * G::PITCH;
    constexpr int E = 16 / int(sizeof(T));  // elements of a 16-byte piece
    constexpr int PIECES = 32 * NB / E;
    const bool wide = (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.ldc % E == 0 &&
                      n0 + 32 * NB <= p.N;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                T *dst = so + col * G::PITCH + 32 * j + acc_row(r, half);
                if constexpr (NT == 3)
                    *reinterpret_cast<f32x4 *>(dst) = f32x4{acc[i][j][r], acc[i][j][r + 1],
                                                            acc[i][j][r + 2], acc[i][j][r + 3]};
                else {
                    u32x2 v;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        v[e] = __builtin_bit_cast(
                            unsigned, __builtin_convertvector(f32x2{acc[i][j][r + 2 * e],
                                                                    acc[i][j][r + 2 * e + 1]},
                                                              bf16x2));
                    *reinterpret_cast<u32x2 *>(dst) = v;
                }
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < PIECES / 2; ++q) {
            const int f = q * 64 + lane, r = f / PIECES, piece = f % PIECES;
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
                        if constexpr (NT == 3)
                            dst[e] = __uint_as_float(v[e]);
                        else
                            dst[e] = u16(v[e >> 1] >> (16 * (e & 1)));
                    }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// C = the planes' sum, in split order (at most kLinMaxSplits), all loads in flight.
template <typename T>
__global__ __launch_bounds__(256) void linear_sum_kernel(const float *part, T *c, int64_t ldc,
                                                         int M, int N, int splits)
{
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t plane = int64_t(M) * N;
    if (i >= plane)
        return;
    float x[kLinMaxSplits];
#pragma unroll
    for (int s = 0; s < kLinMaxSplits; ++s)
        if (s < splits)
            x[s] = part[s * plane + i];
    float sum = x[0];
#pragma unroll
    for (int s = 1; s < kLinMaxSplits; ++s)
        if (s < splits)
            sum += x[s];
    const int64_t m = i / N;
    store_c(c + m * ldc + (i - m * N), sum);
}

// Copies with K padded to a multiple of 128: A with zeros, the weights with zero
// codes of a finite scale.  A thread writes 16 bytes of a row of A, or one group of
// a weight row; the first `a_blocks` workgroups take A.
template <typename T>
__global__ __launch_bounds__(256) void linear_pad_kernel(LinArgs p, T *a, uint8_t *codes,
                                                         uint8_t *scales, int padded,
                                                         unsigned a_blocks)
{
    constexpr int E = 16 / int(sizeof(T));
    if (blockIdx.x < a_blocks) {
        const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
        const int pieces = padded / E;
        const int64_t m = i / pieces;
        if (m >= p.M)
            return;
        const int k0 = int(i - m * pieces) * E;
        const T *row = static_cast<const T *>(p.a) + m * p.lda;
        T v[E];
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = k0 + e < p.K ? row[k0 + e] : T(0);
        u32x4 w;
        __builtin_memcpy(&w, v, 16);
        *reinterpret_cast<u32x4 *>(a + m * padded + k0) = w;
        return;
    }
    const int64_t i = int64_t(blockIdx.x - a_blocks) * 256 + threadIdx.x;
    const int groups = padded / 32;
    const int64_t n = i / groups;
    if (n >= p.N)
        return;
    const int g = int(i - n * groups);
    u32x4 c = {0, 0, 0, 0};
    unsigned s = 127;
    if (g < p.groups) {
        c = *reinterpret_cast<const u32x4 *>(p.codes + (n * p.groups + g) * 16);
        s = p.scales[n * p.groups + g];
    }
    *reinterpret_cast<u32x4 *>(codes + i * 16) = c;
    scales[i] = uint8_t(s);
}

// -------------------------------------------------------------- launches

// Shapes of the staged kernel, MB, NB, WM, WN, KS, S, and of the same with two chunks
// at once.
#define STAGED_BF16(X, cm) \
    X(cm, 0, 3, 2, 2, 4, 1, 2) X(cm, 1, 2, 2, 2, 4, 1, 2) X(cm, 2, 2, 2, 2, 2, 2, 2) \
    X(cm, 3, 1, 2, 2, 2, 2, 3) X(cm, 4, 1, 1, 2, 2, 2, 4) X(cm, 5, 1, 1, 1, 2, 4, 4)
#define PAIRED_BF16(X, cm) \
    X(cm, 3, 1, 2, 2, 2, 2, 2) X(cm, 4, 1, 1, 2, 2, 2, 2) X(cm, 5, 1, 1, 1, 2, 4, 3)
#define STAGED_F32(X, cm) X(cm, 0, 2, 4, 4, 2, 1, 2) X(cm, 1, 1, 4, 4, 2, 1, 3)
#define PAIRED_F32(X, cm) X(cm, 2, 1, 4, 2, 1, 4, 2) X(cm, 3, 1, 2, 1, 1, 4, 3)

#define SHAPE_CHECK(table, i, mb, nb, wm, wn, cm) \
    static_assert(table[i].bm == 32 * mb * wm && table[i].bn == 32 * nb * wn && \
                  (cm == 1 || table[i].pairs), "shape table");
#define CHECK_BF16(cm, i, mb, nb, wm, wn, ks, s) SHAPE_CHECK(kBf16Shapes, i, mb, nb, wm, wn, cm)
#define CHECK_F32(cm, i, mb, nb, wm, wn, ks, s) SHAPE_CHECK(kF32Shapes, i, mb, nb, wm, wn, cm)
STAGED_BF16(CHECK_BF16, 1)
PAIRED_BF16(CHECK_BF16, 2)
STAGED_F32(CHECK_F32, 1)
PAIRED_F32(CHECK_F32, 2)

template <typename T, bool VEC>
bool run_few(LinArgs &p, hipStream_t st)
{
    const int blocks = std::max(1, (p.K + kFewBlock - 1) / kFewBlock);
    const int strips = (p.N + 15) / 16;
    if (strips >= kWideStrips &&
        kTerms<T> * p.M * (int64_t(blocks) * kFewBlock + kFewPad) <= kWideLds) {
        p.chunk = blocks * kFewBlock;
        const dim3 grid(std::min(512, (strips + kWideWaves - 1) / kWideWaves));
        hipLaunchKernelGGL((linear_wide_kernel<T, VEC>), grid, dim3(kWideWaves * 64), 0, st, p);
        return hip_ok(hipGetLastError(), "linear_wide_kernel launch");
    }
    // Elements of K staged at once, in whole blocks, and as many waves as have
    // a block of it each.
    const int room = (kFewLds / (kTerms<T> * p.M) - kFewPad) / kFewBlock;
    const int chunk_blocks = std::min(room, blocks);
    p.chunk = chunk_blocks * kFewBlock;
    const dim3 grid(strips);
    const int waves = chunk_blocks >= 12 ? 16 : chunk_blocks >= 6 ? 8 : 4;
    if (!launch_fits(grid.x, waves * 64))
        return fail("linear_mx4_dev: too many weight rows for one launch");
    if (waves == 16)
        hipLaunchKernelGGL((linear_few_kernel<T, 16, VEC>), grid, dim3(1024), 0, st, p);
    else if (waves == 8)
        hipLaunchKernelGGL((linear_few_kernel<T, 8, VEC>), grid, dim3(512), 0, st, p);
    else
        hipLaunchKernelGGL((linear_few_kernel<T, 4, VEC>), grid, dim3(256), 0, st, p);
    return hip_ok(hipGetLastError(), "linear_few_kernel launch");
}

template <typename T, bool VEC>
bool run_tiles(const LinArgs &p, int shape, dim3 grid, hipStream_t st)
{
    switch (shape) {
    case 0:
        hipLaunchKernelGGL((linear_tile_kernel<T, 32, 128, 1, 4, VEC>), grid, dim3(256), 0, st, p);
        break;
    case 1:
        hipLaunchKernelGGL((linear_tile_kernel<T, 64, 128, 2, 2, VEC>), grid, dim3(256), 0, st, p);
        break;
    default:
        hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2, 2, VEC>), grid, dim3(256), 0, st,
                           p);
        break;
    }
    return hip_ok(hipGetLastError(), "linear_tile_kernel launch");
}

constexpr int kPairs = 16;  // beside a shape's number: two chunks at once
#define STAGED_CASE(cm, i, mb, nb, wm, wn, ks, s)                                                \
    case i + (cm == 2 ? kPairs : 0):                                                             \
        hipLaunchKernelGGL((linear_staged_kernel<T, mb, nb, wm, wn, ks, s, cm>), grid,           \
                           dim3(wm * wn * ks * 64), 0, st, p);                                   \
        break;

template <typename T>
bool run_staged(LinArgs p, const LinPlan &pl, dim3 grid, hipStream_t st)
{
    if (pl.pairs)
        p.per_split /= 2;
    // f32 chunks come in pairs, K being a multiple of 128.
    const int shape = pl.shape + (pl.pairs ? kPairs : 0);
    if constexpr (kTerms<T> == 1) {
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
    return hip_ok(hipGetLastError(), "linear_staged_kernel launch");
}

template <typename T>
bool run_pad(const LinArgs &p, void *a, uint8_t *codes, uint8_t *scales, hipStream_t st)
{
    const int padded = lin_padded(p.K);
    const int64_t a_blocks = (int64_t(p.M) * (padded * int(sizeof(T)) / 16) + 255) / 256;
    const int64_t w_blocks = (int64_t(p.N) * (padded / 32) + 255) / 256;
    if (!launch_fits(a_blocks + w_blocks, 256))
        return fail("linear_mx4_dev: operands too large for one launch");
    hipLaunchKernelGGL(linear_pad_kernel<T>, dim3(unsigned(a_blocks + w_blocks)), dim3(256), 0, st,
                       p, static_cast<T *>(a), codes, scales, padded, unsigned(a_blocks));
    return hip_ok(hipGetLastError(), "linear_pad_kernel launch");
}

template <typename T>
bool run_linear(LinArgs &p, const LinPlan &pl, bool rows16, hipStream_t st)
{
    const bool vec = rows16 && p.K % 8 == 0;
    if (pl.kernel == kFew)
        return vec ? run_few<T, true>(p, st) : run_few<T, false>(p, st);
    const int64_t blocks = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;
    if (!launch_fits(blocks, pl.kernel == kStaged ? 512 : 256))
        return fail("linear_mx4_dev: too many tiles for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    const bool ok = pl.kernel == kStaged ? run_staged<T>(p, pl, grid, st)
                    : vec                ? run_tiles<T, true>(p, pl.shape, grid, st)
                                         : run_tiles<T, false>(p, pl.shape, grid, st);
    if (!ok || pl.splits == 1)
        return ok;
    const int64_t n = int64_t(p.M) * p.N;
    hipLaunchKernelGGL(linear_sum_kernel<T>, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st,
                       p.part, static_cast<T *>(p.c), p.ldc, p.M, p.N, pl.splits);
    return hip_ok(hipGetLastError(), "linear_sum_kernel launch");
}

}  // namespace

size_t linear_mx4_scratch_bytes(int M, int N, int K, Mx4Type type)
{
    if (M <= 0 || N <= 0 || K <= 0)
        return 0;
    // For any pointers and strides.
    const bool f32 = type == kMx4F32;
    return size_t(std::max(lin_scratch(lin_plan(M, N, K, f32, true), M, N, K, f32).bytes,
                           lin_scratch(lin_plan(M, N, K, f32, false), M, N, K, f32).bytes));
}

bool launch_linear_mx4(const void *a, int64_t lda, const uint8_t *codes, const uint8_t *scales,
                       void *c, int64_t ldc, int M, int N, int K, Mx4Type type, void *scratch,
                       size_t scratch_bytes, hipStream_t st)
{
    if (M <= 0 || N <= 0)
        return true;
    const bool f32 = type == kMx4F32;
    const bool rows16 = aligned(a, 16) && lda % (f32 ? 4 : 8) == 0;
    const LinPlan pl = lin_plan(M, N, K, f32, rows16 && lda <= kStagedMaxK / 2);
    const size_t need = linear_mx4_scratch_bytes(M, N, K, type);
    if (need > 0) {
        if (scratch_bytes < need || !scratch)
            return fail("linear_mx4_dev: scratch smaller than anima_hip_linear_mx4_scratch_bytes");
        if (!aligned(scratch, 16))
            return fail("linear_mx4_dev: scratch must be 16-byte aligned");
    }
    const LinScratch parts = lin_scratch(pl, M, N, K, f32);
    char *const mem = static_cast<char *>(scratch);
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
    if (pl.splits > 1)
        p.part = reinterpret_cast<float *>(mem + parts.planes);
    if (pl.pad) {
        void *const pa = mem + parts.a;
        uint8_t *const pc = reinterpret_cast<uint8_t *>(mem + parts.codes);
        uint8_t *const ps = reinterpret_cast<uint8_t *>(mem + parts.scales);
        if (!(f32 ? run_pad<float>(p, pa, pc, ps, st) : run_pad<uint16_t>(p, pa, pc, ps, st)))
            return false;
        p.a = pa;
        p.codes = pc;
        p.scales = ps;
        p.K = lin_padded(K);
        p.lda = p.K;
        p.groups = p.K / 32;
    }
    return f32 ? run_linear<float>(p, pl, rows16, st) : run_linear<uint16_t>(p, pl, rows16, st);
}

}  // namespace anima_hip
