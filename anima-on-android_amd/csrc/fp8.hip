// 8-bit rows (fp8.h): packing and unpacking, and the root-mean-square norm that
// adds the residual and writes its result in 8-bit rows.
#include "fp8.h"

#include <algorithm>

namespace anima_hip {
namespace {

using namespace fp8;

// Packing and unpacking: 16 lanes a group, eight elements each.  Bound by HBM: from cold
// memory 20011 x 1000 f32 packs in 19.5 us and unpacks in 22.9, 8192 x 2048 in 16.8 and 13.3,
// 5.1, 4.4, 5.0 and 6.3 TB/s; eight elements in a row a lane unpack those in 23.3 and 20.6.
// Two or four groups a thread are no faster.
// STREAM: values are stored past the caches, where rows are whole cache lines (8192 x 2048 f32
// 17.4 us, so 13.3; 20011 x 1000 22.9 and 23.6, 9000 x 1003 11.2 and 13.2).
template <typename T>
__global__ __launch_bounds__(256) void fp8_pack_kernel(const T *x, int64_t ldx, uint8_t *codes,
                                                       uint8_t *scales, unsigned groups,
                                                       unsigned total, int K)
{
    const unsigned gi = blockIdx.x * 16u + (threadIdx.x >> 4);
    if (gi >= total)
        return;  // all 16 lanes of a group
    const int piece = threadIdx.x & 15;
    const unsigned row = gi / groups;
    const int g = int(gi - row * groups);
    float v[8];
    load8<kSecond<T>>(x + int64_t(row) * ldx, g * kGroup + run_of<T>(piece), K, v);
    pack_group<T>(v, codes + int64_t(row) * groups * kGroup,
                  scales + int64_t(row) * fp8_scale_bytes(K), g, int(groups), piece,
                  [](float (&)[8]) {});
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void fp8_unpack_kernel(const uint8_t *codes,
                                                         const uint8_t *scales, T *x, int64_t ldx,
                                                         unsigned groups, unsigned total, int K)
{
    const unsigned gi = blockIdx.x * 16u + (threadIdx.x >> 4);
    if (gi >= total)
        return;
    const int piece = threadIdx.x & 15;
    const unsigned row = gi / groups;
    const int g = int(gi - row * groups);
    const int byte = scales[int64_t(row) * fp8_scale_bytes(K) + g];
    const uint8_t *from = codes + int64_t(gi) * kGroup + run_of<T>(piece);
    u32x2 c;
    if constexpr (kSecond<T> == 4)
        c = *reinterpret_cast<const u32x2 *>(from);
    else
        c = u32x2{*reinterpret_cast<const unsigned *>(from),
                  *reinterpret_cast<const unsigned *>(from + kSecond<T>)};
    // 2^(byte - 127), subnormal for byte 0, NaN for 255.
    const float s = byte == 0 ? __uint_as_float(0x400000u)
                    : byte == kNanScale ? __uint_as_float(0x7FC00000u) : scale_of(byte);
    float v[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[i]), false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[i]), true);
        v[4 * i] = lo[0] * s;
        v[4 * i + 1] = lo[1] * s;
        v[4 * i + 2] = hi[0] * s;
        v[4 * i + 3] = hi[1] * s;
    }
    store8<kSecond<T>, STREAM>(x + int64_t(row) * ldx, g * kGroup + run_of<T>(piece), K, v);
}

// ------------------------------------------------------------------ norm

struct NormArgs {
    const void *x, *r;
    const float *w;
    void *sum, *y;
    uint8_t *codes, *scales;
    int64_t ldx, ldr, lds, ldy, rows;
    int K;
    float eps;
};

// Sum of v over the wave, in all lanes.
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int m = 1; m < 64; m <<= 1)
        v += __shfl_xor(v, m);
    return v;
}

// 1 / sqrt(m): the hardware's estimate and two Newton steps; its own value where
// the steps have none (m zero or infinite).
__device__ __forceinline__ double inv_sqrt(double m)
{
    double r = __builtin_amdgcn_rsq(m);
    if (m > 0.0 && m < __builtin_inf()) {
        r = r * fma(-0.5 * m * r, r, 1.5);
        r = r * fma(-0.5 * m * r, r, 1.5);
    }
    return r;
}

// y cut off after f32's 24 bits, the last of them set where anything was lost: rounding this
// to fewer bits is rounding y, also next to a tie.  Below f32's normal numbers, where it has
// fewer bits, the conversion would round once more: to_odd_small.
__device__ __forceinline__ float to_odd(double y)
{
    const u32x2 b = __builtin_bit_cast(u32x2, y);
    // Bit 29 where any below it is set.
    const unsigned lost = (b[0] & 0x1FFFFFFFu) + 0x1FFFFFFFu;
    return float(__builtin_bit_cast(double, u32x2{(b[0] & 0xE0000000u) | (lost & 0x20000000u), b[1]}));
}

// The same at f32's smallest numbers: the nearest one, moved to the odd one beside y.
__device__ __forceinline__ float to_odd_small(double y)
{
    const float f = float(y);
    unsigned bits = __float_as_uint(f);
    if (double(f) != y)
        bits = (bits - (fabs(double(f)) > fabs(y) ? 1u : 0u)) | 1u;
    return __uint_as_float(bits);
}

// h = x + r of eight elements in 64 bits, where it is exact but for values 2^29 apart in f32
// and 2^45 in bf16, and its f32 rounding; zero past K.
template <typename T>
__device__ __forceinline__ void load_sum(const NormArgs &p, int64_t row, int k0, double (&h)[8],
                                         float (&s)[8])
{
    load8<kSecond<T>>(static_cast<const T *>(p.x) + row * p.ldx, k0, p.K, s);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        h[i] = double(s[i]);
    if (p.r) {
        float r[8];
        load8<kSecond<T>>(static_cast<const T *>(p.r) + row * p.ldr, k0, p.K, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i] += r[i];
            h[i] += double(r[i]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_sum(const NormArgs &p, int64_t row, int k0,
                                          const float (&s)[8])
{
    // Past the caches: the sum is read a sub-layer later, the 8-bit rows next (8192 x 2048 bf16
    // between other calls 29.0 us, so 23.4; 2001 x 2047 f32 from cold memory 20.7 and 14.7; sums of
    // 33 MB read back at once 4 to 8 % more).
    if (p.sum)
        store8<kSecond<T>, true>(static_cast<T *>(p.sum) + row * p.lds, k0, p.K, s);
}

template <typename T>
__device__ __forceinline__ void load_weight(const NormArgs &p, int k0, float (&w)[8])
{
    if (p.w) {
        load8<kSecond<T>>(p.w, k0, p.K, w);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = 1.0f;
}

// A piece of the normed row.  The 16 lanes of a group come here together.
template <typename T>
__device__ __forceinline__ void store_normed(const NormArgs &p, int64_t row, int piece,
                                             const double (&h)[8], double inv, int groups)
{
    const int k0 = run_of<T>(piece);
    float w[8], odd[8], nearest[sizeof(T) == 4 ? 8 : 1];
    load_weight<T>(p, k0, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double y = h[i] * inv * double(w[i]);  // past K zero, or NaN like the row
        odd[i] = to_odd(y);
        if constexpr (sizeof(T) == 4)
            nearest[i] = float(y);
    }
    // The elements that f32 has no normal number for.  Looking for them costs bf16 rows with y
    // 3 to 6 % (8192 x 2048 28.1 us, so 28.9), the 8-bit rows, by their scale, nothing.
    const auto small = [&](float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fabsf(x[i]) <= 0x1p-126f)
                x[i] = to_odd_small(h[i] * inv * double(w[i]));
    };
    if (p.y) {
        T *out = static_cast<T *>(p.y) + row * p.ldy;
        if constexpr (sizeof(T) == 4) {
            store8<kSecond<T>, true>(out, k0, p.K, nearest);
        } else {
            float least = fabsf(odd[0]);
#pragma unroll
            for (int i = 1; i < 8; ++i)
                least = __builtin_amdgcn_fmed3f(least, fabsf(odd[i]), 0.0f);  // the smaller
            if (least <= 0x1p-126f)
                small(odd);
            store8<kSecond<T>, true>(out, k0, p.K, odd);
        }
    }
    if (p.codes)
        pack_group<T>(odd, p.codes + row * groups * kGroup, p.scales + row * fp8_scale_bytes(p.K),
                      piece >> 4, groups, piece & 15, small);
}

// A row's threads (64, 256 or 1024) hold it in registers, PIECES times eight
// elements each, so x and r are read once.  Bound by HBM, and in bf16 nearly by the 64-bit
// conversions: 8192 x 2048 with residual from cold memory takes 27.0 us in bf16, 4.4 TB/s,
// and 39.7 in f32, 5.5 (a lane's eight elements in a row 41.8).  f32 arithmetic, whose rows
// differ from the 64-bit result's in one of 10^7 codes, takes 2 us less of 24 where all is in
// the last-level cache; the weights loaded before the sum over the row 2 us more: registers,
// and with them waves.
template <typename T, int THREADS, int PIECES>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void add_rmsnorm_kernel(NormArgs p)
{
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x % THREADS;
    const int64_t row = THREADS < 256 ? int64_t(blockIdx.x) * (256 / THREADS) +
                                            threadIdx.x / THREADS
                                      : int64_t(blockIdx.x);
    if (row >= p.rows)
        return;  // whole waves: one wave per row where a workgroup has several
    const int groups = int(fp8_groups(p.K));
    double h[PIECES][8];
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int k0 = run_of<T>(j * THREADS + tid);
        float s[8];
        load_sum<T>(p, row, k0, h[j], s);
        store_sum<T>(p, row, k0, s);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            ss = fma(h[j][i], h[j][i], ss);
    }
    ss = wave_sum(ss);
    if constexpr (WAVES > 1) {
        __shared__ double part[WAVES];
        if ((tid & 63) == 0)
            part[tid >> 6] = ss;
        __syncthreads();
        ss = part[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            ss += part[w];
    }
    const double inv = inv_sqrt(ss / p.K + double(p.eps));
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
        if (((j * THREADS + tid) >> 4) < groups)
            store_normed<T>(p, row, j * THREADS + tid, h[j], inv, groups);
}

// Longer rows: a workgroup reads its row twice (250 x 32768 f32: 32.2 us, in registers 24.5).  Writes follow the second read
// of the same elements by the same thread, so that outputs may be the inputs.
template <typename T>
__global__ __launch_bounds__(1024) void add_rmsnorm_long_kernel(NormArgs p)
{
    __shared__ double part[16];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const int groups = int(fp8_groups(p.K));
    const int pieces = groups * 16;
    double ss = 0.0;
    for (int piece = tid; piece < pieces; piece += 1024) {
        double h[8];
        float s[8];
        load_sum<T>(p, row, run_of<T>(piece), h, s);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            ss = fma(h[i], h[i], ss);
    }
    ss = wave_sum(ss);
    if ((tid & 63) == 0)
        part[tid >> 6] = ss;
    __syncthreads();
    ss = part[0];
#pragma unroll
    for (int w = 1; w < 16; ++w)
        ss += part[w];
    const double inv = inv_sqrt(ss / p.K + double(p.eps));
    for (int piece = tid; piece < pieces; piece += 1024) {
        double h[8];
        float s[8];
        load_sum<T>(p, row, run_of<T>(piece), h, s);
        store_sum<T>(p, row, run_of<T>(piece), s);
        store_normed<T>(p, row, piece, h, inv, groups);
    }
}

// Groups of a call, 16 threads each, in one launch of at most 2^32 threads.
bool group_count(const char *who, int64_t rows, int64_t groups, unsigned &total)
{
    constexpr int64_t most = (int64_t(1) << 28) - 16;
    if (groups > 0 && rows > most / groups)
        return fail(std::string(who) + ": too many elements");
    total = unsigned(rows * groups);
    return true;
}

// The runtime counts the threads of a launch in 32 bits.
bool norm_grid(int64_t blocks, int threads, dim3 &grid)
{
    if (blocks > UINT32_MAX / threads)
        return fail("add_rmsnorm_fp8_dev: too many rows for one launch");
    grid = dim3(unsigned(blocks));
    return true;
}

template <typename T, int THREADS, int PIECES>
bool run_norm(const NormArgs &p, hipStream_t st)
{
    constexpr int PER = THREADS < 256 ? 256 / THREADS : 1;  // rows of a workgroup
    const dim3 block(THREADS < 256 ? 256 : THREADS);
    dim3 grid;
    if (!norm_grid((p.rows + PER - 1) / PER, block.x, grid))
        return false;
    hipLaunchKernelGGL((add_rmsnorm_kernel<T, THREADS, PIECES>), grid, block, 0, st, p);
    return hip_ok(hipGetLastError(), "add_rmsnorm_kernel launch");
}

template <typename T>
bool launch_norm(const NormArgs &p, hipStream_t st)
{
    // 30000 x 512 bf16: 22.2 us, by 256 threads a row 39.8; one row of 2048 3.0 us, by 64 5.4.
    if (p.K <= 512)
        return run_norm<T, 64, 1>(p, st);
    if (p.K <= 2048)
        return run_norm<T, 256, 1>(p, st);
    // A row a CU at most: latency counts (3 x 8192 bf16: 4.3 us, by 256 threads a row 6.2; 4096 x
    // 4096 30.3 and 22.7).
    if (p.K <= 8192 && p.rows <= 256)
        return run_norm<T, 1024, 1>(p, st);
    if (p.K <= 4096)
        return run_norm<T, 256, 2>(p, st);
    if (p.K <= 8192)
        return run_norm<T, 256, 4>(p, st);
    if (p.K <= 16384)
        return run_norm<T, 1024, 2>(p, st);
    if (p.K <= 32768)
        return run_norm<T, 1024, 4>(p, st);
    dim3 grid;
    if (!norm_grid(p.rows, 1024, grid))
        return false;
    hipLaunchKernelGGL(add_rmsnorm_long_kernel<T>, grid, dim3(1024), 0, st, p);
    return hip_ok(hipGetLastError(), "add_rmsnorm_long_kernel launch");
}

}  // namespace

bool launch_fp8_pack(const void *x, int64_t ldx, Mx4Type type, uint8_t *codes, uint8_t *scales,
                     int64_t rows, int K, hipStream_t st)
{
    const unsigned groups = unsigned(fp8_groups(K));
    unsigned total = 0;
    if (!group_count("fp8_pack_dev", rows, groups, total))
        return false;
    if (total == 0)
        return true;
    const dim3 grid((total + 15) / 16), block(256);
    if (type == kMx4F32)
        hipLaunchKernelGGL(fp8_pack_kernel<float>, grid, block, 0, st,
                           static_cast<const float *>(x), ldx, codes, scales, groups, total, K);
    else
        hipLaunchKernelGGL(fp8_pack_kernel<uint16_t>, grid, block, 0, st,
                           static_cast<const uint16_t *>(x), ldx, codes, scales, groups, total, K);
    return hip_ok(hipGetLastError(), "fp8_pack_kernel launch");
}

bool launch_fp8_unpack(const uint8_t *codes, const uint8_t *scales, void *x, int64_t ldx,
                       Mx4Type type, int64_t rows, int K, hipStream_t st)
{
    const unsigned groups = unsigned(fp8_groups(K));
    unsigned total = 0;
    if (!group_count("fp8_unpack_dev", rows, groups, total))
        return false;
    if (total == 0)
        return true;
    const dim3 grid((total + 15) / 16), block(256);
    const bool stream = flash_tile::aligned(x, 128) && ldx % (type == kMx4F32 ? 32 : 64) == 0;
    const auto launch = [&](auto kernel, auto *out) {
        hipLaunchKernelGGL(kernel, grid, block, 0, st, codes, scales, out, ldx, groups, total, K);
    };
    if (type == kMx4F32)
        launch(stream ? fp8_unpack_kernel<float, true> : fp8_unpack_kernel<float, false>,
               static_cast<float *>(x));
    else
        launch(stream ? fp8_unpack_kernel<uint16_t, true> : fp8_unpack_kernel<uint16_t, false>,
               static_cast<uint16_t *>(x));
    return hip_ok(hipGetLastError(), "fp8_unpack_kernel launch");
}

bool launch_add_rmsnorm_fp8(const AddRmsNorm &a, hipStream_t st)
{
    if (a.rows <= 0 || a.K <= 0)
        return true;
    NormArgs p{};
    p.x = a.x;
    p.r = a.residual;
    p.w = a.w;
    p.sum = a.sum;
    p.y = a.y;
    p.codes = a.codes;
    p.scales = a.scales;
    p.ldx = a.ldx;
    p.ldr = a.ldr;
    p.lds = a.ldsum;
    p.ldy = a.ldy;
    p.rows = a.rows;
    p.K = a.K;
    p.eps = a.eps;
    return a.type == kMx4F32 ? launch_norm<float>(p, st) : launch_norm<uint16_t>(p, st);
}

}  // namespace anima_hip
