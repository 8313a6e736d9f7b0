// Products in 8-bit integers with one scale per position (row of x) and per channel (row of w):
//
//     s_i  = fl(max_k |x_ik| / 127)           q_ik = rint(fl(x_ik / s_i))          afb_quantize_rows
//     y_ij = (sum_k q_ik w_jk) s_i t_j + b_j                                       afb_int8_matmul
//
// fl is the float32 rounding, rint goes to the nearest even.  The sum is exact: |q w| <= 2^14, so int32 holds
// kMaxK = 2^17 - 1 of them.  A row of zeros has s = 0 and q = 0; a row that holds an infinity or a NaN has
// s = NaN and q = 0, so its results are NaN and no other row's.
//
// Kernels: quantize_rows_kernel and quantize_columns_kernel by the layout of x, dot_kernel for one row (quantisation and
// product in one launch), pair_kernel for the rest, on the tensor cores.  The largest magnitude of a row is an
// integer maximum of the magnitudes' bits, which order like the magnitudes and put NaN on top.
#include <cstring>
#include <type_traits>

#include "dtypes.cuh"
#include "tc.cuh"

namespace afb {
namespace {

constexpr int kMaxK = 131071;                   // 2^14 (2^17 - 1) < 2^31
constexpr float kTop = 127.f;
constexpr unsigned kInfBits = 0x7f800000u;

__device__ __forceinline__ float row_scale(unsigned amax_bits) {
    return amax_bits >= kInfBits ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(amax_bits), kTop);
}
// Four rint(fl(x / scale)) as bytes, by the division.  The quotient is within 127 (1 + 2^-23) unless the scale is
// subnormal, where it can round further up.  0 for a scale of 0 or NaN.
__device__ __noinline__ uint32_t quantize4_by_division(float x0, float x1, float x2, float x3, float scale) {
    const float x[4] = {x0, x1, x2, x3};
    uint32_t word = 0u;
    if (scale > 0.f)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            word |= ((uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x[e], scale)), -kTop), kTop) & 0xffu) << (8 * e);
    return word;
}
// The same with inv = fl(1 / scale).  t = x inv is off x / scale by less than 1.6e-5 (127 times two roundings), the
// rounded quotient by 7.6e-6: unless t lies within 4e-5 of a half, both round to the same whole number, which
// t + 1.5 2^23 holds in its low bits.  One element in 12,000 takes the division, and so do the scales whose reciprocal
// is infinite and rows without one (inv NaN).  Rounding and conversion instructions run at a quarter of the rate.
__device__ __forceinline__ uint32_t quantize4(float x0, float x1, float x2, float x3, float scale, float inv) {
    constexpr float kMagic = 12582912.f;
    const float x[4] = {x0, x1, x2, x3};
    float f[4];
    bool near = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t = x[e] * inv;
        f[e] = t + kMagic;
        near |= !(fabsf(t - (f[e] - kMagic)) < 0.49996f);
    }
    if (near) return quantize4_by_division(x0, x1, x2, x3, scale);
    return __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040),
                       __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040), 0x5410);
}
__device__ __forceinline__ float inverse(float scale) { return scale > 0.f ? 1.f / scale : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// RunningNorm in eval mode, as the readout applies it; without statistics the value itself.
struct Norm {
    const float *mean, *var;
    float eps, clip;
    __device__ __forceinline__ float operator()(float x, int64_t k) const {
        if (!mean) return x;
        const float v = (x - mean[k]) / sqrtf(var[k] + eps);
        return v < -clip ? -clip : v > clip ? clip : v;          // NaN stays NaN
    }
};

// The largest magnitude of the values it was given, as bits; 16-bit types two at a time (NaN stays).
template <typename T>
struct LargestOf {
    using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    Two two;
    __device__ __forceinline__ LargestOf() { two.x = two.y = from_float<T>(0.f); }
    __device__ __forceinline__ void add(const Piece<T> &v) {
#pragma unroll
        for (int h = 0; h < 4; ++h) two = __hmax2_nan(two, __habs2(*reinterpret_cast<const Two *>(&v.e[2 * h])));
    }
    __device__ __forceinline__ unsigned bits() const { return max(magnitude(to_float(two.x)), magnitude(to_float(two.y))); }
};
template <>
struct LargestOf<float> {
    unsigned m = 0u;
    __device__ __forceinline__ void add(const Piece<float> &v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, magnitude(v.e[e]));
    }
    __device__ __forceinline__ unsigned bits() const { return m; }
};

constexpr int kRowThreads = 128;

// One CTA per row of x (element (i, k) at x[i ld + k]), P pieces a thread.  The row is read in 16-byte pieces wherever it
// starts and kept in registers (kLong: read in spans, twice, the second time from cache); the quantised bytes are shifted
// to their place through shared memory and leave as 16-byte words, zero past k.  The statistics and the long rows have
// code of their own: with it in the loops they ran out of the instruction cache (35,840 x 2333 float32: 110 us against 76, 5.5 TB/s).
template <typename T, int P, bool kLong, bool kNorm>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(int k_dim, const T *__restrict__ x, int64_t ld, Norm norm,
                                                                    int8_t *__restrict__ q, int64_t ld_q, float *__restrict__ scale) {
    constexpr int kPer = Piece<T>::kPer, kSpan = kRowThreads * P * kPer;
    constexpr int kStep = kSpan - 16;            // elements a span writes: it starts up to 7 before its first
    __shared__ unsigned amax;
    __shared__ uint32_t bytes[kSpan / 4];
    const int64_t i = blockIdx.x;
    const T *row = x + i * ld;
    const int lead = lead_of(row);
    Piece<T> mine[P];
    auto first_of = [&](int base, int p) { return base + ((int)threadIdx.x + p * kRowThreads) * kPer - lead; };
    auto load = [&](int base) {                  // the pieces from element base - lead on
#pragma unroll
        for (int p = 0; p < P; ++p) mine[p] = first_of(base, p) < k_dim ? load_piece(row, first_of(base, p), k_dim, from_float<T>(0.f)) : Piece<T>();
    };
    // with statistics an element takes 32 bits, so it is normalised where it is used
    auto value = [&](int base, int p, int e) {
        const float v = to_float(mine[p].e[e]);
        const int k = first_of(base, p) + e;
        return kNorm && k >= 0 && k < k_dim ? norm(v, k) : v;
    };
    if (threadIdx.x == 0) amax = 0u;
    __syncthreads();
    LargestOf<T> largest;
    unsigned m = 0u;
    for (int base = 0; base < (kLong ? k_dim : 1); base += kStep) {
        load(base);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (kNorm) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) m = max(m, magnitude(value(base, p, e)));
            } else {
                largest.add(mine[p]);
            }
        }
    }
    m = __reduce_max_sync(0xffffffffu, max(m, largest.bits()));
    if ((threadIdx.x & 31) == 0) atomicMax(&amax, m);
    __syncthreads();
    const float s = row_scale(amax), inv = inverse(s);
    if (threadIdx.x == 0) scale[i] = s;
    for (int base = 0; base < (kLong ? k_dim : 1); base += kStep) {
        if (kLong) load(base);
#pragma unroll
        for (int p = 0; p < P; ++p)                                      // byte b of the span: element base - lead + b
#pragma unroll
            for (int w = 0; w < kPer / 4; ++w) {
                uint32_t word = 0u;
                if (first_of(base, p) < k_dim)
                    word = quantize4(value(base, p, 4 * w), value(base, p, 4 * w + 1), value(base, p, 4 * w + 2), value(base, p, 4 * w + 3), s, inv);
                bytes[(p * kRowThreads + threadIdx.x) * (kPer / 4) + w] = word;
            }
        __syncthreads();
        const int n = min(kStep, k_dim - base), by = 8 * (lead & 3);
        for (int b = threadIdx.x * 16; b < n; b += kRowThreads * 16) {
            uint32_t w[5];
#pragma unroll
            for (int e = 0; e < 5; ++e) w[e] = bytes[(b + lead) / 4 + e];
            *reinterpret_cast<uint4 *>(q + i * ld_q + base + b) =
                make_uint4(__funnelshift_r(w[0], w[1], by), __funnelshift_r(w[1], w[2], by), __funnelshift_r(w[2], w[3], by),
                           __funnelshift_r(w[3], w[4], by));
        }
        if (kLong) __syncthreads();
    }
}

constexpr int kColRows = 32;                     // rows of the result per cluster, one per lane
constexpr int kColWarps = 8;
constexpr int kColCluster = 8;                   // most CTAs of a cluster
constexpr int kColKeep = 40;                     // most values a thread keeps

// The transposed layout: element (i, k) at x[k ld + i], lanes along the rows i.  A cluster of up to 8 CTAs shares 32
// rows, each CTA a part of k; the CTAs' largest magnitudes meet through distributed shared memory.  Up to 320 values of k
// a CTA stay in registers, V a thread (beyond 2,560 they are read again, from cache); the bytes are transposed in shared
// memory.  35,840 x 2333 float32: 142 us (2.9 TB/s): a CTA reads, waits for its cluster, then writes.  308 us with statistics,
// a root and a division an element (365 in the row form, which takes them twice).
template <typename T, int V, bool kNorm>
__global__ void __launch_bounds__(32 * kColWarps, V > 24 ? 3 : 4)
    quantize_columns_kernel(int64_t rows, int k_dim, int share, const T *__restrict__ x, int64_t ld, Norm norm, int8_t *__restrict__ q,
                            int64_t ld_q, float *__restrict__ scale) {
    constexpr int kSpan = kColWarps * V, kWords = kSpan / 4;
    __shared__ unsigned amax[kColRows];
    __shared__ uint32_t tile[kColRows][kWords | 1];                      // an odd pitch: lanes write different banks
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ctas = (int)tc::cluster_size();
    const int64_t i0 = (int64_t)(blockIdx.x / ctas) * kColRows, i = i0 + lane;
    const int k0 = share * (int)tc::cluster_rank(), k1 = min(k0 + share, k_dim);
    if (threadIdx.x < kColRows) amax[threadIdx.x] = 0u;
    __syncthreads();
    const bool in = i < rows;
    const T *const column = x + min(i, rows - 1);                        // lanes past the rows read the last one
    float mine[V];
    auto k_of = [&](int p) { return (p / 4 * kColWarps + warp) * 4 + p % 4; };   // a thread's fours are neighbours in k
    auto load = [&](int base) {
#pragma unroll
        for (int p = 0; p < V; p += 4) {
            const int k = base + k_of(p);
            const T *const at = column + (int64_t)k * ld;
            if (k + 4 <= k1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) mine[p + j] = to_float(at[j * ld]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) mine[p + j] = k + j < k1 ? to_float(at[j * ld]) : 0.f;
            }
        }
        if (kNorm)
#pragma unroll
            for (int p = 0; p < V; ++p) {
                const int k = base + k_of(p);
                if (k < k1) mine[p] = norm(mine[p], k);
            }
    };
    unsigned m = 0u;
    for (int base = k0; base < k1; base += kSpan) {
        load(base);
#pragma unroll
        for (int p = 0; p < V; ++p) m = max(m, magnitude(mine[p]));
    }
    atomicMax(&amax[lane], m);
    if (ctas > 1) tc::cluster_sync();
    else __syncthreads();
    m = amax[lane];
    const uint32_t own = (uint32_t)__cvta_generic_to_shared(&amax[lane]);
    for (int c = 0; c < ctas && ctas > 1; ++c) {
        unsigned v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(tc::map_to(own, (uint32_t)c)) : "memory");
        m = max(m, v);
    }
    if (ctas > 1) tc::cluster_arrive();          // the maxima are read
    const float s = row_scale(m), inv = inverse(s);
    if (k0 == 0 && warp == 0 && in) scale[i] = s;
    for (int base = k0; base < k1; base += kSpan) {
        if (share > kSpan) {
            load(base);
            __syncthreads();                     // the tile's readers are done
        }
#pragma unroll
        for (int p = 0; p < V; p += 4) tile[lane][k_of(p) / 4] = quantize4(mine[p], mine[p + 1], mine[p + 2], mine[p + 3], s, inv);
        __syncthreads();
        const int words = (min(kSpan, k1 - base) + 15) / 16 * 4;         // whole 16-byte units, zero past k
        for (int r = warp; r < kColRows && i0 + r < rows; r += kColWarps)
            for (int w = lane; w < words; w += 32) *reinterpret_cast<uint32_t *>(q + (i0 + r) * ld_q + base + 4 * w) = tile[r][w];
    }
    __syncwarp();
    if (ctas > 1) tc::cluster_wait();            // no CTA ends while another may read its maxima
}

// ---- one row -------------------------------------------------------------------------------------------------

constexpr int kDotWarps = 8;
constexpr int kDotThreads = 32 * kDotWarps;
constexpr int kDotMost = 128 * 1024;             // longest row, in bytes of shared memory
constexpr int kAhead = 5;                        // 16-byte words of w a lane fetches before the row is at hand
constexpr int kFours = 4;                        // fours of x a thread keeps: rows up to 4,096

__device__ __forceinline__ int dot16(const uint4 &a, const uint4 &b, int acc) {
    acc = __dp4a((int)a.x, (int)b.x, acc);
    acc = __dp4a((int)a.y, (int)b.y, acc);
    acc = __dp4a((int)a.z, (int)b.z, acc);
    return __dp4a((int)a.w, (int)b.w, acc);
}

// y = x w^T for one row in one launch: every CTA quantises the row into shared memory (kFused; else copies it from q)
// while its first words of w are on the way, then each of its warps takes a channel at a time.  Bound by latency: two
// trips to memory and a barrier; w is 9.7 MB at 2333 x 4171, all of it in flight at once.
template <typename T, typename O, bool kFused>
__global__ void __launch_bounds__(kDotThreads) dot_kernel(int64_t n, int k_dim, const T *__restrict__ x, int64_t k_step, Norm norm,
                                                          const float *__restrict__ q_scale, const int8_t *__restrict__ w, int64_t ld_w,
                                                          const float *__restrict__ w_scale, const float *__restrict__ bias,
                                                          O *__restrict__ y) {
    extern __shared__ uint4 held[];              // the row in 16-byte words, zero past k_dim
    __shared__ unsigned amax;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = (k_dim + 15) / 16;
    const int64_t first = (int64_t)blockIdx.x * kDotWarps + warp, step = (int64_t)gridDim.x * kDotWarps;
    // w's last word may hold anything past k_dim: the row holds zeros there
    auto row_of = [&](int64_t j) { return reinterpret_cast<const uint4 *>(w + j * ld_w); };
    uint4 ahead[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
        ahead[a] = first < n && lane + 32 * a < words ? __ldg(row_of(first) + lane + 32 * a) : make_uint4(0u, 0u, 0u, 0u);
    float scale;
    if (kFused) {
        auto value = [&](int k) { return k < k_dim ? norm(to_float(x[k * k_step]), k) : 0.f; };
        const bool kept = k_dim <= kFours * 4 * kDotThreads;
        float mine[kFours][4];
        unsigned m = 0u;
        if (kept) {
#pragma unroll
            for (int f = 0; f < kFours; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[f][e] = value((f * kDotThreads + (int)threadIdx.x) * 4 + e);
#pragma unroll
            for (int f = 0; f < kFours; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = max(m, magnitude(mine[f][e]));
        } else {
            for (int k = threadIdx.x; k < k_dim; k += kDotThreads) m = max(m, magnitude(value(k)));
        }
        if (threadIdx.x == 0) amax = 0u;
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) atomicMax(&amax, m);
        __syncthreads();
        scale = row_scale(amax);
        const float inv = inverse(scale);
        uint32_t *const fours = reinterpret_cast<uint32_t *>(held);
        if (kept) {
#pragma unroll
            for (int f = 0; f < kFours; ++f) {
                const int at = f * kDotThreads + (int)threadIdx.x;
                if (at < words * 4) fours[at] = quantize4(mine[f][0], mine[f][1], mine[f][2], mine[f][3], scale, inv);
            }
        } else {
            for (int at = threadIdx.x; at < words * 4; at += kDotThreads)
                fours[at] = quantize4(value(at * 4), value(at * 4 + 1), value(at * 4 + 2), value(at * 4 + 3), scale, inv);
        }
    } else {
        scale = *q_scale;
        int8_t *const bytes = reinterpret_cast<int8_t *>(held);
        for (int k = threadIdx.x; k < words * 16; k += kDotThreads) bytes[k] = k < k_dim ? (int8_t)x[k] : (int8_t)0;
    }
    __syncthreads();
    for (int64_t j = first; j < n; j += step) {
        int acc = 0;
        if (j != first)
#pragma unroll
            for (int a = 0; a < kAhead; ++a) ahead[a] = lane + 32 * a < words ? __ldg(row_of(j) + lane + 32 * a) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (lane + 32 * a < words) acc = dot16(held[lane + 32 * a], ahead[a], acc);
        for (int c = lane + 32 * kAhead; c < words; c += 32) acc = dot16(held[c], __ldg(row_of(j) + c), acc);
        acc = __reduce_add_sync(0xffffffffu, acc);
        if (lane == 0) y[j] = from_float<O>(fmaf((float)acc * w_scale[j], scale, bias ? bias[j] : 0.f));
    }
}

// One row, which fits the shared memory of a CTA.  (Two rows are as fast on the tensor cores: 11.8 us at 2333 x 4171, where
// one row takes 7.2 here, most of it the quantisation that every CTA repeats.)
static_assert((kMaxK + 15) / 16 * 16 <= kDotMost, "the longest row");
bool one_row(int64_t rows) { return rows == 1; }

template <typename T, bool kFused>
void launch_dot(int64_t n, int64_t k, const T *x, int64_t k_step, const Norm &norm, const float *q_scale, const int8_t *w, int64_t ld_w,
                const float *w_scale, const float *bias, void *y, int y_type, cudaStream_t s) {
    const size_t shared = (size_t)((k + 15) / 16 * 16);
    with_type(y_type, [&](auto t) {
        using O = decltype(t);
        constexpr auto kernel = dot_kernel<T, O, kFused>;
        allow_shared<kernel>(shared);
        const int64_t ctas = std::min<int64_t>((n + kDotWarps - 1) / kDotWarps, resident<kernel>(kDotThreads, shared));
        kernel<<<(unsigned)ctas, kDotThreads, shared, s>>>(n, (int)k, x, k_step, norm, q_scale, w, ld_w, w_scale, bias, static_cast<O *>(y));
    });
    AFB_LAUNCHED();
}

// ---- the tensor-core product --------------------------------------------------------------------------------

constexpr int kHalf = 128;                       // channels per CTA of a pair
constexpr int kBK8 = 128;                        // k per stage: one 128-byte swizzle row
constexpr int kMmaK8 = 32;
constexpr int kRingBytes = 196608;               // 192 KB of stages, whatever the tile
constexpr int kSlotBytes = 2048;                 // an epilogue warp stages 32 channels x 16 (float32) or 32 rows

constexpr int kEpiParts = 4;                     // epilogue warps per quarter of the TMEM lanes
constexpr int kEpiWarps = 4 * kEpiParts;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;    // warp 0 TMA, warp 1 MMA, the rest epilogue
constexpr int kABytes = kHalf * kBK8;
constexpr int kMaxRows = 256, kRowStep = 32;     // rows of y per tile (MMA N)
constexpr int kMaxStages = kRingBytes / (kABytes + kRowStep / 2 * kBK8);
constexpr int kPairSmem = kRingBytes + kEpiWarps * kSlotBytes + 1024 /* barriers */ + 1024 /* alignment */;
constexpr uint32_t kTmemCols = 2 * kMaxRows;

__device__ __forceinline__ void mma_pair_s8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// y in tiles of 2 kHalf channels (MMA M) x tile_rows rows (MMA N), each a pair of CTAs' (cluster of two, two-SM MMA, M 256,
// K 32): the pipeline of the float16 input map, in 8 bits.  CTA r of a pair holds channels 128 r .. + 127 and half of the
// rows of every k block; per block an SM loads 16 KB of w and up to 16 KB of q for 4 MMAs of 128 cycles.  Channels lie
// along the TMEM lanes, so a row's results are one line.  Two accumulators alternate: the epilogue of a tile (16 warps:
// int32 to float32, scales, bias, one rounding) runs under the products of the next.  Persistent, channels fastest, so
// concurrent pairs share rows.  Bound by the tensor pipe in large products: 35,840 x 2333 -> 4171 in 207 to 220 us by the
// clock, 3,170 to 3,370 TOP/s (0.94 to 1.0 of twice the measured bf16 rate); by the store of y where k is short: 2,048 x 838
// -> 17937 in 34 us, 2.2 TB/s.
// Every wait is bounded and gives up once the status word is set; TMEM is always released.
template <typename O>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q,
                const __grid_constant__ CUtensorMap map_y, int tile_rows, int rows, int n, int k_dim, const float *__restrict__ q_scale,
                const float *__restrict__ w_scale, const float *__restrict__ bias, O *__restrict__ y, int64_t ld_y, int n_tma,
                int *__restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    const int stage_bytes = kABytes + tile_rows / 2 * kBK8, stages = kRingBytes / stage_bytes;
    const uint32_t idesc = tc::idesc_s8(2 * kHalf, tile_rows);
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;                        // stage s: w half, then q half
    const uint32_t staging = ring + kRingBytes;          // a slot per epilogue warp
    const uint32_t bars = staging + kEpiWarps * kSlotBytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };
    auto tfull = [&](int b) { return bars + 8u * (2 * kMaxStages + b); };
    auto tempty = [&](int b) { return bars + 8u * (2 * kMaxStages + 2 + b); };
    const uint32_t tmem_slot = bars + 8u * (2 * kMaxStages + 4);
    unsigned char *const slot_ptr = smem_raw + (tmem_slot - raw);

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int n_kb = (k_dim + kBK8 - 1) / kBK8;
    const int m_tiles = (n + 2 * kHalf - 1) / (2 * kHalf);
    const int total = m_tiles * ((rows + tile_rows - 1) / tile_rows);
    const int first = (int)tc::cluster_id(), step = (int)tc::cluster_count();

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            tc::bar_init(full(s), 1);
            tc::bar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::bar_init(tfull(b), 1);
            tc::bar_init(tempty(b), 2 * kEpiWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
    }
    if (warp == 0) {                                                     // warp 0 of both CTAs allocates
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    tc::cluster_sync();                                                  // both CTAs' barriers are initialised
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(slot_ptr);

    if (warp == 0) {                                                     // TMA producer (both CTAs), a converged warp
        const bool issuer = tc::elect_one();
        const uint32_t leader_bars = tc::map_to(bars, 0);                // `full` comes first
        int s = 0, use = 0;
        bool ok = true;
        for (int t = first; t < total && ok; t += step) {
            const int m0 = (t % m_tiles) * 2 * kHalf + (int)rank * kHalf, i0 = (t / m_tiles) * tile_rows + (int)rank * (tile_rows / 2);
            for (int kb = 0; kb < n_kb; ++kb) {
                if (use > 0 && !__all_sync(0xffffffffu, tc::wait_bar(empty(s), (use - 1) & 1, status))) {
                    if (issuer) tc::fail(status, 1);
                    ok = false;
                    break;
                }
                if (issuer) {
                    const uint32_t a_dst = ring + s * stage_bytes;
                    if (rank == 0) tc::bar_expect_tx(full(s), 2 * stage_bytes);
                    tc::tma_load_pair(a_dst, &map_w, kb * kBK8, m0, leader_bars + 8u * s);
                    tc::tma_load_pair(a_dst + kABytes, &map_q, kb * kBK8, i0, leader_bars + 8u * s);
                }
                __syncwarp();
                if (++s == stages) s = 0, ++use;
            }
        }
        // after a failure no copy may outlive the CTA: wait, with a limit, for the last of each stage (both CTAs' bytes)
        if (!ok && rank == 0)
            for (int d = 0; d < stages; ++d) {
                const int last = d < s ? use : use - 1;
                if (last >= 0) tc::bar_wait(full(d), last & 1);
            }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {                                 // MMA issuer (leader): the whole warp, so that
        int s = 0, use = 0, ti = 0;                                      // its state is uniform; one lane issues
        bool ok = true;
        const bool issuer = tc::elect_one();
        for (int t = first; t < total && ok; t += step, ++ti) {
            const int b = ti & 1, use_b = ti >> 1;
            if (use_b > 0 && !__all_sync(0xffffffffu, tc::wait_bar(tempty(b), (use_b - 1) & 1, status))) {
                if (issuer) tc::fail(status, 2);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const uint32_t d = tmem + (uint32_t)(b * kMaxRows);
            for (int kb = 0; kb < n_kb; ++kb) {
                if (!__all_sync(0xffffffffu, tc::wait_bar(full(s), use & 1, status))) {
                    if (issuer) tc::fail(status, 4);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t a_src = ring + s * stage_bytes;
                const uint64_t a_desc = tc::smem_desc(a_src), b_desc = tc::smem_desc(a_src + kABytes);
                // the last k block takes only the 32-wide steps that hold data; the others would add zero fill
                const int nj = min(kBK8 / kMmaK8, (k_dim - kb * kBK8 + kMmaK8 - 1) / kMmaK8);
                if (issuer) {
#pragma unroll
                    for (int j = 0; j < kBK8 / kMmaK8; ++j)              // a step of 32 bytes: 2 in the descriptor's units
                        if (j < nj) mma_pair_s8(d, a_desc + 2 * j, b_desc + 2 * j, idesc, (kb > 0 || j > 0) ? 1u : 0u);
                    tc::commit_both(empty(s));                           // the stage is free in both CTAs once these
                    if (kb == n_kb - 1) tc::commit_both(tfull(b));       // MMAs have read it; the accumulator is complete
                }
                __syncwarp();
                if (++s == stages) s = 0, ++use;
            }
        }
    } else if (warp >= 2) {                                              // epilogue (both CTAs)
        // lanes 32 quarter .. + 31; of the tile's 32-row chunks every kEpiParts-th
        const int quarter = warp & 3, part = (warp - 2) >> 2, chunks = tile_rows / 32;
        constexpr int kChunks = kMaxRows / 32 / kEpiParts;
        const uint32_t leader_tempty0 = tc::map_to(tempty(0), 0), leader_tempty1 = tc::map_to(tempty(1), 0);
        int ti = 0;
        for (int t = first; t < total; t += step, ++ti) {
            const int b = ti & 1, use_b = ti >> 1;
            const int m = (t % m_tiles) * 2 * kHalf + (int)rank * kHalf + quarter * 32 + lane, i0 = (t / m_tiles) * tile_rows + part * 32;
            // this tile's scales, fetched while its products run: lane l holds its chunks' l-th rows'
            const float ws = m < n ? w_scale[m] : 0.f, bm = m < n && bias ? bias[m] : 0.f;
            float qs[kChunks];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int i = i0 + c * kEpiParts * 32 + lane;
                qs[c] = part + c * kEpiParts < chunks && i < rows ? q_scale[i] : 0.f;
            }
            if (!__all_sync(0xffffffffu, tc::wait_bar(tfull(b), use_b & 1, status))) {
                if (lane == 0) tc::fail(status, 8);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int i = i0 + c * kEpiParts * 32, left = rows - i;
                if (part + c * kEpiParts >= chunks || left <= 0) break;  // uniform over the warp
                uint32_t r[32];
                tc::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * kMaxRows + (part + c * kEpiParts) * 32), r);
                tc::tmem_wait_ld();
                O v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    v[j] = from_float<O>(fmaf((float)(int)r[j] * ws, __shfl_sync(0xffffffffu, qs[c], j), bm));
                // lanes run along the channels: one row of the chunk is one line, in shared memory or of y
                if (n_tma > 0) {
                    constexpr int kSlotRows = kSlotBytes / (32 * (int)sizeof(O));
#pragma unroll
                    for (int h = 0; h < 32 / kSlotRows; ++h) {
                        O *const dst = reinterpret_cast<O *>(smem_raw + (staging - raw) + (warp - 2) * kSlotBytes) + lane;
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");   // the slot is free
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < kSlotRows; ++j) dst[j * 32] = v[h * kSlotRows + j];
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0 && m < n_tma && h * kSlotRows < left)   // what lies past the map is clipped
                            tc::tma_store(&map_y, m, i + h * kSlotRows, staging + (uint32_t)(warp - 2) * kSlotBytes);
                        if (lane == 0) asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
                    }
                }
                if (m >= n_tma && m < n) {
                    O *const out = y + (int64_t)i * ld_y + m;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (j < left) out[j * ld_y] = v[j];
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::arrive_remote_relaxed(b ? leader_tempty1 : leader_tempty0);          // this accumulator is drained
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    tc::cluster_sync();                                                  // both CTAs are done with TMEM and barriers
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// y: rows x n elements of O (n whole 16-byte units: a store rounds its row up to one), row stride ld, boxes of one staging slot (32 channels).
template <typename O>
void encode_result(CUtensorMap *map, O *y, int64_t rows, int64_t n, int64_t ld) {
    const cuuint64_t dim[2] = {(cuuint64_t)n, (cuuint64_t)rows};
    const cuuint64_t stride[1] = {(cuuint64_t)ld * sizeof(O)};
    const cuuint32_t box[2] = {32u, (cuuint32_t)(kSlotBytes / (32 * sizeof(O)))};
    const cuuint32_t estride[2] = {1, 1};
    const CUtensorMapDataType type = sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    const CUresult r = tc::tensor_map_encoder()(map, type, 2, y, dim, stride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    AFB_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (result) failed with code " + std::to_string((int)r));
}

// The launch of pairs of CTAs, and how many pairs the current device holds at once (one CTA per SM).
struct PairLaunch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    explicit PairLaunch(cudaStream_t s) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.blockDim = dim3(kPairThreads, 1, 1);
        cfg.dynamicSmemBytes = kPairSmem;
        cfg.stream = s;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
};

template <typename O>
int device_pairs() {
    static std::mutex lock;
    static int pairs[kMaxDevices] = {0};
    const int dev = current_device();
    const std::lock_guard<std::mutex> held(lock);
    if (!pairs[dev]) {
        AFB_CUDA(cudaFuncSetAttribute(pair_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
        int sms = 0, n = 0;
        AFB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        PairLaunch launch(nullptr);
        launch.cfg.gridDim = dim3((unsigned)(sms / 2 * 2), 1, 1);
        AFB_CUDA(cudaOccupancyMaxActiveClusters(&n, pair_kernel<O>, &launch.cfg));
        AFB_CHECK(n >= 1, "no pair of CTAs of the 8-bit product fits on this device");
        pairs[dev] = n;
    }
    return pairs[dev];
}

// Rows of y per tile: the fewest rounds of tiles times the time of one, which is near proportional to 128 + r: 3.3,
// 4.2, 5.5 and 6.7 us a round at r = 64, 128, 192 and 256 and k = 2333.  1,120 x 2333 -> 4171 takes 17.0 us with the
// 160 rows that this gives and 19.3 with 256, which are the best for large products.
int pick_tile_rows(int64_t rows, int64_t n, int64_t pairs) {
    const int64_t m_tiles = (n + 2 * kHalf - 1) / (2 * kHalf);
    int best = kMaxRows;
    int64_t best_cost = INT64_MAX;
    for (int r = kMaxRows; r >= kRowStep; r -= kRowStep) {
        const int64_t cost = (m_tiles * ((rows + r - 1) / r) + pairs - 1) / pairs * (128 + r);
        if (cost < best_cost) best = r, best_cost = cost;
    }
    return best;
}

template <typename O>
void launch_pairs(int64_t rows, int64_t n, int64_t k, const int8_t *q, int64_t ld_q, const float *q_scale, const int8_t *w,
                  int64_t ld_w, const float *w_scale, const float *bias, O *y, int64_t ld_y, int *status, cudaStream_t s) {
    const int64_t pairs = device_pairs<O>();
    const int tile_rows = pick_tile_rows(rows, n, pairs);
    CUtensorMap map_w, map_q, map_y;
    tc::encode_operand_s8(&map_w, w, n, k, ld_w, kHalf);
    tc::encode_operand_s8(&map_q, q, rows, k, ld_q, (uint32_t)tile_rows / 2);
    // the channels that TMA stores: all but the last few, or none where y's rows do not start on 16 bytes
    const int unit = 16 / (int)sizeof(O);
    const int n_tma = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && ld_y % unit == 0 ? (int)n / unit * unit : 0;
    if (n_tma) encode_result(&map_y, y, rows, n_tma, ld_y);
    else std::memset(&map_y, 0, sizeof(map_y));
    const int64_t total = (n + 2 * kHalf - 1) / (2 * kHalf) * ((rows + tile_rows - 1) / tile_rows);
    AFB_CHECK(total < (1LL << 31), "too many rows for one launch");
    PairLaunch launch(s);
    launch.cfg.gridDim = dim3((unsigned)(2 * std::min(total, pairs)), 1, 1);
    AFB_CUDA(cudaLaunchKernelEx(&launch.cfg, pair_kernel<O>, map_w, map_q, map_y, tile_rows, (int)rows, (int)n, (int)k, q_scale, w_scale,
                                bias, y, ld_y, n_tma, status));
}

void check_rows16(const void *p, int64_t ld, const char *what) {
    AFB_CHECK((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 16 == 0, std::string(what) + " rows must start on 16-byte boundaries");
}

template <typename T>
void quantize_columns(int64_t rows, int k, const T *x, int64_t ld_x, const Norm &norm, int8_t *q, int64_t ld_q, float *scale, cudaStream_t s) {
    // as many CTAs a cluster as give each at most the values it can keep
    int ctas = 1;
    while (ctas < kColCluster && ctas * kColWarps * kColKeep < k) ctas *= 2;
    const int share = ((k + ctas - 1) / ctas + 15) / 16 * 16;            // whole 16-byte words
    const int64_t blocks = (rows + kColRows - 1) / kColRows * ctas;
    AFB_CHECK(blocks < (1LL << 31), "too many rows for one launch");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(32 * kColWarps, 1, 1);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (norm.mean) AFB_CUDA(cudaLaunchKernelEx(&cfg, quantize_columns_kernel<T, V, true>, rows, k, share, x, ld_x, norm, q, ld_q, scale));
        else AFB_CUDA(cudaLaunchKernelEx(&cfg, quantize_columns_kernel<T, V, false>, rows, k, share, x, ld_x, norm, q, ld_q, scale));
    };
    if (share <= kColWarps * 8) go(std::integral_constant<int, 8>{});
    else if (share <= kColWarps * 16) go(std::integral_constant<int, 16>{});
    else if (share <= kColWarps * 24) go(std::integral_constant<int, 24>{});
    else if (share <= kColWarps * 32) go(std::integral_constant<int, 32>{});
    else go(std::integral_constant<int, kColKeep>{});
}

void quantize(int64_t rows, int64_t k, int type, const void *x, int64_t ld_x, int x_trans, const Norm &norm, int8_t *q,
              int64_t ld_q, float *scale, cudaStream_t s) {
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const T *src = static_cast<const T *>(x);
        if (x_trans) {
            quantize_columns<T>(rows, (int)k, src, ld_x, norm, q, ld_q, scale, s);
            return;
        }
        // as few pieces a thread as hold the row wherever it starts
        const int64_t pieces = (k + 16) / Piece<T>::kPer + 1;
        auto go = [&](auto p, auto is_long) {
            constexpr int P = decltype(p)::value;
            constexpr bool kLong = decltype(is_long)::value;
            if (norm.mean) quantize_rows_kernel<T, P, kLong, true><<<(unsigned)rows, kRowThreads, 0, s>>>((int)k, src, ld_x, norm, q, ld_q, scale);
            else quantize_rows_kernel<T, P, kLong, false><<<(unsigned)rows, kRowThreads, 0, s>>>((int)k, src, ld_x, norm, q, ld_q, scale);
        };
        if (pieces <= kRowThreads) go(std::integral_constant<int, 1>{}, std::false_type{});
        else if (pieces <= 2 * kRowThreads) go(std::integral_constant<int, 2>{}, std::false_type{});
        else if (pieces <= 3 * kRowThreads) go(std::integral_constant<int, 3>{}, std::false_type{});
        else if (pieces <= 5 * kRowThreads) go(std::integral_constant<int, 5>{}, std::false_type{});
        else if (pieces <= 8 * kRowThreads) go(std::integral_constant<int, 8>{}, std::false_type{});
        else go(std::integral_constant<int, 8>{}, std::true_type{});
    });
    AFB_LAUNCHED();
}

void matmul(int64_t rows, int64_t n, int64_t k, const int8_t *q, int64_t ld_q, const float *q_scale, const int8_t *w, int64_t ld_w,
            const float *w_scale, const float *bias, void *y, int y_type, int64_t ld_y, int *status, cudaStream_t s) {
    if (one_row(rows)) {
        launch_dot<int8_t, false>(n, k, q, 1, Norm{}, q_scale, w, ld_w, w_scale, bias, y, y_type, s);
        return;
    }
    with_type(y_type, [&](auto t) {
        using O = decltype(t);
        launch_pairs<O>(rows, n, k, q, ld_q, q_scale, w, ld_w, w_scale, bias, static_cast<O *>(y), ld_y, status, s);
    });
}

// Rows of the quantised matrices in the workspace: a k-block of 128 bytes is then one line of L2 and not two.
int64_t round128(int64_t k) { return (k + 127) / 128 * 128; }
size_t align256(size_t b) { return (b + 255) / 256 * 256; }

void check_sizes(int64_t rows, int64_t n, int64_t k) {
    AFB_CHECK(rows >= 0 && n >= 0 && k >= 0, "negative size");
    AFB_CHECK(rows < (1LL << 31) && n < (1LL << 31), "size above 2^31");
    AFB_CHECK(k <= kMaxK, "k above 131071: the int32 sums could overflow");
}

void check_source(int64_t rows, int64_t k, int type, const void *x, int64_t ld_x, int x_trans, const float *mean, const float *var) {
    AFB_CHECK(known_type(type), "unknown element type");
    AFB_CHECK(x, "NULL pointer");
    AFB_CHECK((mean == nullptr) == (var == nullptr), "mean and var come together");
    AFB_CHECK(reinterpret_cast<uintptr_t>(x) % type_size(type) == 0, "x is not aligned to its elements");
    AFB_CHECK(ld_x >= (x_trans ? rows : k), "a leading dimension is below the row length");
}

void check_product(int64_t n, int64_t k, const void *w, int64_t ld_w, const float *w_scale, const void *y, int y_type, int64_t ld_y) {
    AFB_CHECK(known_type(y_type), "unknown element type");
    AFB_CHECK(w && w_scale && y, "NULL pointer");
    AFB_CHECK(ld_w >= k && ld_y >= n, "a leading dimension is below the row length");
    AFB_CHECK(reinterpret_cast<uintptr_t>(y) % type_size(y_type) == 0, "y is not aligned to its elements");
    check_rows16(w, ld_w, "w");
}

}  // namespace
}  // namespace afb

using namespace afb;

extern "C" {

int afb_quantize_rows(int64_t rows, int64_t k, int x_type, const void *x, int64_t ld_x, int x_trans, const float *mean,
                      const float *var, float eps, float clip, int8_t *q, int64_t ld_q, float *scale, void *stream) {
    return guarded([&] {
        check_sizes(rows, 0, k);
        if (rows == 0) return;
        AFB_CHECK(scale, "NULL pointer");
        if (k == 0) {
            AFB_CUDA(cudaMemsetAsync(scale, 0, (size_t)rows * 4, as_stream(stream)));
            return;
        }
        AFB_CHECK(q, "NULL pointer");
        AFB_CHECK(ld_q >= k, "a leading dimension is below the row length");
        check_rows16(q, ld_q, "q");
        check_source(rows, k, x_type, x, ld_x, x_trans, mean, var);
        quantize(rows, k, x_type, x, ld_x, x_trans, Norm{mean, var, eps, clip}, q, ld_q, scale, as_stream(stream));
    });
}

int afb_int8_matmul(int64_t rows, int64_t n, int64_t k, const int8_t *q, int64_t ld_q, const float *q_scale, const int8_t *w,
                    int64_t ld_w, const float *w_scale, const float *bias, void *y, int y_type, int64_t ld_y, int *status,
                    void *stream) {
    return guarded([&] {
        check_sizes(rows, n, k);
        if (rows == 0 || n == 0) return;
        AFB_CHECK(k >= 1, "k must be positive");
        AFB_CHECK(q && q_scale, "NULL pointer");
        AFB_CHECK(ld_q >= k, "a leading dimension is below the row length");
        check_rows16(q, ld_q, "q");
        check_product(n, k, w, ld_w, w_scale, y, y_type, ld_y);
        matmul(rows, n, k, q, ld_q, q_scale, w, ld_w, w_scale, bias, y, y_type, ld_y, status, as_stream(stream));
    });
}

size_t afb_int8_linear_workspace(int64_t rows, int64_t k) {
    if (rows <= 0 || k <= 0 || one_row(rows)) return 0;
    return align256((size_t)rows * round128(k)) + align256((size_t)rows * 4) + 256;
}

int afb_int8_linear(int64_t rows, int64_t n, int64_t k, int x_type, const void *x, int64_t ld_x, int x_trans, const float *mean,
                    const float *var, float eps, float clip, const int8_t *w, int64_t ld_w, const float *w_scale,
                    const float *bias, void *y, int y_type, int64_t ld_y, void *workspace, size_t workspace_bytes, int *status,
                    void *stream) {
    return guarded([&] {
        check_sizes(rows, n, k);
        if (rows == 0 || n == 0) return;
        AFB_CHECK(k >= 1, "k must be positive");
        check_source(rows, k, x_type, x, ld_x, x_trans, mean, var);
        check_product(n, k, w, ld_w, w_scale, y, y_type, ld_y);
        const size_t need = afb_int8_linear_workspace(rows, k);
        AFB_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace too small (afb_int8_linear_workspace)");
        const Norm norm{mean, var, eps, clip};
        if (one_row(rows)) {
            with_type(x_type, [&](auto t) {
                using T = decltype(t);
                launch_dot<T, true>(n, k, static_cast<const T *>(x), x_trans ? ld_x : 1, norm, nullptr, w, ld_w, w_scale, bias, y, y_type,
                                    as_stream(stream));
            });
            return;
        }
        char *ws = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
        int8_t *q = reinterpret_cast<int8_t *>(ws);
        float *scale = reinterpret_cast<float *>(ws + align256((size_t)rows * round128(k)));
        const cudaStream_t s = as_stream(stream);
        quantize(rows, k, x_type, x, ld_x, x_trans, norm, q, round128(k), scale, s);
        matmul(rows, n, k, q, round128(k), scale, w, ld_w, w_scale, bias, y, y_type, ld_y, status, s);
    });
}

}  // extern "C"
