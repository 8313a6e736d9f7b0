// Products in 8-bit integers with one scale per position (row of x) and per channel (row of w):
//
//     s_i  = fl(max_k |x_ik| / 127)           q_ik = rint(fl(x_ik / s_i))          afb_quantize_rows
//     y_ij = (sum_k q_ik w_jk) s_i t_j + b_j                                       afb_int8_matmul
//
// fl is the float32 rounding, rint goes to the nearest even.  The sum is exact: |q w| <= 2^14, so int32 holds
// kMaxK = 2^17 - 1 of them.  A row of zeros has s = 0 and q = 0; a row that holds an infinity or a NaN has
// s = NaN and q = 0, so its results are NaN and no other row's.
//
// quantize_rows_kernel, quantize_columns_kernel: one pass for the largest magnitude (integer maxima of the
//   magnitudes' bits, which order like the magnitudes and put NaN on top) and one that divides and packs; the
//   second finds its data in cache.
// dot_kernel: one warp per channel and up to kRows rows, the rows' 8-bit values in shared memory, __dp4a.
#include "dtypes.cuh"

namespace afb {
namespace {

constexpr int kMaxK = 131071;                   // 2^14 (2^17 - 1) < 2^31
constexpr float kTop = 127.f;
constexpr unsigned kInfBits = 0x7f800000u;

__device__ __forceinline__ float row_scale(unsigned amax_bits) {
    return amax_bits >= kInfBits ? __uint_as_float(0x7fc00000u) : __fdiv_rn(__uint_as_float(amax_bits), kTop);
}
// The quotient is within 127 (1 + 2^-23) unless the scale is subnormal, where it can round further up.
__device__ __forceinline__ int quantize_one(float x, float scale) {
    if (!(scale > 0.f)) return 0;
    return (int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -kTop), kTop);
}
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// RunningNorm in eval mode, as the readout applies it; without statistics the value itself.
struct Norm {
    const float *mean, *var;
    float eps, clip;
    __device__ __forceinline__ float operator()(float x, int64_t k) const {
        if (!mean) return x;
        return fminf(fmaxf((x - mean[k]) / sqrtf(var[k] + eps), -clip), clip);
    }
};

constexpr int kRowThreads = 128;

// One CTA per row of x (element (i, k) at x[i ld + k]).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(int64_t k_dim, const T *__restrict__ x, int64_t ld, Norm norm,
                                                                    int8_t *__restrict__ q, int64_t ld_q,
                                                                    float *__restrict__ scale) {
    __shared__ unsigned amax;
    const int64_t i = blockIdx.x;
    const T *row = x + i * ld;
    if (threadIdx.x == 0) amax = 0u;
    __syncthreads();
    unsigned m = 0u;
    for (int64_t k = threadIdx.x; k < k_dim; k += kRowThreads) m = max(m, magnitude(norm(to_float(row[k]), k)));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) atomicMax(&amax, m);
    __syncthreads();
    const float s = row_scale(amax);
    if (threadIdx.x == 0) scale[i] = s;
    for (int64_t k = threadIdx.x; k < k_dim; k += kRowThreads)
        q[i * ld_q + k] = (int8_t)quantize_one(norm(to_float(row[k]), k), s);
}

constexpr int kColRows = 32;                    // rows of the result per CTA, one per lane
constexpr int kColWarps = 16;
constexpr int kColK = 64;                       // k per shared tile

// The transposed layout: element (i, k) at x[k ld + i].  A CTA takes kColRows rows; lanes run along them.
template <typename T>
__global__ void __launch_bounds__(32 * kColWarps) quantize_columns_kernel(int64_t rows, int64_t k_dim, const T *__restrict__ x,
                                                                          int64_t ld, Norm norm, int8_t *__restrict__ q,
                                                                          int64_t ld_q, float *__restrict__ scale) {
    __shared__ unsigned amax[kColRows];
    __shared__ int8_t tile[kColRows][kColK + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t i0 = (int64_t)blockIdx.x * kColRows, i = i0 + lane;
    if (threadIdx.x < kColRows) amax[threadIdx.x] = 0u;
    __syncthreads();
    unsigned m = 0u;
    if (i < rows)
        for (int64_t k = warp; k < k_dim; k += kColWarps) m = max(m, magnitude(norm(to_float(x[k * ld + i]), k)));
    atomicMax(&amax[lane], m);
    __syncthreads();
    const float s = row_scale(amax[lane]);
    if (warp == 0 && i < rows) scale[i] = s;
    for (int64_t k0 = 0; k0 < k_dim; k0 += kColK) {
        for (int kk = warp; kk < kColK; kk += kColWarps) {
            const int64_t k = k0 + kk;
            tile[lane][kk] = (i < rows && k < k_dim) ? (int8_t)quantize_one(norm(to_float(x[k * ld + i]), k), s) : (int8_t)0;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < kColRows * kColK; e += 32 * kColWarps) {
            const int r = e / kColK, kk = e % kColK;
            if (i0 + r < rows && k0 + kk < k_dim) q[(i0 + r) * ld_q + k0 + kk] = tile[r][kk];
        }
        __syncthreads();
    }
}

constexpr int kDotWarps = 8;
constexpr int kDotRows = 8;

// y rows [kDotRows blockIdx.y, ...), channels [kDotWarps blockIdx.x, ...): one warp per channel.  Rows of q and w
// start on 16 bytes; the 16-byte words past k_dim are not read, and the last word's bytes past it are cleared.
template <typename O>
__global__ void __launch_bounds__(32 * kDotWarps) dot_kernel(int64_t rows, int64_t n, int k_dim, const int8_t *__restrict__ q,
                                                             int64_t ld_q, const float *__restrict__ q_scale,
                                                             const int8_t *__restrict__ w, int64_t ld_w,
                                                             const float *__restrict__ w_scale, const float *__restrict__ bias,
                                                             O *__restrict__ y, int64_t ld_y) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * kDotWarps + warp, i0 = (int64_t)blockIdx.y * kDotRows;
    if (j >= n) return;
    int acc[kDotRows] = {};
    const int full = k_dim & ~3;
    const int8_t *wr = w + j * ld_w;
    for (int k = lane * 4; k < full; k += 128) {
        const int wv = *reinterpret_cast<const int *>(wr + k);
#pragma unroll
        for (int r = 0; r < kDotRows; ++r)
            if (i0 + r < rows) acc[r] = __dp4a(*reinterpret_cast<const int *>(q + (i0 + r) * ld_q + k), wv, acc[r]);
    }
    for (int k = full + lane; k < k_dim; k += 32)
#pragma unroll
        for (int r = 0; r < kDotRows; ++r)
            if (i0 + r < rows) acc[r] += (int)q[(i0 + r) * ld_q + k] * (int)wr[k];
#pragma unroll
    for (int r = 0; r < kDotRows; ++r) {
        const int v = __reduce_add_sync(0xffffffffu, acc[r]);
        if (lane == 0 && i0 + r < rows)
            y[(i0 + r) * ld_y + j] = from_float<O>(fmaf((float)v * w_scale[j], q_scale[i0 + r], bias ? bias[j] : 0.f));
    }
}

void check_rows16(const void *p, int64_t ld, const char *what) {
    AFB_CHECK((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 16 == 0, std::string(what) + " rows must start on 16-byte boundaries");
}

void quantize(int64_t rows, int64_t k, int type, const void *x, int64_t ld_x, int x_trans, const Norm &norm, int8_t *q,
              int64_t ld_q, float *scale, cudaStream_t s) {
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const T *src = static_cast<const T *>(x);
        if (x_trans) {
            const int64_t blocks = (rows + kColRows - 1) / kColRows;
            quantize_columns_kernel<T><<<(unsigned)blocks, 32 * kColWarps, 0, s>>>(rows, k, src, ld_x, norm, q, ld_q, scale);
        } else {
            quantize_rows_kernel<T><<<(unsigned)rows, kRowThreads, 0, s>>>(k, src, ld_x, norm, q, ld_q, scale);
        }
    });
    AFB_LAUNCHED();
}

void matmul(int64_t rows, int64_t n, int64_t k, const int8_t *q, int64_t ld_q, const float *q_scale, const int8_t *w, int64_t ld_w,
            const float *w_scale, const float *bias, void *y, int y_type, int64_t ld_y, int *, cudaStream_t s) {
    const dim3 grid((unsigned)((n + kDotWarps - 1) / kDotWarps), (unsigned)((rows + kDotRows - 1) / kDotRows));
    AFB_CHECK(grid.y < 65536, "too many rows for one launch");
    with_type(y_type, [&](auto t) {
        using O = decltype(t);
        dot_kernel<O><<<grid, 32 * kDotWarps, 0, s>>>(rows, n, (int)k, q, ld_q, q_scale, w, ld_w, w_scale, bias,
                                                      static_cast<O *>(y), ld_y);
    });
    AFB_LAUNCHED();
}

int64_t round16(int64_t k) { return (k + 15) / 16 * 16; }
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
    if (rows <= 0 || k <= 0) return 0;
    return align256((size_t)rows * round16(k)) + align256((size_t)rows * 4) + 256;
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
        AFB_CHECK(workspace && workspace_bytes >= afb_int8_linear_workspace(rows, k), "workspace too small (afb_int8_linear_workspace)");
        char *ws = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
        int8_t *q = reinterpret_cast<int8_t *>(ws);
        float *scale = reinterpret_cast<float *>(ws + align256((size_t)rows * round16(k)));
        const cudaStream_t s = as_stream(stream);
        quantize(rows, k, x_type, x, ld_x, x_trans, Norm{mean, var, eps, clip}, q, round16(k), scale, s);
        matmul(rows, n, k, q, round16(k), scale, w, ld_w, w_scale, bias, y, y_type, ld_y, status, s);
    });
}

}  // extern "C"
