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
#include <cstring>

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

// ---- the tensor-core product --------------------------------------------------------------------------------

constexpr int kHalf = 128;                       // channels per CTA of a pair
constexpr int kBK8 = 128;                        // k per stage: one 128-byte swizzle row
constexpr int kMmaK8 = 32;
constexpr int kRingBytes = 196608;               // 192 KB of stages, whatever the tile
constexpr int kSlotBytes = 2048;                 // an epilogue warp stages 32 channels x 16 (float32) or 32 rows

// A tile: 2 kHalf channels (MMA M) x kRows rows of y (MMA N).
template <int kRows>
struct Tile {
    static constexpr int a_bytes = kHalf * kBK8, b_bytes = kRows / 2 * kBK8, stage_bytes = a_bytes + b_bytes;
    static constexpr int stages = kRingBytes / stage_bytes;
    static constexpr int parts = kRows >= 128 ? 4 : 2;                    // epilogue warps per quarter of the TMEM lanes
    static constexpr int epi_warps = 4 * parts;
    static constexpr int threads = 64 + 32 * epi_warps;                  // warp 0 TMA, warp 1 MMA, the rest epilogue
    static constexpr int smem = stages * stage_bytes + epi_warps * kSlotBytes + 1024 /* barriers */ + 1024 /* alignment */;
    static constexpr uint32_t tmem_cols = 2 * kRows;
    static constexpr uint32_t idesc = tc::idesc_s8(2 * kHalf, kRows);
};

__device__ __forceinline__ void mma_pair_s8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

template <typename O, int kRows>
__global__ void __launch_bounds__(Tile<kRows>::threads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q,
                const __grid_constant__ CUtensorMap map_y, int rows, int n, int k_dim, const float *__restrict__ q_scale,
                const float *__restrict__ w_scale, const float *__restrict__ bias, O *__restrict__ y, int64_t ld_y, int n_tma,
                int *__restrict__ status) {
    using S = Tile<kRows>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;                        // stage s: w half, then q half
    const uint32_t staging = ring + S::stages * S::stage_bytes;          // a slot per epilogue warp
    const uint32_t bars = staging + S::epi_warps * kSlotBytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (S::stages + s); };
    auto tfull = [&](int b) { return bars + 8u * (2 * S::stages + b); };
    auto tempty = [&](int b) { return bars + 8u * (2 * S::stages + 2 + b); };
    const uint32_t tmem_slot = bars + 8u * (2 * S::stages + 4);
    unsigned char *const slot_ptr = smem_raw + (tmem_slot - raw);

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int n_kb = (k_dim + kBK8 - 1) / kBK8;
    const int m_tiles = (n + 2 * kHalf - 1) / (2 * kHalf);
    const int total = m_tiles * ((rows + kRows - 1) / kRows);
    const int first = (int)tc::cluster_id(), step = (int)tc::cluster_count();

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::stages; ++s) {
            tc::bar_init(full(s), 1);
            tc::bar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::bar_init(tfull(b), 1);
            tc::bar_init(tempty(b), 2 * S::epi_warps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
    }
    if (warp == 0) {                                                     // warp 0 of both CTAs allocates
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tmem_slot), "r"(S::tmem_cols)
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
            const int m0 = (t % m_tiles) * 2 * kHalf + (int)rank * kHalf, i0 = (t / m_tiles) * kRows + (int)rank * (kRows / 2);
            for (int kb = 0; kb < n_kb; ++kb) {
                if (use > 0 && !__all_sync(0xffffffffu, tc::wait_bar(empty(s), (use - 1) & 1, status))) {
                    if (issuer) tc::fail(status, 1);
                    ok = false;
                    break;
                }
                if (issuer) {
                    const uint32_t a_dst = ring + s * S::stage_bytes;
                    if (rank == 0) tc::bar_expect_tx(full(s), 2 * S::stage_bytes);
                    tc::tma_load_pair(a_dst, &map_w, kb * kBK8, m0, leader_bars + 8u * s);
                    tc::tma_load_pair(a_dst + S::a_bytes, &map_q, kb * kBK8, i0, leader_bars + 8u * s);
                }
                __syncwarp();
                if (++s == S::stages) s = 0, ++use;
            }
        }
    } else if (warp == 1 && rank == 0) {                                 // MMA issuer (leader): the whole warp, so that
        int it = 0, ti = 0;                                              // its state is uniform; one lane issues
        bool ok = true;
        const bool issuer = tc::elect_one();
        for (int t = first; t < total && ok; t += step, ++ti) {
            const int b = ti & 1, use_b = ti >> 1;
            if (use_b > 0 && !__all_sync(0xffffffffu, tc::wait_bar(tempty(b), (use_b - 1) & 1, status))) {
                if (issuer) tc::fail(status, 2);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const uint32_t d = tmem + (uint32_t)(b * kRows);
            for (int kb = 0; kb < n_kb; ++kb, ++it) {
                const int s = it % S::stages, use = it / S::stages;
                if (!__all_sync(0xffffffffu, tc::wait_bar(full(s), use & 1, status))) {
                    if (issuer) tc::fail(status, 4);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t a_src = ring + s * S::stage_bytes;
                const uint64_t a_desc = tc::smem_desc(a_src), b_desc = tc::smem_desc(a_src + S::a_bytes);
                // the last k block takes only the 32-wide steps that hold data; the others would add zero fill
                const int nj = min(kBK8 / kMmaK8, (k_dim - kb * kBK8 + kMmaK8 - 1) / kMmaK8);
                if (issuer) {
#pragma unroll
                    for (int j = 0; j < kBK8 / kMmaK8; ++j)              // a step of 32 bytes: 2 in the descriptor's units
                        if (j < nj) mma_pair_s8(d, a_desc + 2 * j, b_desc + 2 * j, S::idesc, (kb > 0 || j > 0) ? 1u : 0u);
                    tc::commit_both(empty(s));                           // the stage is free in both CTAs once these
                    if (kb == n_kb - 1) tc::commit_both(tfull(b));       // MMAs have read it; the accumulator is complete
                }
                __syncwarp();
            }
        }
    } else if (warp >= 2) {                                              // epilogue (both CTAs)
        const int quarter = warp & 3, part = (warp - 2) >> 2;            // lanes, and share of the tile's rows
        constexpr int kPart = kRows / S::parts;
        const uint32_t leader_tempty0 = tc::map_to(tempty(0), 0), leader_tempty1 = tc::map_to(tempty(1), 0);
        int ti = 0;
        for (int t = first; t < total; t += step, ++ti) {
            const int b = ti & 1, use_b = ti >> 1;
            const int m = (t % m_tiles) * 2 * kHalf + (int)rank * kHalf + quarter * 32 + lane, i0 = (t / m_tiles) * kRows + part * kPart;
            // this tile's scales, fetched while its products run: lane l holds those of rows 32 c + l
            const float ws = m < n ? w_scale[m] : 0.f, bm = m < n && bias ? bias[m] : 0.f;
            float qs[kPart / 32];
#pragma unroll
            for (int c = 0; c < kPart / 32; ++c) qs[c] = i0 + c * 32 + lane < rows ? q_scale[i0 + c * 32 + lane] : 0.f;
            if (!__all_sync(0xffffffffu, tc::wait_bar(tfull(b), use_b & 1, status))) {
                if (lane == 0) tc::fail(status, 8);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
            for (int c = 0; c < kPart / 32; ++c) {
                const int i = i0 + c * 32, left = rows - i;
                if (left <= 0) break;                                    // uniform over the warp
                uint32_t r[32];
                tc::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * kRows + part * kPart + c * 32), r);
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
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::tmem_cols) : "memory");
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

// Pairs of CTAs that the device holds at once (one CTA per SM).
int device_pairs() {
    static int pairs[64] = {0};
    int dev = 0;
    AFB_CUDA(cudaGetDevice(&dev));
    AFB_CHECK(dev >= 0 && dev < 64, "device index out of range");
    if (!pairs[dev]) {
        int sms = 0;
        AFB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        pairs[dev] = sms / 2;
    }
    return pairs[dev];
}

template <typename O, int kRows>
void launch_pairs(int64_t rows, int64_t n, int64_t k, const int8_t *q, int64_t ld_q, const float *q_scale, const int8_t *w,
                  int64_t ld_w, const float *w_scale, const float *bias, O *y, int64_t ld_y, int *status, cudaStream_t s) {
    using S = Tile<kRows>;
    CUtensorMap map_w, map_q, map_y;
    tc::encode_operand_s8(&map_w, w, n, k, ld_w, kHalf);
    tc::encode_operand_s8(&map_q, q, rows, k, ld_q, kRows / 2);
    // the channels that TMA stores: all but the last few, or none where y's rows do not start on 16 bytes
    const int unit = 16 / (int)sizeof(O);
    const int n_tma = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && ld_y % unit == 0 ? (int)n / unit * unit : 0;
    if (n_tma) encode_result(&map_y, y, rows, n_tma, ld_y);
    else std::memset(&map_y, 0, sizeof(map_y));
    const int64_t total = (n + 2 * kHalf - 1) / (2 * kHalf) * ((rows + kRows - 1) / kRows);
    AFB_CHECK(total < (1LL << 31), "too many rows for one launch");
    const int64_t pairs = std::min<int64_t>(total, device_pairs());
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
    cfg.blockDim = dim3(S::threads, 1, 1);
    cfg.dynamicSmemBytes = S::smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    AFB_CUDA(cudaFuncSetAttribute(pair_kernel<O, kRows>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem));
    AFB_CUDA(cudaLaunchKernelEx(&cfg, pair_kernel<O, kRows>, map_w, map_q, map_y, (int)rows, (int)n, (int)k, q_scale, w_scale,
                                bias, y, ld_y, n_tma, status));
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
            const float *w_scale, const float *bias, void *y, int y_type, int64_t ld_y, int *status, cudaStream_t s) {
    if (rows > kDotRows) {
        with_type(y_type, [&](auto t) {
            using O = decltype(t);
            O *out = static_cast<O *>(y);
            // the tile that takes the fewest rounds of its size; the wide one moves the fewest bytes a product
            const int64_t m_tiles = (n + 2 * kHalf - 1) / (2 * kHalf), pairs = device_pairs();
            auto cost = [&](int64_t r, int64_t unit) { return ((m_tiles * ((rows + r - 1) / r) + pairs - 1) / pairs) * unit; };
            const int64_t c256 = cost(256, 32), c128 = cost(128, 24), c64 = cost(64, 20);
            auto go = [&](auto tile) { launch_pairs<O, decltype(tile)::value>(rows, n, k, q, ld_q, q_scale, w, ld_w, w_scale, bias, out, ld_y, status, s); };
            if (c256 <= c128 && c256 <= c64) go(std::integral_constant<int, 256>{});
            else if (c128 <= c64) go(std::integral_constant<int, 128>{});
            else go(std::integral_constant<int, 64>{});
        });
        return;
    }
    const dim3 grid((unsigned)((n + kDotWarps - 1) / kDotWarps), (unsigned)((rows + kDotRows - 1) / kDotRows));
    AFB_CHECK(grid.y < 65536, "too many rows for one launch");
    with_type(y_type, [&](auto t) {
        using O = decltype(t);
        dot_kernel<O><<<grid, 32 * kDotWarps, 0, s>>>(rows, n, (int)k, q, ld_q, q_scale, w, ld_w, w_scale, bias,
                                                      static_cast<O *>(y), ld_y);
    });
    AFB_LAUNCHED();
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
        AFB_CHECK(workspace && workspace_bytes >= afb_int8_linear_workspace(rows, k), "workspace too small (afb_int8_linear_workspace)");
        char *ws = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
        int8_t *q = reinterpret_cast<int8_t *>(ws);
        float *scale = reinterpret_cast<float *>(ws + align256((size_t)rows * round128(k)));
        const cudaStream_t s = as_stream(stream);
        quantize(rows, k, x_type, x, ld_x, x_trans, Norm{mean, var, eps, clip}, q, round128(k), scale, s);
        matmul(rows, n, k, q, round128(k), scale, w, ld_w, w_scale, bias, y, y_type, ld_y, status, s);
    });
}

}  // extern "C"
