// Distillation from a teacher's best moves: their selection, and the loss of a student against them with its
// gradient.
//
// top_kernel: for each row of logits l over a support (all moves, or the row's listed moves) the k largest, ties to
//   the lowest move, and  log_rest = log sum exp(l / T)  over the support's moves that are not among them.  NaN and
//   -inf are outside the support.  One CTA per row.  A lower bound of the k-th largest comes from the largest value
//   of each of kGroups groups of moves (k different moves are at least the k-th largest of those); the moves at or
//   above the bound are collected and ranked by counting.
// loss_kernel: with p the teacher's distribution over its named moves C (softmax of t / T; with `rest` one more
//   outcome, any other move, at exp(log_rest)) and q = softmax(s / T) of the student over its support,
//       loss = T^2 sum_c p_c (log p_c - log q_c)                          q_rest = the sum of q outside C
//       dloss / ds_j = T (q_j - p_j)  in C,   T q_j (1 - p_rest / q_rest)  outside C,  0 outside the support.
//   The shares of C and of the rest come from the log odds d = lse(C) - lse(rest) as log share(rest) =
//   -log(1 + exp(d)), so that neither the loss nor the gradient takes a difference of nearly equal sums.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "dtypes.cuh"

namespace afb {
namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 256;                    // largest k
constexpr int kMaxListed = 4096;                // longest list of moves
constexpr int64_t kMaxMoves = 1 << 20;          // the bitmap of a row's moves fits in shared memory
constexpr int kGroups = 512;                    // at least kMaxTop
constexpr int kCandidates = 1024;
static_assert(kGroups >= kMaxTop && kCandidates >= kMaxTop, "k groups and k candidates");

// Order of the values as unsigned integers, -0 and +0 alike; 0 for what is never selected (NaN, -inf).
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x > -kInf)) return 0u;
    const unsigned b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

template <typename F>
__device__ __forceinline__ float warp_reduce(float x, F &&f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
// The same value in every thread; `scratch` holds kWarps floats and may be used again after the next barrier.
template <typename F>
__device__ __forceinline__ float block_reduce(float x, float *scratch, float unit, F &&f) {
    x = warp_reduce(x, f);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = unit;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) x = f(x, scratch[w]);
    return x;
}
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
__device__ __forceinline__ int block_count(int x, int *scratch) {
    x = __reduce_add_sync(0xffffffffu, x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) x += scratch[w];
    return x;
}

// A row's list: moves[l] the l-th listed move, -1 where it does not take part (not valid, out of range, or named before
// in the list), values[l] its logit.  `bitmap` (n_words) comes back with the moves' bits.
template <typename T>
__device__ void read_list(const int64_t *list, const uint8_t *valid, int n_listed, int64_t n_moves, const T *row, unsigned *bitmap,
                          int n_words, int *moves, float *values) {
    for (int w = threadIdx.x; w < n_words; w += kThreads) bitmap[w] = 0u;
    __syncthreads();
    int again = 0;
    for (int l = threadIdx.x; l < n_listed; l += kThreads) {
        const int64_t m = list[l];
        const bool in = valid[l] && m >= 0 && m < n_moves;
        moves[l] = in ? (int)m : -1;
        if (!in) continue;
        const unsigned bit = 1u << (m & 31);
        again |= (atomicOr(&bitmap[m >> 5], bit) & bit) != 0u;
        values[l] = to_float(row[m]);
    }
    if (__syncthreads_or(again)) {               // rare: keep the first place of each move, whatever the order above
        for (int l0 = 0; l0 < n_listed; l0 += kThreads) {
            const int l = n_listed - 1 - l0 - (int)threadIdx.x;             // later places first: theirs are not looked at again
            bool drop = false;
            if (l >= 0 && moves[l] >= 0)
                for (int d = 0; d < l; ++d) drop |= moves[d] == moves[l];
            __syncthreads();
            if (drop) moves[l] = -1;
            __syncthreads();
        }
    }
}

struct TopShared {
    unsigned group[kGroups];
    unsigned long long cand[kCandidates];
    float scratch[kWarps];
    int iscratch[kWarps];
    int count;
    unsigned bound;
    unsigned long long last;                     // the key of the k-th selected
};

// A move's key: its value's order, then the lower move.  Distinct for distinct moves; 0 in the upper half: absent.
__device__ __forceinline__ unsigned long long key_of(unsigned order, int move) {
    return ((unsigned long long)order << 32) | (unsigned)~move;
}

// A lower bound of the k-th largest of the first G shared group maxima, in warp 0: bit by bit from the first in which they
// differ, the largest value that k of them reach, until few more than k do.
template <int G>
__device__ unsigned kth_of_groups(const unsigned *group, int k) {
    unsigned mine[G / 32], all = ~0u, any = 0u;
#pragma unroll
    for (int g = 0; g < G / 32; ++g) {
        mine[g] = group[g * 32 + (threadIdx.x & 31)];
        all &= mine[g];
        any |= mine[g];
    }
    all = __reduce_and_sync(0xffffffffu, all);
    any = __reduce_or_sync(0xffffffffu, any);
    if (all == any) return all;
    unsigned bit = 0x80000000u >> __clz(all ^ any), t = all & ~(2u * bit - 1u);
    for (int reach = G; bit && reach > k + k / 8; bit >>= 1) {
        const unsigned probe = t | bit;
        int c = 0;
#pragma unroll
        for (int g = 0; g < G / 32; ++g) c += mine[g] >= probe;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= k) t = probe, reach = c;
    }
    return t;
}

// Selects from `n` entries, get(e, order, move).  A row with too many entries at the bound (many equal values) finds
// the k-th key itself bit by bit.
template <int NT, typename Get>
__device__ void select_top(TopShared &sh, int n, int k, float inv_t, Get &&get, float *values, int64_t *moves, float *log_rest) {
    for (int g = threadIdx.x; g < kGroups; g += NT) sh.group[g] = 0u;
    if (threadIdx.x == 0) sh.count = 0;
    // entry e belongs to group e mod kGroups
    unsigned best[kGroups / NT] = {};
    for (int e0 = 0; e0 < n; e0 += kGroups)
#pragma unroll
        for (int h = 0; h < kGroups / NT; ++h) {
            const int e = e0 + h * NT + (int)threadIdx.x;
            if (e >= n) break;
            unsigned o;
            int m;
            get(e, o, m);
            best[h] = max(best[h], o);
        }
#pragma unroll
    for (int h = 0; h < kGroups / NT; ++h) sh.group[h * NT + threadIdx.x] = best[h];
    __syncthreads();
    if (threadIdx.x < 32) {
        const unsigned t = kth_of_groups<kGroups>(sh.group, k);
        if (threadIdx.x == 0) sh.bound = max(t, 1u);                      // 0: fewer than k groups hold a move
    }
    __syncthreads();
    unsigned bound = sh.bound;
    for (int e = threadIdx.x; e < n; e += NT) {
        unsigned o;
        int m;
        get(e, o, m);
        if (o >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCandidates) sh.cand[at] = key_of(o, m);
        }
    }
    __syncthreads();
    int found = sh.count;
    if (found > kCandidates) {
        unsigned long long t = 0ull;
        for (int b = 63; b >= 0; --b) {
            const unsigned long long probe = t | (1ull << b);
            int c = 0;
            for (int e = threadIdx.x; e < n; e += NT) {
                unsigned o;
                int m;
                get(e, o, m);
                c += o && key_of(o, m) >= probe;
            }
            if (block_count(c, sh.iscratch) >= k) t = probe;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        for (int e = threadIdx.x; e < n; e += NT) {
            unsigned o;
            int m;
            get(e, o, m);
            if (o && key_of(o, m) >= t) sh.cand[atomicAdd(&sh.count, 1)] = key_of(o, m);   // k of them
        }
        __syncthreads();
        found = sh.count;
    }
    if (threadIdx.x == 0) sh.last = 0ull;
    __syncthreads();
    for (int c = threadIdx.x; c < found; c += NT) {
        const unsigned long long key = sh.cand[c];
        int rank = 0;
        for (int d = 0; d < found; ++d) rank += sh.cand[d] > key;
        if (rank < k) {
            values[rank] = value_of((unsigned)(key >> 32));
            moves[rank] = (int64_t) ~(unsigned)key;
            if (rank == k - 1) sh.last = key;
        }
    }
    for (int r = found + threadIdx.x; r < k; r += NT) {
        values[r] = -kInf;
        moves[r] = -1;
    }
    __syncthreads();
    // what is left: nothing unless k moves were found
    const unsigned long long last = sh.last;
    float m = -kInf;
    if (last)
        for (int e = threadIdx.x; e < n; e += NT) {
            unsigned o;
            int mv;
            get(e, o, mv);
            if (o && key_of(o, mv) < last) m = fmaxf(m, value_of(o));
        }
    m = block_reduce(m, sh.scratch, -kInf, Max());
    float sum = 0.f;
    if (m > -kInf)
        for (int e = threadIdx.x; e < n; e += NT) {
            unsigned o;
            int mv;
            get(e, o, mv);
            if (o && key_of(o, mv) < last) sum += expf((value_of(o) - m) * inv_t);
        }
    sum = block_reduce(sum, sh.scratch, 0.f, Sum());
    if (threadIdx.x == 0) *log_rest = m > -kInf && m < kInf ? m * inv_t + logf(sum) : m;
}

// The rows' listed moves: all entries are at hand in shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) top_listed_kernel(int64_t n_moves, const T *__restrict__ logits, int64_t ld, int k, float inv_t,
                                                              const int64_t *__restrict__ list, const uint8_t *__restrict__ valid,
                                                              int n_listed, float *__restrict__ values, int64_t *__restrict__ moves,
                                                              float *__restrict__ log_rest) {
    extern __shared__ unsigned dynamic[];
    __shared__ TopShared sh;
    const int64_t i = blockIdx.x;
    const T *row = logits + i * ld;
    const int n_words = (int)((n_moves + 31) / 32);
    int *listed = reinterpret_cast<int *>(dynamic + n_words);
    float *at = reinterpret_cast<float *>(listed + n_listed);
    read_list(list + i * n_listed, valid + i * n_listed, n_listed, n_moves, row, dynamic, n_words, listed, at);
    select_top<kThreads>(sh, n_listed, k, inv_t, [&](int e, unsigned &o, int &m) { m = listed[e]; o = m < 0 ? 0u : order_of(at[e]); },
               values + i * k, moves + i * k, log_rest + i);
}

// 2^x; below 2^-126 it is 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

constexpr int kRanked = 96;                      // candidates that one warp ranks by itself

// The largest of each of four subsets of a thread's moves (a maximum passes NaN over); 16-bit types two at a time.
template <typename T>
struct FourMax {
    using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    Two two[4];
    __device__ __forceinline__ FourMax() {
#pragma unroll
        for (int h = 0; h < 4; ++h) two[h].x = two[h].y = from_float<T>(-kInf);
    }
    __device__ __forceinline__ void add(const Piece<T> &v) {
#pragma unroll
        for (int h = 0; h < 4; ++h) two[h] = __hmax2(two[h], *reinterpret_cast<const Two *>(&v.e[2 * h]));
    }
    __device__ __forceinline__ float get(int h) const { return fmaxf(to_float(two[h].x), to_float(two[h].y)); }
};
template <>
struct FourMax<float> {
    float one[4] = {-kInf, -kInf, -kInf, -kInf};
    __device__ __forceinline__ void add(const Piece<float> &v) {
#pragma unroll
        for (int h = 0; h < 4; ++h) one[h] = fmaxf(one[h], v.e[h]);
    }
    __device__ __forceinline__ float get(int h) const { return one[h]; }
};

// All moves of a row: one CTA per row, of NT threads, P pieces a thread in registers (P = 0: any length, the row is read
// twice, the second time from cache).  One pass takes the groups' maxima, one collects the moves at or above the bound
// and sums the exponentials of the others relative to it; one warp ranks the candidates.
template <typename T, int NT, int P>
__global__ void __launch_bounds__(NT) top_kernel(int n_moves, const T *__restrict__ logits, int64_t ld, int k, float inv_t,
                                                 float *__restrict__ values, int64_t *__restrict__ moves,
                                                 float *__restrict__ log_rest) {
    constexpr int kPer = Piece<T>::kPer, kChunk = P ? P : 4;             // pieces at hand at once
    __shared__ TopShared sh;
    const int64_t i = blockIdx.x;
    const T *row = logits + i * ld;
    const int lead = lead_of(row), lane = threadIdx.x & 31;
    Piece<T> mine[kChunk];
    auto load = [&](int at) {                    // the chunk whose first piece starts at `at`
#pragma unroll
        for (int p = 0; p < kChunk; ++p) mine[p] = load_piece(row, at + p * NT * kPer, n_moves, from_float<T>(-kInf));
    };
    const int first = (int)threadIdx.x * kPer - lead, step = kChunk * NT * kPer;
    FourMax<T> max4;
    for (int at = first; at < n_moves; at += step) {
        load(at);
#pragma unroll
        for (int p = 0; p < kChunk; ++p) max4.add(mine[p]);
        if (P) break;
    }
    float best[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) best[h] = max4.get(h);
    // up to four groups a thread, as many as give k of them a good bound
    const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    if (4 * k <= NT) {
        sh.group[threadIdx.x] = order_of(most);
    } else if (2 * k <= NT || kGroups == 2 * NT) {
        sh.group[threadIdx.x] = order_of(fmaxf(best[0], best[2]));
        sh.group[threadIdx.x + NT] = order_of(fmaxf(best[1], best[3]));
    } else {
#pragma unroll
        for (int h = 0; h < 4; ++h)
            if (h * NT < kGroups) sh.group[h * NT + threadIdx.x] = order_of(best[h]);
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        const unsigned t = 4 * k <= NT ? kth_of_groups<NT>(sh.group, k)
                           : 2 * k <= NT || kGroups == 2 * NT ? kth_of_groups<2 * NT>(sh.group, k) : kth_of_groups<kGroups>(sh.group, k);
        // at least the lowest finite value, so that -inf stays below it
        if (lane == 0) sh.bound = max(t, order_of(-FLT_MAX));
    }
    __syncthreads();
    const float bound = value_of(sh.bound), c = inv_t * kLog2e;
    const float bc = fmaxf(bound * c, -FLT_MAX);
    float below = 0.f;
    for (int at = first; at < n_moves; at += step) {
        if (!P) load(at);
        if (most >= bound) {                     // few threads; the moves are marked first, which keeps the code short
            constexpr int kPieces = 32 / kPer;   // of a word of marks
#pragma unroll
            for (int p0 = 0; p0 < kChunk; p0 += kPieces) {
                uint32_t marks = 0u;
#pragma unroll
                for (int u = 0; u < kPieces && p0 + u < kChunk; ++u)
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (to_float(mine[p0 + u < kChunk ? p0 + u : 0].e[e]) >= bound) marks |= 1u << (u * kPer + e);
                for (; marks; marks &= marks - 1) {
                    const int bit = __ffs((int)marks) - 1, m = at + (p0 + bit / kPer) * NT * kPer + bit % kPer;
                    const int place = atomicAdd(&sh.count, 1);
                    if (place < kCandidates) sh.cand[place] = key_of(order_of(to_float(row[m])), m);
                }
            }
        }
#pragma unroll
        for (int p = 0; p < kChunk; ++p)
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const float v = to_float(mine[p].e[e]), x = exp2_fast(fmaf(v, c, -bc));
                if (v < bound) below += x;
            }
        if (P) break;
    }
    below = warp_reduce(below, Sum());
    if (lane == 0) sh.scratch[threadIdx.x >> 5] = below;
    __syncthreads();
    const int found = sh.count;
    values += i * k;
    moves += i * k;
    if (found > kCandidates) {                   // many equal values at the bound
        __syncthreads();                         // all have read the count
        select_top<NT>(sh, n_moves, k, inv_t, [&](int e, unsigned &o, int &m) { o = order_of(to_float(row[e])); m = e; }, values, moves,
                   log_rest + i);
        return;
    }
    below = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) below += sh.scratch[w];
    // `step` threads, t of them this one, rank the candidates (how many are larger) and close the row
    auto close = [&](int t, int step, auto per, auto &&reduce) {
        constexpr int U = decltype(per)::value;  // candidates a thread ranks
        unsigned long long key[U];
        int rank[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            key[u] = u * step + t < found ? sh.cand[u * step + t] : 0ull;
            rank[u] = 0;
        }
#pragma unroll 4
        for (int d = 0; d < found; ++d) {
            const unsigned long long other = sh.cand[d];
#pragma unroll
            for (int u = 0; u < U; ++u) rank[u] += other > key[u];
        }
        float ref = -kInf;                       // the largest candidate that is not among the k
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * step + t >= found) break;
            const float v = value_of((unsigned)(key[u] >> 32));
            if (rank[u] < k) {
                values[rank[u]] = v;
                moves[rank[u]] = (int64_t) ~(unsigned)key[u];
            } else {
                ref = fmaxf(ref, v);
            }
        }
        for (int r = found + t; r < k; r += step) {
            values[r] = -kInf;
            moves[r] = -1;
        }
        float left = 0.f, out = -kInf;
        if (found > k) {                         // ref is at least the bound: the largest of all that are left
            ref = reduce(ref, -kInf, Max());
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u * step + t < found && rank[u] >= k) left += exp2_fast((value_of((unsigned)(key[u] >> 32)) - ref) * c);
            left = reduce(left, 0.f, Sum());
            out = ref * inv_t + logf(left + below * exp2_fast((bound - ref) * c));
        } else if (found == k && below > 1e-25f) {
            out = bound * inv_t + logf(below);
        } else if (found == k) {                 // all that is left lies far below the bound, or nothing is
            for (int e = t; e < n_moves; e += step) {
                const float v = to_float(row[e]);
                if (v < bound) ref = fmaxf(ref, v);
            }
            ref = reduce(ref, -kInf, Max());
            if (ref > -kInf)
                for (int e = t; e < n_moves; e += step) {
                    const float v = to_float(row[e]);
                    if (v < bound) left += exp2_fast((v - ref) * c);
                }
            left = reduce(left, 0.f, Sum());
            if (ref > -kInf) out = ref * inv_t + logf(left);
        }
        if (t == 0) log_rest[i] = ref == kInf ? kInf : out;           // -inf for fewer than k moves
    };
    auto in_block = [&](float x, float unit, auto &&f) { return block_reduce(x, sh.scratch, unit, f); };
    auto in_warp = [&](float x, float, auto &&f) { return warp_reduce(x, f); };
    if (found > kRanked) {
        if (found <= NT) close((int)threadIdx.x, NT, std::integral_constant<int, 1>{}, in_block);
        else if (found <= 2 * NT) close((int)threadIdx.x, NT, std::integral_constant<int, 2>{}, in_block);
        else close((int)threadIdx.x, NT, std::integral_constant<int, kCandidates / NT>{}, in_block);
    } else if (threadIdx.x < 32) {
        if (found <= 32) close(lane, 32, std::integral_constant<int, 1>{}, in_warp);
        else if (found <= 64) close(lane, 32, std::integral_constant<int, 2>{}, in_warp);
        else close(lane, 32, std::integral_constant<int, kRanked / 32>{}, in_warp);
    }
}

__device__ __forceinline__ float softplus(float d) { return fmaxf(d, 0.f) + log1pf(expf(-fabsf(d))); }
struct LossArgs {
    int64_t n_moves;
    int64_t ld;                                 // of the student's logits
    const float *t;                             // (rows, k) the teacher's logits
    const int64_t *named;                       // (rows, k) their moves
    const float *log_rest;                      // (rows) or NULL: the named moves alone
    int k;
    float temperature;
    const int64_t *list;                        // (rows, n_listed) the student's support, or NULL: all moves
    const uint8_t *valid;
    int n_listed;
    const float *weight;                        // (rows) or NULL
    float scale;                                // of the gradient beside the weight: 1 / rows for a mean
    const float *upstream;                      // NULL: 1.  The gradient that arrives, row i at upstream[i upstream_step]
    int64_t upstream_step;
    int skip_ones;                              // rows whose upstream gradient is 1 are left as they are
    float *loss;                                // (rows) weight * loss, or NULL
    int64_t ld_g;                               // of the gradient
};

template <typename T>
__global__ void __launch_bounds__(kThreads) loss_kernel(LossArgs a, const T *__restrict__ logits, T *__restrict__ grad) {
    extern __shared__ unsigned dynamic[];
    __shared__ float scratch[kWarps];
    __shared__ int named[kMaxTop];
    __shared__ float z[kMaxTop], s_at[kMaxTop];
    const int64_t i = blockIdx.x;
    const float up = a.upstream ? a.upstream[i * a.upstream_step] : 1.f;
    if (a.skip_ones && up == 1.f) return;
    const T *row = logits + i * a.ld;
    T *g = grad ? grad + i * a.ld_g : nullptr;
    const float inv_t = 1.f / a.temperature, weight = a.weight ? a.weight[i] : 1.f;
    const int n_words = (int)((a.n_moves + 31) / 32);
    unsigned *const bitmap = dynamic;           // the named moves
    unsigned *const support = dynamic + n_words;                           // the listed moves, their values after them
    int *const listed = reinterpret_cast<int *>(support + n_words);
    float *const listed_at = reinterpret_cast<float *>(listed + a.n_listed);

    const int n = a.list ? a.n_listed : (int)a.n_moves;
    if (a.list) read_list(a.list + i * a.n_listed, a.valid + i * a.n_listed, a.n_listed, a.n_moves, row, support, n_words, listed, listed_at);
    for (int w = threadIdx.x; w < n_words; w += kThreads) bitmap[w] = 0u;
    for (int c = threadIdx.x; c < a.k; c += kThreads) {
        const int64_t m = a.named[i * a.k + c];
        const float t = a.t[i * a.k + c];
        bool keep = m >= 0 && m < a.n_moves && t != -kInf;
        if (keep && a.list) keep = (support[m >> 5] >> (m & 31)) & 1u;
        named[c] = keep ? (int)m : -1;
        z[c] = t;
    }
    __syncthreads();
    // a move named twice counts at its first place
    bool twice[(kMaxTop + kThreads - 1) / kThreads];
#pragma unroll
    for (int u = 0; u < (kMaxTop + kThreads - 1) / kThreads; ++u) {
        const int c = u * kThreads + threadIdx.x;
        twice[u] = false;
        if (c < a.k && named[c] >= 0)
            for (int d = 0; d < c; ++d) twice[u] |= named[d] == named[c];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < (kMaxTop + kThreads - 1) / kThreads; ++u) {
        const int c = u * kThreads + threadIdx.x;
        if (c >= a.k) break;
        if (twice[u]) named[c] = -1;
        s_at[c] = named[c] >= 0 ? to_float(row[named[c]]) : -kInf;
        if (named[c] >= 0) atomicOr(&bitmap[named[c] >> 5], 1u << (named[c] & 31));
    }
    __syncthreads();

    // over the named moves: the teacher's and the student's log sums
    float mz = -kInf, ms = -kInf;
    int some = 0;
    for (int c = threadIdx.x; c < a.k; c += kThreads)
        if (named[c] >= 0) {
            some = 1;
            mz = fmaxf(mz, z[c]);
            ms = fmaxf(ms, s_at[c]);
        }
    some = __syncthreads_or(some);
    mz = block_reduce(mz, scratch, -kInf, Max());
    ms = block_reduce(ms, scratch, -kInf, Max());
    const float base_s = ms > -kInf ? ms : 0.f;
    float sz = 0.f, ss = 0.f;
    for (int c = threadIdx.x; c < a.k; c += kThreads)
        if (named[c] >= 0) {
            sz += expf((z[c] - mz) * inv_t);
            ss += expf((s_at[c] - base_s) * inv_t);
        }
    sz = block_reduce(sz, scratch, 0.f, Sum());
    ss = block_reduce(ss, scratch, 0.f, Sum());
    const float log_sz = logf(sz), log_ss = logf(ss);

    // over the other moves of the support
    auto other = [&](int e, float &s) {
        const int m = a.list ? listed[e] : e;
        if (m < 0) return false;
        s = a.list ? listed_at[e] : to_float(row[e]);
        return !((bitmap[m >> 5] >> (m & 31)) & 1u);
    };
    float m = -kInf;
    for (int e = threadIdx.x; e < n; e += kThreads) {
        float s;
        if (other(e, s)) m = fmaxf(m, s);
    }
    m = block_reduce(m, scratch, -kInf, Max());
    const float base = m > -kInf ? m : 0.f;
    float sum = 0.f;
    for (int e = threadIdx.x; e < n; e += kThreads) {
        float s;
        if (other(e, s)) sum += expf((s - base) * inv_t);
    }
    sum = block_reduce(sum, scratch, 0.f, Sum());
    // no move with any probability at all (a NaN is one, and a maximum passes it over)
    if (ss == 0.f && sum == 0.f) some = 0;

    // log odds and log shares of the named moves against the rest: the student's, and the teacher's where it has a rest.
    // The maxima are subtracted first: the size of the logits does not matter.
    const float log_sum = logf(sum);
    const float odds_q = sum == 0.f ? kInf : ss == 0.f ? -kInf : (base_s - base) * inv_t + (log_ss - log_sum);
    const float log_q_rest = -softplus(odds_q), log_q_named = -softplus(-odds_q);
    float odds_p = 0.f, p_rest = 0.f, log_p_named = 0.f;
    if (a.log_rest && a.log_rest[i] != -kInf) {
        odds_p = mz * inv_t - a.log_rest[i] + log_sz;
        p_rest = expf(-softplus(odds_p));
        log_p_named = -softplus(-odds_p);
    }
    auto log_p = [&](int c) { return (z[c] - mz) * inv_t - log_sz + log_p_named; };
    auto log_q = [&](int c) { return s_at[c] == -kInf ? -kInf : (s_at[c] - base_s) * inv_t - log_ss + log_q_named; };
    if (a.loss) {
        float part = 0.f;
        for (int c = threadIdx.x; c < a.k; c += kThreads)
            if (named[c] >= 0) {
                const float lp = log_p(c), p = expf(lp);
                if (!(p == 0.f)) part += p * (lp - log_q(c));
            }
        part = block_reduce(part, scratch, 0.f, Sum());
        if (threadIdx.x == 0) {
            if (!(p_rest == 0.f)) part += p_rest * (softplus(odds_q) - softplus(odds_p));
            a.loss[i] = some ? part * (a.temperature * a.temperature) * weight : 0.f;
        }
    }
    if (!g) return;
    const float f = some ? a.temperature * a.scale * weight * up : 0.f;
    // outside the named moves: the softmax over the rest, times what the student holds there beyond the teacher
    const float beyond = sum == 0.f ? 0.f : f * (expf(log_q_rest) - p_rest) / sum;
    if (a.list) {
        for (int64_t e = threadIdx.x; e < a.n_moves; e += kThreads) g[e] = from_float<T>(0.f);
        __syncthreads();
    }
    for (int e = threadIdx.x; e < n; e += kThreads) {
        float s;
        if (other(e, s)) g[a.list ? listed[e] : e] = from_float<T>(some ? beyond * expf((s - base) * inv_t) : 0.f);
    }
    for (int c = threadIdx.x; c < a.k; c += kThreads)
        if (named[c] >= 0) g[named[c]] = from_float<T>(some ? f * (expf(log_q(c)) - expf(log_p(c))) : 0.f);
}

// out = scale * sum of the losses, in one fixed order.
__global__ void __launch_bounds__(1024) sum_kernel(int64_t rows, const float *__restrict__ loss, double scale, float *__restrict__ out) {
    __shared__ double part[32];
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) x += (double)loss[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x < 32) {
        x = part[threadIdx.x];
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (threadIdx.x == 0) *out = (float)(x * scale);
    }
}

template <typename K>
void allow_shared(K kernel, size_t bytes) {
    if (bytes > 32 * 1024) AFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
}

void check_rows(int64_t rows, int64_t n_moves, int type, const void *logits, int64_t ld, int k, float temperature,
                const int64_t *list, const uint8_t *valid, int64_t n_listed) {
    AFB_CHECK(rows >= 0 && n_moves >= 0 && n_listed >= 0, "negative size");
    AFB_CHECK(rows < (1LL << 31), "size above 2^31");
    AFB_CHECK(n_moves <= kMaxMoves, "more than 1048576 moves");
    AFB_CHECK(known_type(type), "unknown element type");
    AFB_CHECK(k >= 1 && k <= kMaxTop, "k must be between 1 and 256");
    AFB_CHECK(temperature > 0.f && std::isfinite(temperature) && std::isfinite(1.f / temperature), "the temperature must be positive and finite");
    AFB_CHECK((list == nullptr) == (valid == nullptr), "a list of moves comes with its valid flags");
    AFB_CHECK(n_listed <= kMaxListed, "more than 4096 listed moves a position");
    AFB_CHECK(ld >= n_moves, "a leading dimension is below the row length");
    AFB_CHECK(rows == 0 || n_moves == 0 || logits, "NULL pointer");
    AFB_CHECK(reinterpret_cast<uintptr_t>(logits) % type_size(type) == 0, "the logits are not aligned to their elements");
}

}  // namespace
}  // namespace afb

using namespace afb;

extern "C" {

int afb_top_logits(int64_t rows, int64_t n_moves, int type, const void *logits, int64_t ld, int k, float temperature,
                   const int64_t *legal, const uint8_t *valid, int64_t n_listed, float *values, int64_t *moves, float *log_rest,
                   void *stream) {
    return guarded([&] {
        check_rows(rows, n_moves, type, logits, ld, k, temperature, legal, valid, n_listed);
        if (rows == 0) return;
        AFB_CHECK(values && moves && log_rest, "NULL pointer");
        const cudaStream_t s = as_stream(stream);
        const float inv_t = 1.f / temperature;
        with_type(type, [&](auto e) {
            using T = decltype(e);
            const T *x = static_cast<const T *>(logits);
            if (legal) {
                const size_t shared = (size_t)((n_moves + 31) / 32) * 4 + (size_t)n_listed * 8;
                allow_shared(top_listed_kernel<T>, shared);
                top_listed_kernel<T><<<(unsigned)rows, kThreads, shared, s>>>(n_moves, x, ld, k, inv_t, legal, valid, (int)n_listed,
                                                                              values, moves, log_rest);
                return;
            }
            // as few pieces a thread as hold a row wherever it starts; the fewer threads, the more rows at once
            auto go = [&](auto threads, auto p) {
                constexpr int NT = decltype(threads)::value;
                top_kernel<T, NT, decltype(p)::value><<<(unsigned)rows, NT, 0, s>>>((int)n_moves, x, ld, k, inv_t, values, moves, log_rest);
            };
            const int64_t pieces = (n_moves + 2 * Piece<T>::kPer - 2) / Piece<T>::kPer;
            using Few = std::integral_constant<int, 128>;
            using Many = std::integral_constant<int, 256>;
            if (pieces <= 128) go(Few{}, std::integral_constant<int, 1>{});
            else if (pieces <= 3 * 128) go(Few{}, std::integral_constant<int, 3>{});
            else if (pieces <= 5 * 128) go(Few{}, std::integral_constant<int, 5>{});
            else if (pieces <= 9 * 128) go(Few{}, std::integral_constant<int, 9>{});
            else go(Many{}, std::integral_constant<int, 0>{});
        });
        AFB_LAUNCHED();
    });
}

int afb_distill_loss(int64_t rows, int64_t n_moves, int type, const void *logits, int64_t ld, int k, const float *values,
                     const int64_t *moves, const float *log_rest, float temperature, const int64_t *legal, const uint8_t *valid,
                     int64_t n_listed, const float *weight, float scale, const float *upstream, int64_t upstream_step,
                     int skip_ones, float *row_loss, float *loss, void *grad, int64_t ld_grad, void *stream) {
    return guarded([&] {
        check_rows(rows, n_moves, type, logits, ld, k, temperature, legal, valid, n_listed);
        AFB_CHECK(upstream_step >= 0, "negative size");
        if (rows == 0) {
            if (loss) AFB_CUDA(cudaMemsetAsync(loss, 0, 4, as_stream(stream)));
            return;
        }
        AFB_CHECK(!loss || row_loss, "the loss needs row_loss");
        AFB_CHECK(values && moves, "NULL pointer");
        if (grad) {
            AFB_CHECK(ld_grad >= n_moves, "a leading dimension is below the row length");
            AFB_CHECK(reinterpret_cast<uintptr_t>(grad) % type_size(type) == 0, "the gradient is not aligned to its elements");
        }
        const LossArgs a{n_moves, ld, values, moves, log_rest, k, temperature, legal, valid, (int)n_listed, weight, scale, upstream,
                         upstream_step, skip_ones, row_loss, ld_grad};
        const size_t words = (size_t)((n_moves + 31) / 32) * 4;
        const size_t shared = legal ? 2 * words + (size_t)n_listed * 8 : words;
        with_type(type, [&](auto e) {
            using T = decltype(e);
            allow_shared(loss_kernel<T>, shared);
            loss_kernel<T><<<(unsigned)rows, kThreads, shared, as_stream(stream)>>>(a, static_cast<const T *>(logits), static_cast<T *>(grad));
        });
        AFB_LAUNCHED();
        if (loss) {
            sum_kernel<<<1, 1024, 0, as_stream(stream)>>>(rows, row_loss, (double)scale, loss);
            AFB_LAUNCHED();
        }
    });
}

}  // extern "C"
