// Distillation from a teacher's best moves: their selection, and the loss of a student against them with its
// gradient.
//
// Selection (top_kernel, top_listed_kernel): for each row of logits l over a support (all moves, or the row's listed
//   moves) the k largest, ties to the lowest move, and  log_rest = log sum exp(l / T)  over the support's moves that are
//   not among them.  NaN and -inf are outside the support.  A lower bound of the k-th largest comes from the largest
//   value of each of 128 to 512 groups of moves (k different moves are at least the k-th largest of those); the few moves
//   at or above the bound are collected and ranked by counting, the others' exponentials summed in the same pass.
// Loss (loss_kernel, loss_listed_kernel, loss_long_kernel): with p the teacher's distribution over its named moves C
//   (softmax of t / T; with `rest` one more outcome, any other move, at exp(log_rest)) and q = softmax(s / T) of the
//   student over its support,
//       loss = T^2 sum_c p_c (log p_c - log q_c)                          q_rest = the sum of q outside C
//       dloss / ds_j = T (q_j - p_j)  in C,   T q_j (1 - p_rest / q_rest)  outside C,  0 outside the support.
//   The sums over C and over the rest are taken apart (the rest is not a total less C), so neither the shares nor the
//   gradient take a difference of nearly equal sums.
// All sums and exponentials are float32; a gradient is rounded to the logits' type once, scaled.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "dtypes.cuh"

namespace afb {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kThreads = 128;                   // of a CTA, where nothing else is said
constexpr int kWarps = 16;                      // at most
constexpr int kListThreads = 64;                // of a CTA that takes the loss over a row's list (16,000 x 64: 71 us, 109 with 128)
constexpr int kLongThreads = 256;               // for rows that a CTA does not hold
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
template <int NT, typename T>
__device__ void read_list(const int64_t *list, const uint8_t *valid, int n_listed, int64_t n_moves, const T *row, unsigned *bitmap,
                          int n_words, int *moves, float *values) {
    for (int w = threadIdx.x; w < n_words; w += NT) bitmap[w] = 0u;
    __syncthreads();
    int again = 0;
    for (int l = threadIdx.x; l < n_listed; l += NT) {
        const int64_t m = list[l];
        const bool in = valid[l] && m >= 0 && m < n_moves;
        moves[l] = in ? (int)m : -1;
        if (!in) continue;
        const unsigned bit = 1u << (m & 31);
        again |= (atomicOr(&bitmap[m >> 5], bit) & bit) != 0u;
        values[l] = to_float(row[m]);
    }
    if (__syncthreads_or(again)) {               // rare: keep the first place of each move, whatever the order above
        for (int l0 = 0; l0 < n_listed; l0 += NT) {
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

// Entries that are ranked without a bound.  35,840 lists of 33, 48, 64, 72, 80, 96 and 128, k = 8: 77, 87, 92, 110, 125, 141
// and 186 us without, 105, 107, 108, 115, 122, 131 and 157 with it (k = 32 the same within 4%); fewer rows would gain up to
// 112 entries (1,120 lists of 96: 9.9 us without, 10.7 with).
constexpr int kFew = 72;

// Selects from `n` entries, get(e, order, move).  A row with too many entries at the bound (many equal values) finds
// the k-th key itself bit by bit.
template <int NT, typename Get>
__device__ void select_top(TopShared &sh, int n, int k, float inv_t, Get &&get, float *values, int64_t *moves, float *log_rest) {
    if (threadIdx.x == 0) sh.count = 0;
    unsigned bound = 1u;                         // 0: no move
    if (n > kFew) {
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
            if (threadIdx.x == 0) sh.bound = max(t, 1u);                  // fewer than k groups hold a move
        }
        __syncthreads();
        bound = sh.bound;
    } else {
        __syncthreads();
    }
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

// The rows' listed moves: all entries are at hand in shared memory.  Latency of the list, then of the gather (a 32-byte
// sector a move): 1,120 rows of 64, k = 8: 7.4 us; 35,840 of them 92 us; 35,840 of 218, k = 32: 205 us.
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
    read_list<kThreads>(list + i * n_listed, valid + i * n_listed, n_listed, n_moves, row, dynamic, n_words, listed, at);
    select_top<kThreads>(sh, n_listed, k, inv_t, [&](int e, unsigned &o, int &m) { m = listed[e]; o = m < 0 ? 0u : order_of(at[e]); },
               values + i * k, moves + i * k, log_rest + i);
}

// 2^x; below 2^-126 it is 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Candidates that one warp ranks by itself where many rows keep the SM busy (35,840 x 4168 float32, k = 128: 363 us, 406 with
// the whole CTA; a single row of k = 64: 6.7 us and 6.0).  Fewer in larger CTAs, of which an SM holds few.  With at most 64, 96
// and 160: 2,048 x 32000 bfloat16 62, 58 and 58 us at k = 64, 67, 67 and 71 at k = 100, 71, 71 and 77 at k = 130; float32 82, 77 and
// 78 at k = 64; 4,096 x 26000 float16 112, 102 and 102 at k = 64.  More rows would take more: 8,000 x 12000 float32 119, 107 and
// 99 at k = 64, 157, 157 and 153 at k = 130.
constexpr int kRanked = 160, kRankedLarge = 96, kManyRows = 256;

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
// and sums the exponentials of the others relative to it; one warp ranks the candidates.  35,840 x 4168 float32: 112 us
// for k = 1 (5.3 TB/s), 160 for 32, 361 for 128; 2,048 x 32000 bfloat16, k = 64: 58 us.  Bound by what a row costs beside
// its elements: the search for the bound and the ranking are one warp's, while the other CTAs of the SM load.
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
    // no piece is partly of the row: shorter code for float32 (168 us against 158 at 35,840 x 4168), none for 16-bit types
    const bool whole = sizeof(T) == 4 && lead == 0 && n_moves % kPer == 0;
    Piece<T> nothing;
#pragma unroll
    for (int e = 0; e < kPer; ++e) nothing.e[e] = from_float<T>(-kInf);
    auto load = [&](int at) {                    // the chunk whose first piece starts at `at`
        if (whole) {
#pragma unroll
            for (int p = 0; p < kChunk; ++p)
                mine[p].raw = at + p * NT * kPer < n_moves ? __ldg(reinterpret_cast<const uint4 *>(row + at + p * NT * kPer)) : nothing.raw;
        } else {
#pragma unroll
            for (int p = 0; p < kChunk; ++p) mine[p] = load_piece(row, at + p * NT * kPer, n_moves, from_float<T>(-kInf));
        }
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
    // one to four groups a thread, as many as give k of them a good bound
    const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    const bool one = 4 * k <= NT || NT == kGroups;
    if (one) {
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
        const unsigned t = one ? kth_of_groups<NT>(sh.group, k)
                           : 2 * k <= NT || kGroups == 2 * NT
                               ? kth_of_groups<(2 * NT < kGroups ? 2 * NT : kGroups)>(sh.group, k)
                               : kth_of_groups<kGroups>(sh.group, k);
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
    // `step` threads, t of them this one, rank the candidates (how many are larger) and close the row.  Candidates lie in the
    // order in which they were found, which differs from run to run: what is summed is put in the order of the ranks first
    // (1% of 35,840 x 4168, k = 32: 159 -> 161 us)
    auto close = [&](int t, int step, auto per, auto &&reduce, auto &&sync) {
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
        if (found > k) sync();                   // all candidates are ranked
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * step + t >= found) break;
            if (rank[u] < k) {
                values[rank[u]] = value_of((unsigned)(key[u] >> 32));
                moves[rank[u]] = (int64_t) ~(unsigned)key[u];
            } else {
                sh.cand[rank[u]] = key[u];
            }
        }
        for (int r = found + t; r < k; r += step) {
            values[r] = -kInf;
            moves[r] = -1;
        }
        float ref = -kInf, left = 0.f, out = -kInf;
        if (found > k) {                         // the largest of them is at least the bound: the largest of all that are left
            sync();
            ref = value_of((unsigned)(sh.cand[k] >> 32));
            for (int r = k + t; r < found; r += step) left += exp2_fast((value_of((unsigned)(sh.cand[r] >> 32)) - ref) * c);
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
    auto block_sync = [] { __syncthreads(); };
    auto warp_sync = [] { __syncwarp(); };
    using std::integral_constant;
    constexpr int kAlone = NT == kThreads ? kRanked : kRankedLarge;
    if (found > (gridDim.x >= kManyRows ? kAlone : 32)) {
        if (found <= NT) close((int)threadIdx.x, NT, integral_constant<int, 1>{}, in_block, block_sync);
        else if (found <= 2 * NT) close((int)threadIdx.x, NT, integral_constant<int, 2>{}, in_block, block_sync);
        else if (4 * NT < kCandidates && found <= 3 * NT) close((int)threadIdx.x, NT, integral_constant<int, 3>{}, in_block, block_sync);
        else if (4 * NT < kCandidates && found <= 4 * NT) close((int)threadIdx.x, NT, integral_constant<int, 4>{}, in_block, block_sync);
        else close((int)threadIdx.x, NT, integral_constant<int, kCandidates / NT>{}, in_block, block_sync);
    } else if (threadIdx.x < 32) {
        if (found <= 32) close(lane, 32, integral_constant<int, 1>{}, in_warp, warp_sync);
        else if (found <= 64) close(lane, 32, integral_constant<int, 2>{}, in_warp, warp_sync);
        else if (found <= 96) close(lane, 32, integral_constant<int, 3>{}, in_warp, warp_sync);
        else close(lane, 32, integral_constant<int, kAlone / 32>{}, in_warp, warp_sync);
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

// The moves that a teacher names in one row, and what is known of them before the row's other moves are summed, all in
// shared memory.
struct NamedSums {
    float p_rest, log_p_rest;                   // of any other move (0 and -inf without a rest)
    float ms, ss, log_ss;                       // largest s (0 for -inf), sum exp((s - ms) / T) and its log
    int some;                                   // a move is named
};
struct Named {
    int *move;                                  // -1: left out
    float *z, *s, *p;                           // the teacher's logit, then log p; the student's logit; p
    NamedSums *sums;
    __host__ __device__ static constexpr size_t bytes(int k) { return (size_t)k * 16; }
    __device__ __forceinline__ Named(unsigned char *at, int k, NamedSums *sums) : move(reinterpret_cast<int *>(at)), sums(sums) {
        z = reinterpret_cast<float *>(at) + k;
        s = z + k;
        p = s + k;
    }
};

// A thread's first named move, asked for before anything else of the row.
struct FirstNamed {
    int64_t move = -1;
    float t = 0.f;
    __device__ __forceinline__ FirstNamed(const LossArgs &a, int64_t i) {
        if ((int)threadIdx.x < a.k) move = a.named[i * a.k + threadIdx.x], t = a.t[i * a.k + threadIdx.x];
    }
};

// Reads row i's named moves and marks them (all threads; the marks are complete after the return).  keeps(move): whether
// the student's support has it; value(move): the student's logit; mark(move): sets its mark, whether it was set already.
// kOneMap: marks change what keeps() reads, so every move is asked for first.
template <bool kOneMap, typename T, typename Keeps, typename Value, typename Mark>
__device__ __forceinline__ void read_named(const Named &nm, const LossArgs &a, int64_t i, const T *row, const FirstNamed &first,
                                           Keeps &&keeps, Value &&value, Mark &&mark) {
    int again = 0;
    for (int c = threadIdx.x; c < a.k; c += blockDim.x) {
        const bool fetched = c == (int)threadIdx.x;
        const int64_t m = fetched ? first.move : a.named[i * a.k + c];
        const float t = fetched ? first.t : a.t[i * a.k + c];
        const bool keep = m >= 0 && m < a.n_moves && t != -kInf && keeps((int)m);
        nm.move[c] = keep ? (int)m : -1;
        nm.z[c] = t;
        nm.s[c] = keep ? value((int)m) : -kInf;
        if (!kOneMap && keep) again |= mark((int)m);
    }
    if (kOneMap) {
        __syncthreads();
        for (int c = threadIdx.x; c < a.k; c += blockDim.x)
            if (nm.move[c] >= 0) again |= mark(nm.move[c]);
    }
    if (__syncthreads_or(again)) {              // rare: a move named twice counts at its first place
        for (int c0 = 0; c0 < a.k; c0 += blockDim.x) {
            const int c = a.k - 1 - c0 - (int)threadIdx.x;                  // later places first
            bool drop = false;
            if (c >= 0 && nm.move[c] >= 0)
                for (int d = 0; d < c; ++d) drop |= nm.move[d] == nm.move[c];
            __syncthreads();
            if (drop) nm.move[c] = -1;
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.k; c += blockDim.x)
            if (nm.move[c] >= 0) nm.s[c] = to_float(row[nm.move[c]]);       // whichever of them had read it
        __syncthreads();
    }
}

// One warp: the teacher's distribution.  The shares of the named moves and of the rest follow from their log odds.
__device__ __forceinline__ void teach(const Named &nm, const LossArgs &a, int64_t i, float c, float inv_t) {
    const int lane = threadIdx.x & 31;
    float mz = -kInf, sz = 0.f;
    int some = 0;
    for (int e = lane; e < a.k; e += 32)
        if (nm.move[e] >= 0) mz = fmaxf(mz, nm.z[e]), some = 1;
    mz = warp_reduce(mz, Max());
    for (int e = lane; e < a.k; e += 32)
        if (nm.move[e] >= 0) sz += exp2_fast((nm.z[e] - mz) * c);
    sz = warp_reduce(sz, Sum());
    const float log_sz = logf(sz), log_rest = a.log_rest ? a.log_rest[i] : -kInf;
    // inf without a rest, also where mz / T leaves the range (a mask of the type's lowest value, T < 1)
    const float odds = log_rest == -kInf ? kInf : mz * inv_t - log_rest + log_sz;
    const float log_p_rest = -softplus(odds), log_p_named = -softplus(-odds);
    for (int e = lane; e < a.k; e += 32)
        if (nm.move[e] >= 0) {
            nm.z[e] = (nm.z[e] - mz) * inv_t - log_sz + log_p_named;
            nm.p[e] = expf(nm.z[e]);
        }
    some = __any_sync(0xffffffffu, some);
    if (lane == 0) nm.sums->p_rest = expf(log_p_rest), nm.sums->log_p_rest = log_p_rest, nm.sums->some = some;
}

// One warp: the student's log sum over the named moves.
__device__ __forceinline__ void sum_named(const Named &nm, int k, float c) {
    const int lane = threadIdx.x & 31;
    float ms = -kInf, ss = 0.f;
    for (int e = lane; e < k; e += 32)
        if (nm.move[e] >= 0) ms = fmaxf(ms, nm.s[e]);
    ms = warp_reduce(ms, Max());
    ms = ms > -kInf ? ms : 0.f;
    for (int e = lane; e < k; e += 32)
        if (nm.move[e] >= 0) ss += exp2_fast((nm.s[e] - ms) * c);
    ss = warp_reduce(ss, Sum());
    if (lane == 0) nm.sums->ms = ms, nm.sums->ss = ss, nm.sums->log_ss = logf(ss);
}

// The student's log odds of the named moves against the others, whose terms sum to `sum` relative to exp(reference); gap:
// by how much ms / T exceeds the reference.  The maxima are subtracted first: the size of the logits does not matter.
__device__ __forceinline__ float odds_of(const Named &nm, float gap, float sum) {
    return sum == 0.f ? (nm.sums->log_ss == -kInf ? 0.f : kInf) : gap + (nm.sums->log_ss - logf(sum));
}
// Whether a row has something to learn: a named move, and a move with any probability (a NaN is one).
__device__ __forceinline__ bool alive(const Named &nm, float sum) { return nm.sums->some && !(nm.sums->log_ss == -kInf && sum == 0.f); }

// The gradient at a move that is not named over its term of `sum`: the softmax over those moves, times what the student
// holds there beyond the teacher (1 / (1 + exp(odds)) - p_rest).
__device__ __forceinline__ float beyond_of(const Named &nm, float odds, float sum, float f) {
    return sum == 0.f || !alive(nm, sum) ? 0.f : f * (1.f / (1.f + expf(odds)) - nm.sums->p_rest) / sum;
}
// The gradient at a move from its term: 0 where nothing is to be learnt, whatever the term.
__device__ __forceinline__ float times(float beyond, float term) { return beyond == 0.f ? 0.f : beyond * term; }

// log q of the e-th named move.
__device__ __forceinline__ float log_q_of(const Named &nm, int e, float log_q_named, float inv_t) {
    const float s = nm.s[e];
    return s == -kInf ? -kInf : (s - nm.sums->ms) * inv_t + log_q_named;
}
__device__ __forceinline__ float log_q_named_of(const Named &nm, float odds) { return -softplus(-odds) - nm.sums->log_ss; }

// One warp: a row's loss.
__device__ __forceinline__ void write_loss(const Named &nm, const LossArgs &a, int64_t i, float odds, float sum, float inv_t, float weight) {
    const float log_q_named = log_q_named_of(nm, odds);
    float part = 0.f;
    for (int e = threadIdx.x & 31; e < a.k; e += 32)
        if (nm.move[e] >= 0) {
            const float p = nm.p[e];
            if (!(p == 0.f)) part += p * (nm.z[e] - log_q_of(nm, e, log_q_named, inv_t));
        }
    part = warp_reduce(part, Sum());
    if (!(nm.sums->p_rest == 0.f)) part += nm.sums->p_rest * (nm.sums->log_p_rest + softplus(odds));
    if ((threadIdx.x & 31) == 0) a.loss[i] = alive(nm, sum) ? part * (a.temperature * a.temperature) * weight : 0.f;
}

// The gradient at the named moves (all threads, over what stands there).
template <typename T>
__device__ __forceinline__ void write_named(const Named &nm, int k, float odds, float sum, float inv_t, float f, T *g) {
    const bool some = alive(nm, sum);
    for (int e = threadIdx.x; e < k; e += blockDim.x)
        if (nm.move[e] >= 0)
            g[nm.move[e]] = from_float<T>(some ? f * (expf(log_q_of(nm, e, log_q_named_of(nm, odds), inv_t)) - nm.p[e]) : 0.f);
}

// Over a row's listed moves: one CTA per row, the lists and their logits in shared memory.  The gradient's zeros are most of
// the traffic (16,000 x 4168 float32 with 64 listed: 75 us, 3.5 TB/s of zeros); the rest is the latency of list, gather and sums.
template <typename T>
__global__ void __launch_bounds__(kListThreads, 20) loss_listed_kernel(LossArgs a, int64_t rows, const T *__restrict__ logits, T *__restrict__ grad) {
    extern __shared__ unsigned dynamic[];
    __shared__ float scratch[kWarps];
    __shared__ NamedSums named_sums;
    const int n_words = (int)((a.n_moves + 31) / 32), n = a.n_listed;
    unsigned *const support = dynamic;          // a bit for each listed move, the named ones taken out again; then the list, its
    int *const listed = reinterpret_cast<int *>(support + n_words);      // logits, the named moves
    float *const at = reinterpret_cast<float *>(listed + n);
    const Named nm(reinterpret_cast<unsigned char *>(at + n), a.k, &named_sums);
    const float inv_t = 1.f / a.temperature, c = kLog2e * inv_t;
    for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const float up = a.upstream ? a.upstream[i * a.upstream_step] : 1.f;
        if (a.skip_ones && up == 1.f) {
            if (a.upstream_step == 0) return;
            continue;
        }
        const T *row = logits + i * a.ld;
        const FirstNamed first_named(a, i);
        const float weight = a.weight ? a.weight[i] : 1.f;
        T *g = grad ? grad + i * a.ld_g : nullptr;
        __syncthreads();                        // the row before is done with the shared memory
        read_list<kListThreads>(a.list + i * n, a.valid + i * n, n, a.n_moves, row, support, n_words, listed, at);
        if (g) {                                // zeros everywhere, the listed moves over them after a barrier
            constexpr int kPer = Piece<T>::kPer;
            const int moves = (int)a.n_moves, head = min((kPer - lead_of(g)) % kPer, moves), tail = head + (moves - head) / kPer * kPer;
#pragma unroll 4
            for (int e = head + (int)threadIdx.x * kPer; e < tail; e += kListThreads * kPer)
                *reinterpret_cast<uint4 *>(g + e) = make_uint4(0u, 0u, 0u, 0u);
            if ((int)threadIdx.x < head) g[threadIdx.x] = from_float<T>(0.f);
            if (tail + (int)threadIdx.x < moves) g[tail + threadIdx.x] = from_float<T>(0.f);
        }
        auto in_support = [&](int m) { return ((support[m >> 5] >> (m & 31)) & 1u) != 0u; };
        read_named<true>(nm, a, i, row, first_named, in_support, [&](int m) { return to_float(row[m]); },
                         [&](int m) { return (int)((~atomicAnd(&support[m >> 5], ~(1u << (m & 31))) >> (m & 31)) & 1u); });
        const int role = (int)(threadIdx.x >> 5);
        if (role == 0) sum_named(nm, a.k, c);
        else if (role == 1) teach(nm, a, i, c, inv_t);
        auto other = [&](int e) { return listed[e] >= 0 && in_support(listed[e]); };     // takes part and is not named
        float m = -kInf, sum = 0.f;
        for (int e = threadIdx.x; e < n; e += kListThreads)
            if (other(e)) m = fmaxf(m, at[e]);
        m = block_reduce(m, scratch, -kInf, Max());
        const float base = m > -kInf ? m : 0.f;
        for (int e = threadIdx.x; e < n; e += kListThreads)
            if (other(e)) sum += exp2_fast((at[e] - base) * c);
        sum = block_reduce(sum, scratch, 0.f, Sum());
        const float f = a.temperature * a.scale * weight * up, odds = odds_of(nm, (nm.sums->ms - base) * inv_t, sum);
        if (a.loss && role == 0) write_loss(nm, a, i, odds, sum, inv_t, weight);
        if (!g) continue;
        write_named(nm, a.k, odds, sum, inv_t, f, g);
        const float beyond = beyond_of(nm, odds, sum, f);
        for (int e = threadIdx.x; e < n; e += kListThreads)
            if (other(e)) g[listed[e]] = from_float<T>(times(beyond, exp2_fast((at[e] - base) * c)));
    }
}

// Where a row's elements lie in shared memory: float32 from the start, so that the order of the sums does not depend on
// where the row starts in memory; 16-bit types as far from 16 bytes as there, so that they move in 16-byte pieces.
template <typename T>
__device__ __forceinline__ int shift_of(const T *row) { return sizeof(T) == 4 ? 0 : lead_of(row); }

template <int kBytes>
__device__ __forceinline__ void copy_async(void *shared, const void *global) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(shared);
    if (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(global) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(global) : "memory");
}
template <int kPending>
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;\n" ::"n"(kPending) : "memory"); }

// Starts the copy of a row of n elements to held[shift_of(row)] on; what is not of the row in its 16-byte pieces is -inf.
template <int NT, typename T>
__device__ __forceinline__ void fetch_row(T *held, const T *row, int n) {
    constexpr int kPer = Piece<T>::kPer;
    const int shift = shift_of(row), whole = (shift + n) / kPer;         // pieces that end within the row
    if (lead_of(row) == shift) {                 // pieces start on 16 bytes: the first is whole without a shift
        const T *const from = row - shift;
        for (int p = (shift ? 1 : 0) + (int)threadIdx.x; p < whole; p += NT) copy_async<16>(held + p * kPer, from + p * kPer);
        if (shift && threadIdx.x < kPer)
            held[threadIdx.x] = (int)threadIdx.x >= shift && (int)threadIdx.x < shift + n ? from[threadIdx.x] : from_float<T>(-kInf);
    } else {
        for (int m = threadIdx.x; m < whole * kPer; m += NT) copy_async<4>(held + m, row + m);
    }
    const int m = max(whole, shift ? 1 : 0) * kPer + (int)threadIdx.x;   // the last piece, where it is not whole
    if (threadIdx.x < kPer) held[m] = m < shift + n ? row[m - shift] : from_float<T>(-kInf);
    asm volatile("cp.async.commit_group;\n" ::: "memory");
}

// Over all moves, rows held in shared memory, NT threads a row.  The CTAs stay: with kAhead a CTA's next row is on its way
// (into a second buffer) while it works on one, so that only shared memory is waited for.  The named moves are taken out
// of the row (-inf), so that its sum is the rest's.  The terms are relative to the teacher's best move: no maximum is
// taken, one barrier joins the sums.  Sums outside kSmall .. kLarge (logits 69 T from that move's, no such move, NaN,
// values whose product with 1 / T overflows) are taken again, after subtracting the largest.  35,840 x 4168 float32: 205
// us with the gradient (5.8 TB/s of reads and writes), 145 without; 4,096 x 32000 bfloat16 with it 113 us (4.6 TB/s), where
// the exponentials, each taken twice, fill half of their pipe's time.
constexpr float kSmall = 1e-30f, kLarge = 1e30f;

template <typename T, int NT, bool kAhead>
__global__ void __launch_bounds__(NT, 768 / NT) loss_kernel(LossArgs a, int64_t rows, int held_bytes, const T *__restrict__ logits,
                                                  T *__restrict__ grad) {
    constexpr int kPer = Piece<T>::kPer;
    constexpr bool kKeep = sizeof(T) == 4;      // the terms replace the logits in shared memory
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ float scratch[kWarps];
    __shared__ NamedSums named_sums;
    // the rows' buffers, the named moves, their marks
    const Named nm(raw + (kAhead ? 2 : 1) * held_bytes, a.k, &named_sums);
    unsigned *const marks = reinterpret_cast<unsigned *>(nm.p + a.k);
    const int n = (int)a.n_moves, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv_t = 1.f / a.temperature, c = kLog2e * inv_t;
    auto held_of = [&](int turn) { return reinterpret_cast<T *>(raw + (kAhead ? turn * held_bytes : 0)); };
    // the first row of this CTA from i on that is not left as it is
    auto next = [&](int64_t i) {
        if (a.skip_ones)
            while (i < rows && a.upstream[i * a.upstream_step] == 1.f) i = a.upstream_step ? i + gridDim.x : rows;
        return i;
    };
    int64_t i = next(blockIdx.x);
    if (i >= rows) return;
    for (int w = threadIdx.x; w < (n + 31) / 32; w += NT) marks[w] = 0u;
    FirstNamed first_named(a, i);
    fetch_row<NT>(held_of(0), logits + i * a.ld, n);
    for (int turn = 0; i < rows; turn ^= 1) {
        const T *row = logits + i * a.ld;
        T *g = grad ? grad + i * a.ld_g : nullptr;
        T *const held = held_of(turn);
        const int shift = shift_of(row), pieces = (shift + n + kPer - 1) / kPer;
        const int64_t after = next(i + gridDim.x);
        if (kAhead && after < rows) {
            fetch_row<NT>(held_of(turn ^ 1), logits + after * a.ld, n);
            copies_done<1>();
        } else {
            copies_done<0>();
        }
        __syncthreads();
        read_named<false>(nm, a, i, row, first_named, [](int) { return true; }, [&](int m) { return to_float(held[shift + m]); },
                   [&](int m) {
                       held[shift + m] = from_float<T>(-kInf);
                       return (int)((atomicOr(&marks[m >> 5], 1u << (m & 31)) >> (m & 31)) & 1u);
                   });
        if (after < rows) first_named = FirstNamed(a, after);
        const float ref = nm.s[0] * c;          // a term is 2^(s c - ref): one rounding of the exponent
        float sum = 0.f;
#pragma unroll 4
        for (int p = threadIdx.x; p < pieces; p += NT) {
            Piece<T> v;
            v.raw = *reinterpret_cast<const uint4 *>(held + p * kPer);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const float x = exp2_fast(fmaf(to_float(v.e[e]), c, -ref));
                if constexpr (kKeep) v.e[e] = x;
                sum += x;
            }
            if constexpr (kKeep) *reinterpret_cast<uint4 *>(held + p * kPer) = v.raw;
        }
        if (warp == 0) sum_named(nm, a.k, c);
        else if (warp == 1) teach(nm, a, i, c, inv_t);
        sum = warp_reduce(sum, Sum());
        if (lane == 0) scratch[warp] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) sum += scratch[w];
        const float weight = a.weight ? a.weight[i] : 1.f;
        const float f = a.temperature * a.scale * weight * (a.upstream ? a.upstream[i * a.upstream_step] : 1.f);
        // the named moves' terms, and all
        const float to_ref = exp2_fast(fmaf(nm.sums->ms, c, -ref)), named = nm.sums->ss * to_ref, total = sum + named;
        if (sum > kSmall && named > kSmall && total < kLarge) {
            if (a.loss && warp == 0) {
                const float log_total = logf(total);
                float part = 0.f;
                for (int e = lane; e < a.k; e += 32)
                    if (nm.move[e] >= 0 && !(nm.p[e] == 0.f)) part += nm.p[e] * (nm.z[e] - (fmaf(nm.s[e], c, -ref) * kLn2 - log_total));
                part = warp_reduce(part, Sum());
                if (!(nm.sums->p_rest == 0.f)) part += nm.sums->p_rest * (nm.sums->log_p_rest + log1pf(named / sum));
                if (lane == 0) a.loss[i] = part * (a.temperature * a.temperature) * weight;
            }
            if (g) {
                // outside the named moves: the softmax, less the teacher's rest spread like the student's
                const float per_term = f * (__fdividef(1.f, total) - __fdividef(nm.sums->p_rest, sum));
                auto gradient = [&](T v) { return from_float<T>(per_term * (kKeep ? to_float(v) : exp2_fast(fmaf(to_float(v), c, -ref)))); };
                if (lead_of(g) == shift) {
#pragma unroll 4
                    for (int p = threadIdx.x; p < pieces; p += NT) {
                        Piece<T> v;
                        v.raw = *reinterpret_cast<const uint4 *>(held + p * kPer);
#pragma unroll
                        for (int e = 0; e < kPer; ++e) v.e[e] = gradient(v.e[e]);
                        store_piece(g, p * kPer - shift, n, v);
                    }
                } else {
                    for (int m = threadIdx.x; m < n; m += NT) g[m] = gradient(held[shift + m]);
                }
                __syncthreads();
                for (int e = threadIdx.x; e < a.k; e += NT)
                    if (nm.move[e] >= 0)
                        g[nm.move[e]] = from_float<T>(f * (__fdividef(exp2_fast(fmaf(nm.s[e], c, -ref)), total) - nm.p[e]));
            }
        } else {
            // rare: the row again, its largest values subtracted, the shares by their log odds
            __syncthreads();
            float base = -kInf;
            for (int m = threadIdx.x; m < n; m += NT) {
                held[shift + m] = (marks[m >> 5] >> (m & 31)) & 1u ? from_float<T>(-kInf) : row[m];
                base = fmaxf(base, to_float(held[shift + m]));
            }
            base = block_reduce(base, scratch, -kInf, Max());
            base = base > -kInf ? base : 0.f;
            sum = 0.f;
            for (int m = threadIdx.x; m < n; m += NT) sum += exp2_fast((to_float(held[shift + m]) - base) * c);
            sum = block_reduce(sum, scratch, 0.f, Sum());
            const float odds = odds_of(nm, (nm.sums->ms - base) * inv_t, sum);
            if (a.loss && warp == 0) write_loss(nm, a, i, odds, sum, inv_t, weight);
            if (g) {
                const float beyond = beyond_of(nm, odds, sum, f);
                for (int m = threadIdx.x; m < n; m += NT)
                    g[m] = from_float<T>(times(beyond, exp2_fast((to_float(held[shift + m]) - base) * c)));
                __syncthreads();
                write_named(nm, a.k, odds, sum, inv_t, f, g);
            }
        }
        for (int e = threadIdx.x; e < a.k; e += NT)
            if (nm.move[e] >= 0) marks[nm.move[e] >> 5] = 0u;
        if (!kAhead && after < rows) fetch_row<NT>(held_of(0), logits + after * a.ld, n);
        i = after;
    }
}

// Rows too long for shared memory: read twice, the second time from cache (2,048 x 32000 float32 with the gradient: 132 us).
template <typename T>
__global__ void __launch_bounds__(kLongThreads) loss_long_kernel(LossArgs a, int64_t rows, const T *__restrict__ logits, T *__restrict__ grad) {
    constexpr int kPer = Piece<T>::kPer, kChunk = 4;
    extern __shared__ unsigned marks[];
    __shared__ float scratch[kWarps];
    __shared__ NamedSums named_sums;
    const int n = (int)a.n_moves, words = (n + 31) / 32, warp = threadIdx.x >> 5;
    const Named nm(reinterpret_cast<unsigned char *>(marks + words), a.k, &named_sums);
    const float inv_t = 1.f / a.temperature, c = kLog2e * inv_t;
    for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const float up = a.upstream ? a.upstream[i * a.upstream_step] : 1.f;
        if (a.skip_ones && up == 1.f) {
            if (a.upstream_step == 0) return;
            continue;
        }
        const T *row = logits + i * a.ld;
        T *g = grad ? grad + i * a.ld_g : nullptr;
        const int shift = shift_of(row), first = (int)threadIdx.x * kPer - shift, step = kLongThreads * kPer;
        const bool whole = lead_of(row) == shift;
        const FirstNamed first_named(a, i);
        __syncthreads();                        // the row before is done with the shared memory
        for (int w = threadIdx.x; w < words; w += kLongThreads) marks[w] = 0u;
        __syncthreads();
        read_named<false>(nm, a, i, row, first_named, [](int) { return true; }, [&](int m) { return to_float(row[m]); },
                   [&](int m) { return (int)((atomicOr(&marks[m >> 5], 1u << (m & 31)) >> (m & 31)) & 1u); });
        if (warp == 0) sum_named(nm, a.k, c);
        else if (warp == 1) teach(nm, a, i, c, inv_t);
        // f(piece, its first element) of this thread's pieces, the named moves -inf
        auto each = [&](auto &&f) {
            for (int at0 = first; at0 < n; at0 += kChunk * step) {
                Piece<T> v[kChunk];
#pragma unroll
                for (int p = 0; p < kChunk; ++p) {
                    const int at = at0 + p * step;
                    if (whole) {
                        v[p] = load_piece(row, at, n, from_float<T>(-kInf));
                    } else {
#pragma unroll
                        for (int e = 0; e < kPer; ++e) v[p].e[e] = at + e < n ? row[at + e] : from_float<T>(-kInf);
                    }
                }
#pragma unroll
                for (int p = 0; p < kChunk; ++p) {
                    const int at = at0 + p * step;
                    if (at >= n) break;
                    // the marks of elements at .. at + kPer - 1, which may lie in two words
                    const int from = max(at, 0);
                    const unsigned low = marks[from >> 5], high = marks[min((from >> 5) + 1, words - 1)];
                    unsigned bits = __funnelshift_r(low, high, from & 31) << (from - at);
                    if (bits & ((1u << kPer) - 1u))
#pragma unroll
                        for (int e = 0; e < kPer; ++e)
                            if ((bits >> e) & 1u) v[p].e[e] = from_float<T>(-kInf);
                    f(v[p], at);
                }
            }
        };
        // as above: relative to the teacher's best move, or, where that does not do, to the largest
        float base = nm.s[0] > -kInf ? nm.s[0] : 0.f, sum = 0.f;
        auto add = [&](const Piece<T> &v, int) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) sum += exp2_fast((to_float(v.e[e]) - base) * c);
        };
        each(add);
        sum = block_reduce(sum, scratch, 0.f, Sum());
        if (!(sum > kSmall && sum < kLarge)) {
            base = -kInf;
            each([&](const Piece<T> &v, int) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) base = fmaxf(base, to_float(v.e[e]));
            });
            base = block_reduce(base, scratch, -kInf, Max());
            base = base > -kInf ? base : 0.f;
            sum = 0.f;
            each(add);
            sum = block_reduce(sum, scratch, 0.f, Sum());
        }
        const float weight = a.weight ? a.weight[i] : 1.f, f = a.temperature * a.scale * weight * up;
        const float odds = odds_of(nm, (nm.sums->ms - base) * inv_t, sum);
        if (a.loss && warp == 0) write_loss(nm, a, i, odds, sum, inv_t, weight);
        if (!g) continue;
        const float beyond = beyond_of(nm, odds, sum, f);
        const bool aligned = lead_of(g) == shift;
        each([&](const Piece<T> &v, int at) {
            Piece<T> out;
#pragma unroll
            for (int e = 0; e < kPer; ++e) out.e[e] = from_float<T>(times(beyond, exp2_fast((to_float(v.e[e]) - base) * c)));
            if (aligned) {
                store_piece(g, at, n, out);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (at + e >= 0 && at + e < n) g[at + e] = out.e[e];
            }
        });
        __syncthreads();
        write_named(nm, a.k, odds, sum, inv_t, f, g);
    }
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

// Threads of a CTA and 16-byte pieces a thread for rows of n elements: as few as hold a row wherever it starts (few
// threads: many rows at once); 0, no row in registers, beyond 4,605 float32 or 9,209 16-bit elements.  There the threads
// grow with the row: 8,192 x 5000 float32 53 us with 128 threads, 62 with 256; 2,048 x 32000 bfloat16 64, 57 and 62 with
// 128, 256 and 512; 2,048 x 32000 float32 104, 96 and 78.
template <typename T, typename F>
void by_row_length(int64_t n, F &&f) {
    const int64_t pieces = (n + 2 * Piece<T>::kPer - 2) / Piece<T>::kPer;
    using Few = std::integral_constant<int, kThreads>;
    if (pieces <= kThreads) f(Few{}, std::integral_constant<int, 1>{});
    else if (pieces <= 3 * kThreads) f(Few{}, std::integral_constant<int, 3>{});
    else if (pieces <= 5 * kThreads) f(Few{}, std::integral_constant<int, 5>{});
    else if (pieces <= 9 * kThreads) f(Few{}, std::integral_constant<int, 9>{});
    else if (pieces <= 20 * kThreads) f(Few{}, std::integral_constant<int, 0>{});
    else if (pieces <= 24 * 256) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 0>{});
    else f(std::integral_constant<int, 512>{}, std::integral_constant<int, 0>{});
}

void check_rows(int64_t rows, int64_t n_moves, int type, const void *logits, int64_t ld, int k, float temperature,
                const int64_t *list, const uint8_t *valid, int64_t n_listed) {
    AFB_CHECK(rows >= 0 && n_moves >= 0 && n_listed >= 0, "negative size");
    AFB_CHECK(rows < (1LL << 31), "size above 2^31");
    AFB_CHECK(n_moves <= kMaxMoves, "more than 1048576 moves");
    AFB_CHECK(known_type(type), "unknown element type");
    AFB_CHECK(k >= 1 && k <= kMaxTop, "k must be between 1 and 256");
    // the kernels take logits times log2(e) / T
    AFB_CHECK(temperature > 0.f && std::isfinite(temperature) && std::isfinite(kLog2e * (1.f / temperature)),
              "the temperature must be positive and finite, and so its inverse");
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
                allow_shared<top_listed_kernel<T>>(shared);
                top_listed_kernel<T><<<(unsigned)rows, kThreads, shared, s>>>(n_moves, x, ld, k, inv_t, legal, valid, (int)n_listed,
                                                                              values, moves, log_rest);
                return;
            }
            by_row_length<T>(n_moves, [&](auto threads, auto p) {
                constexpr int NT = decltype(threads)::value;
                top_kernel<T, NT, decltype(p)::value><<<(unsigned)rows, NT, 0, s>>>((int)n_moves, x, ld, k, inv_t, values, moves, log_rest);
            });
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
        AFB_CHECK(std::isfinite(temperature * temperature), "the square of the temperature must be finite");
        AFB_CHECK(upstream_step >= 0, "negative size");
        AFB_CHECK(upstream || !skip_ones, "skip_ones needs the upstream gradient");
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
        const cudaStream_t s = as_stream(stream);
        with_type(type, [&](auto e) {
            using T = decltype(e);
            const T *x = static_cast<const T *>(logits);
            T *g = static_cast<T *>(grad);
            if (legal) {
                const size_t shared = (size_t)((n_moves + 31) / 32) * 4 + (size_t)n_listed * 8 + Named::bytes(k);
                allow_shared<loss_listed_kernel<T>>(shared);
                // a call that may have nothing to do is not worth a CTA per row
                const unsigned grid = (unsigned)(skip_ones ? std::min<int64_t>(rows, 148 * 8) : rows);
                loss_listed_kernel<T><<<grid, kListThreads, shared, s>>>(a, rows, x, g);
                return;
            }
            const size_t held = ((size_t)(n_moves + 2 * Piece<T>::kPer) * sizeof(T) + 15) / 16 * 16;
            const size_t more = Named::bytes(k) + (size_t)((n_moves + 31) / 32) * 4;
            auto go = [&](auto threads, auto ahead) {
                constexpr int NT = decltype(threads)::value;
                constexpr auto kernel = loss_kernel<T, NT, decltype(ahead)::value>;
                const size_t shared = (decltype(ahead)::value ? 2 : 1) * held + more;
                allow_shared<kernel>(shared);
                kernel<<<(unsigned)std::min<int64_t>(rows, resident<kernel>(NT, shared)), NT, shared, s>>>(a, rows, (int)held, x, g);
            };
            // few threads a row, since what every warp does once a row costs more than its share of the elements (35,840 x 4168
            // float32, 16.7 KB: 205 us with 128 threads, 333 with 256, 768 with 512; 16,000 x 4168 bfloat16 97 us with 128, 83
            // with 64); the next row on its way where several CTAs fit an SM all the same (4,096 x 16000 bfloat16, 32 KB: 70 us
            // with it, 61 without and twice the CTAs)
            if (held <= 10 * 1024) go(std::integral_constant<int, 64>{}, std::true_type{});
            else if (held <= 20 * 1024) go(std::integral_constant<int, 128>{}, std::true_type{});
            else if (held <= 40 * 1024) go(std::integral_constant<int, 128>{}, std::false_type{});
            else if (held + more <= 112 * 1024) go(std::integral_constant<int, 256>{}, std::false_type{});
            else {
                const size_t shared = more;
                allow_shared<loss_long_kernel<T>>(shared);
                loss_long_kernel<T><<<(unsigned)std::min<int64_t>(rows, resident<loss_long_kernel<T>>(kLongThreads, shared)), kLongThreads, shared, s>>>(a, rows, x, g);
            }
        });
        AFB_LAUNCHED();
        if (loss) {
            sum_kernel<<<1, 1024, 0, as_stream(stream)>>>(rows, row_loss, (double)scale, loss);
            AFB_LAUNCHED();
        }
    });
}

}  // extern "C"
