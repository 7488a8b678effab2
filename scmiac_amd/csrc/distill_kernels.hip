// A teacher's top logits and the loss of learning from them.
//
//   top_logits       values, idx = the k largest of each row, by (value descending, index ascending);
//                    lse = log sum_j exp(x_j / T)
//   distill forward  t_i = exp(a_i / Ta - c)  over the listed classes, c their log-sum-exp or the teacher's own,
//                    tau = sum t_i,   L = sum_i t_i (log t_i - x[idx_i] / T) + tau lse(x / T)
//   distill backward dL/dx_j = (tau p_j - sum_{i: idx_i = j} t_i) / T,   p = softmax(x / T)
//
// All of it is bound by reading the rows once (and, backward, writing them once): one pass keeps a running
// maximum m and sum of exponentials s per lane, s = sum exp2((x - m) c) with c = log2(e) / T for v_exp_f32.  In the
// loss the difference comes first (LseAcc): x c alone overflows for the lowest values of float32 and bfloat16, which serve as
// masks, and near the maximum, where the weight is, it is exact.  top_logits folds it into one multiply-add as long as
// |x| c is below 2^24 (WaveLse).  A row belongs to one wave (short
// rows), to the four waves of a block, or to several blocks whose results a second kernel joins (few rows).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "train_common.h"
#include "train_kernels.h"

namespace scmiac {
namespace {

using namespace train;

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;        // one entry per lane of a wave
constexpr int kGather = 4;         // candidates of a row, in 64s, that are sorted out in one go (>= kWaves)
// Up to kShortRow classes a wave takes a whole row: a block's four waves would find less than one 16-byte vector per lane
// each.  4096 x 1000 float32, k = 8, with a wave a row / four: loss 10.8 / 12.7 us, top logits 12.1 / 11.8 (k = 8 leaves
// little to sort out); 256 x 2000 7.7 / 7.0 and 9.2 / 8.4.
constexpr int kShortRow = 1024;
// So it does with longer rows where there are many.  Top logits: sorting out a row's candidates is one wave's work, and
// this keeps all of them at it (4096 x 10412 bfloat16, k = 30: 38.6 / 57.0 us).  Loss and gradient, k = 30:
// 4096 x 2000 bfloat16 26.0 / 29.8, 8192 x 4000 53.2 / 58.0, float32 82.7 / 85.2; but 8192 x 8000 float32 184 / 178,
// 2048 x 4000 28.4 / 27.4.
constexpr int kShortTopRow = 16384, kManyTopRows = 2048;
constexpr int kShortLossRow = 4096, kManyLossRows = 4096;
inline bool wave_per_row(long long n, long long v) { return v <= kShortRow || (v <= kShortLossRow && n >= kManyLossRows); }
constexpr int kLoads = 4;          // vectors a lane has in flight
constexpr int kAhead = 4;          // vectors fetched ahead of the one at work, where the k best are kept

// ------------------------------------------------------------------ running log-sum-exp

struct LseAcc {
    float m, r, s;   // maximum; the same, or 0 while that is -inf; sum of exp2((x - r) c)
    __device__ __forceinline__ void init() { m = -INFINITY, r = 0.f, s = 0.f; }
    __device__ __forceinline__ void raise(float vm, float c) {
        if (vm > m) {
            s *= fast_exp2((m - vm) * c);   // m = -inf: 0
            m = r = vm;
        }
    }
    __device__ __forceinline__ void add(float x, float c) { s += fast_exp2((x - r) * c); }
    // another sum, of entries up to its maximum om
    __device__ __forceinline__ void join(float om, float os, float c) {
        raise(om, c);
        s += om == m || om == -INFINITY ? os : os * fast_exp2((om - r) * c);      // (om may be +inf; of -inf, os is 0 or NaN)
    }
    // all lanes of the wave
    __device__ __forceinline__ void join_wave(float c) {
        const float top = wave_max(m);
        s = wave_sum((m == -INFINITY || m == top) ? s : s * fast_exp2((m - top) * c));   // (a NaN stays)
        m = top;
        r = (top == -INFINITY) ? 0.f : top;
    }
};
// joins n (m, s) pairs; the result is the same in whatever lane it is computed
__device__ __forceinline__ LseAcc join_pairs(const float2* p, int n, float c) {
    LseAcc a;
    a.init();
    for (int i = 0; i < n; ++i) a.m = fmaxf(a.m, p[i].x);
    a.r = (a.m == -INFINITY) ? 0.f : a.m;
    for (int i = 0; i < n; ++i) a.s += (p[i].x == -INFINITY || p[i].x == a.m) ? p[i].y : p[i].y * fast_exp2((p[i].x - a.r) * c);
    return a;
}
__device__ __forceinline__ float lse_value(const LseAcc& a, float inv_t) {
    if (a.m == INFINITY && a.s == a.s) return a.m;
    if (a.s == 0.f) return -INFINITY;               // every entry -inf
    return fmaf(a.m == -INFINITY ? 0.f : a.m, inv_t, kLn2 * log2f(a.s));
}

// The same for a wave that has seen a sample of its entries: one reference r for all lanes and no running
// maximum.  An entry may exceed r by up to 64 in the exponent before it is moved (the sum stays
// far from overflow), and (x - r) c is one multiply-add with the product r c rounded; what that rounding does to
// all terms alike, a factor 2^err, is taken out at the end.  From |r| c = 2^24 on (finite masks like -1e9 and below, a
// type's lowest value, small temperatures) the difference comes first: err, up to half a step of r c, is at most 1/2 below and would
// soon be an exponent that overflows.
struct WaveLse {
    float r, rc, err, limit, s;
    int far;
    __device__ __forceinline__ void init(float sample_max, float c) {
        r = -INFINITY, rc = err = s = 0.f, far = 0, limit = -INFINITY;
        if (sample_max != -INFINITY) refer(sample_max, c);
    }
    __device__ __forceinline__ void refer(float to, float c) {
        s *= fast_exp2((r - to) * c - err);
        r = to;
        far = uniform((int)!(fabsf(r) * c < 16777216.f));
        rc = far ? 0.f : r * c;
        err = far ? 0.f : fmaf(r, c, -rc);
        limit = r + 64.f / c;
        s *= fast_exp2(err);
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&f)[N], float vm, float c) {
        if (any_lane(vm > limit)) refer(uniform(wave_max(vm)), c);
        if (!far) {
#pragma unroll
            for (int i = 0; i < N; ++i) s += fast_exp2(fmaf(f[i], c, -rc));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s += f[i] == r ? 1.f : fast_exp2((f[i] - r) * c);      // (r may be +inf)
        }
    }
    __device__ __forceinline__ LseAcc finish() {
        LseAcc a;
        a.s = wave_sum(s) * fast_exp2(-err);
        a.m = r;
        a.r = (r == -INFINITY) ? 0.f : r;
        return a;
    }
};

// ------------------------------------------------------------------ a row, vector by vector

// Calls body(f, first index) for the 16-byte vectors of columns [lo, hi) of a row and one(x, index, valid)
// for the elements in front of the first aligned vector and behind the last, ascending in index for
// every wave.  Wave `w` of `W` takes every W-th kilobyte.
template <typename T, typename Body, typename One>
__device__ __forceinline__ void stream_row(const T* __restrict__ row, long long lo, long long hi, int w, int W, Body body,
                                           One one) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(row + lo);
    long long head = (long long)(((16 - (addr & 15)) & 15) / sizeof(T));
    if (head > hi - lo) head = hi - lo;
    const long long nv = (hi - lo - head) / N;
    const long long tail0 = lo + head + nv * N;
    if (w == 0 && head > 0) {
        const bool valid = lane < head;
        one(valid ? to_f32(row[lo + lane]) : -INFINITY, lo + lane, valid);
    }
    const u32x4* __restrict__ vec = reinterpret_cast<const u32x4*>(row + lo + head);
    const long long step = (long long)W * 64;
    long long v0 = (long long)w * 64;
    for (; v0 + step * (kLoads - 1) + 64 <= nv; v0 += step * kLoads) {
        Vec16<T> buf[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) buf[u].raw = vec[v0 + step * u + lane];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) body(buf[u], lo + head + (v0 + step * u + lane) * N, true);
    }
    for (; v0 < nv; v0 += step) {
        const bool valid = v0 + lane < nv;
        Vec16<T> buf;
        buf.raw = vec[valid ? v0 + lane : nv - 1];
        body(buf, lo + head + (v0 + lane) * N, valid);
    }
    if (w == 0 && tail0 < hi) {
        const bool valid = tail0 + lane < hi;
        one(valid ? to_f32(row[tail0 + lane]) : -INFINITY, tail0 + lane, valid);
    }
}

template <typename T>
__device__ __forceinline__ float unpack(const Vec16<T>& v, float (&f)[Vec16<T>::N]) {
#pragma unroll
    for (int i = 0; i < Vec16<T>::N; ++i) f[i] = v.get(i);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < Vec16<T>::N; ++i) m = fmaxf(m, f[i]);
    return m;
}

// ------------------------------------------------------------------ top k

// An entry: the value as a whole number of the same order in the upper half, ~index in the lower;
// larger is better, and no entry is 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);   // -0 and +0 are the same value
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ u64 make_entry(float x, long long index) {
    return ((u64)order_key(x) << 32) | (uint32_t)~(uint32_t)index;
}

// Candidates lie in the lists as they were read, the value's bits in the upper half and the index in the lower (most
// are dropped again, and turning them into entries would be half of what keeping one costs).
__device__ __forceinline__ u64 raw_candidate(float x, uint32_t index) { return ((u64)__float_as_uint(x) << 32) | index; }
__device__ __forceinline__ u64 entry_of(u64 raw) { return make_entry(__uint_as_float((uint32_t)(raw >> 32)), (uint32_t)raw); }
__device__ __forceinline__ u64 raw_of(u64 entry) { return raw_candidate(key_value((uint32_t)(entry >> 32)), ~(uint32_t)entry); }

// The largest t in [lo, hi] with count(t) >= k, where count falls and count(lo) >= k; an earlier one as soon as its count is
// at most k + slack.  Three thresholds a step: the steps depend on each other, a step's counts do not.
template <typename Count>
__device__ __forceinline__ uint32_t search_threshold(uint32_t lo, uint32_t hi, int k, int slack, bool& exact, int steps, Count count) {
    exact = false;
    while (lo < hi && steps-- > 0) {
        const uint32_t t2 = lo + (hi - lo) / 2 + 1, t1 = lo + (t2 - lo + 1) / 2, t3 = t2 + (hi - t2 + 1) / 2;
        const int c1 = count(t1), c2 = count(t2), c3 = count(t3);
        int c = k + slack + 1;
        if (c3 >= k) lo = t3, c = c3;
        else if (c2 >= k) lo = t2, hi = t3 - 1, c = c2;
        else if (c1 >= k) lo = t1, hi = t2 - 1, c = c1;
        else hi = t1 - 1;
        if (c <= k + slack) {
            exact = true;
            break;
        }
    }
    return lo;
}

// The smallest entry of a selection of at least k of the wave's entries e[0..R) (0: none): exactly the k
// best where slack is 0, up to `slack` more otherwise; k of them reach `from`, if that many are there.  A search over the values, then over the
// indices of one value, each step a compare and a population count per 64 entries.
template <int R>
__device__ __forceinline__ u64 select_from(const u64 (&e)[R], int k, int slack, uint32_t from = 1u) {
    auto count_hi = [&](uint32_t t) {
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) c += __popcll(ballot((uint32_t)(e[r] >> 32) >= t));
        return c;
    };
    if (count_hi(1u) <= k) return 1ull;
    bool exact;
    const uint32_t lo = search_threshold(from, 0xffffffffu, k, slack, exact, 64, count_hi);
    if (exact) return (u64)lo << 32;
    // more than k + slack entries >= lo, fewer than k above it: the rest by index among those of value lo
    int above = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) above += __popcll(ballot((uint32_t)(e[r] >> 32) > lo));
    const int need = k - above;
    const uint32_t l2 = search_threshold(0u, 0xffffffffu, need, 0, exact, 64, [&](uint32_t t) {
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) c += __popcll(ballot((uint32_t)(e[r] >> 32) == lo && (uint32_t)e[r] >= t));
        return c;
    });
    return ((u64)lo << 32) | l2;
}

// writes the entries >= t of the wave to dst[0..), in any order; returns how many
template <int R, bool kRaw = false>
__device__ __forceinline__ int keep_entries(const u64 (&e)[R], u64 t, u64* dst) {
    int n = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const u64 mask = ballot(e[r] >= t);
        if (e[r] >= t) dst[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u))] = kRaw ? raw_of(e[r]) : e[r];
        n += __popcll(mask);
    }
    return n;
}

// the k best (up to `slack` more) of buf[0..cnt) to the front of buf; t: the smallest kept
template <int R>
__device__ __forceinline__ int shrink_list(u64* buf, int cnt, int k, int slack, u64& t) {
    const int lane = threadIdx.x & 63;
    u64 e[R];
    wave_lds_fence();
#pragma unroll
    for (int r = 0; r < R; ++r) e[r] = (r * 64 + lane < cnt) ? entry_of(buf[r * 64 + lane]) : 0ull;
    t = select_from<R>(e, k, slack);
    const int n = keep_entries<R, true>(e, t, buf);
    wave_lds_fence();
    return n;
}

// The candidates of one wave, in LDS: everything that may still be among the k best of what the wave has seen.
template <typename T>
struct WaveList {
    static constexpr int kTrigger = 256;
    static constexpr int kCap = kTrigger + 64 * 4;             // a lot of push_careful adds up to 256 entries
    u64* buf;
    int cnt, k;
    float tau;      // k entries of the list are >= tau; all of them came earlier, so a later entry must exceed it
    bool open;      // fewer than k entries seen: everything is taken
    __device__ __forceinline__ void init(u64* b, int k_) { buf = b, cnt = 0, k = k_, tau = -INFINITY, open = true; }
    __device__ __forceinline__ void shrink(int slack) {
        u64 t;
        // (registers for as many entries as there are: a step of the selection costs three instructions per 64)
        if (cnt <= kTrigger) cnt = shrink_list<kTrigger / 64>(buf, cnt, k, slack, t);
        else if (cnt <= 384) cnt = shrink_list<6>(buf, cnt, k, slack, t);
        else cnt = shrink_list<kCap / 64>(buf, cnt, k, slack, t);
        if (cnt >= k) {
            tau = key_value((uint32_t)(t >> 32));
            open = false;
        }
    }
    // The lanes that `take`: their candidates go behind the others, in the lanes' order; what there is no room for lands in
    // one slot behind the list, and cnt says so (kept free of conditions: cnt stays in a scalar register).
    __device__ __forceinline__ void append(u64 mask, bool take, float x, uint32_t index) {
        if (take) {
            const int at = cnt + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
            buf[min(at, kCap)] = raw_candidate(x, index);
        }
        cnt += __popcll(mask);
    }
    // what of a vector of every lane exceeds tau
    template <int N>
    __device__ __forceinline__ void push(const float (&f)[N], uint32_t first) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool take = f[i] > tau;
            append(ballot(take), take, f[i], first + i);
        }
    }
    // The same with room made first; also while everything is taken (`valid` entries of the lane are real).  256 entries at a
    // time, ascending in index from one lot to the next (of the half types' eight a lane, 32 lanes each): tau may move in
    // between, and leaves out an equal value only if k entries in front of it are kept.
    template <int N>
    __device__ __forceinline__ void push_careful(const float (&f)[N], uint32_t first, int valid) {
        constexpr int kLots = N / 4;
#pragma unroll 1
        for (int h = 0; h < kLots; ++h) {
            const int mine = kLots == 1 || (int)(threadIdx.x & 63) / (64 / kLots) == h ? valid : 0;
            if (!any_lane(mine > 0)) continue;       // (single elements are the first lanes')
            room();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool take = i < mine && (open || f[i] > tau);
                append(ballot(take), take, f[i], first + i);
            }
        }
    }
    __device__ __forceinline__ void room() {
        if (cnt > kTrigger) shrink(k / 4);
    }
};

// Rank of each lane's entry among the wave's (0: the best); lanes from n on have none (0).
__device__ __forceinline__ int rank_of(u64 e, int n) {
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < ((n + 7) & ~7); ++j) {
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(e >> 32), j), lo = __builtin_amdgcn_readlane((uint32_t)e, j);
        rank += ((((u64)hi << 32) | lo) > e) ? 1 : 0;
    }
    return rank;
}

template <typename T>
__device__ __forceinline__ void write_top(u64 e, int found, int k, T* __restrict__ values, int* __restrict__ idx) {
    const int lane = threadIdx.x & 63;
    if (lane < found) {
        const int r = rank_of(e, found);
        values[r] = from_f32<T>(key_value((uint32_t)(e >> 32)));
        idx[r] = (int)~(uint32_t)e;
    } else if (lane < k) {       // fewer classes than k: the tables' padding
        values[lane] = from_f32<T>(-INFINITY);
        idx[lane] = -1;
    }
}

// A value that at least k of the row's (or split's) entries reach, from the largest entry of every lane's first few
// vectors (of a row with one wave, the largest two): the k-th largest of 256 (128) such maxima is
// rarely far below the k-th largest entry, so that of those few thousand entries little more than k become
// candidates instead of all.  0: there are fewer than k maxima.  `keys`: 64 WPR words of LDS of this row.
template <int WPR>
__device__ __forceinline__ uint32_t bound_of_maxima(float max1, float max2, bool any, int k, uint32_t* keys, int w) {
    constexpr int R = WPR == 1 ? 2 : WPR;
    const int lane = threadIdx.x & 63;
    uint32_t e[R];
    e[0] = any ? order_key(max1) : 0u;
    if constexpr (WPR == 1) {
        e[1] = any ? order_key(max2) : 0u;
    } else {
        keys[w * 64 + lane] = e[0];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < WPR; ++q) e[q] = keys[q * 64 + lane];
    }
    auto count = [&](uint32_t t) {
        int c = 0;
#pragma unroll
        for (int q = 0; q < R; ++q) c += __popcll(ballot(e[q] >= t));
        return c;
    };
    if (count(1u) < k) return 0u;
    bool exact;      // (near is enough: ten steps end within 2^12 of it, a two-thousandth of an octave)
    return search_threshold(1u, 0xffffffffu, k, k / 8, exact, 10, count);
}

// Block (row group, split).  WPR: waves per row.  Bound by the stream of logits where rows are long, each class costing a compare
// and an exponential on the way (4096 x 100 000 float16, k = 64: 217 us, 3.8 TB/s), and by the choice among a row's
// candidates where they are short (4096 x 10412 bfloat16, k = 30: 38 us, 2.2 TB/s).
template <typename T, int WPR>
__global__ __launch_bounds__(kThreads) void top_logits_kernel(const T* __restrict__ x, long long ld, long long n, int v,
                                                              int k, float c, float inv_t, int splits, int split_len,
                                                              T* __restrict__ values, int* __restrict__ idx,
                                                              float* __restrict__ lse, u64* __restrict__ part,
                                                              float2* __restrict__ part_ms) {
    constexpr int N = Vec16<T>::N;
    __shared__ u64 lists[kWaves][WaveList<T>::kCap + 1];
    __shared__ float2 ms[kWaves];
    __shared__ int counts[kWaves];
    __shared__ uint32_t maxima[kThreads];
    const int wave = wave_id(), lane = threadIdx.x & 63;
    const int w = wave % WPR;
    const long long row = (long long)blockIdx.x * (kWaves / WPR) + wave / WPR;
    const bool live = row < n;
    const int split = blockIdx.y;
    const int lo = split * split_len, hi = (int)min((long long)v, (long long)lo + split_len);   // (positions in a row fit 31 bits)

    WaveLse sum;
    sum.init(-INFINITY, c);
    WaveList<T> list;
    list.init(lists[wave], k);
    if (live) {
        const T* xr = x + row * ld;
        int head = (int)(((16 - (reinterpret_cast<uintptr_t>(xr + lo) & 15)) & 15) / sizeof(T));
        if (head > hi - lo) head = hi - lo;
        const int nv = (hi - lo - head) / N, body = lo + head, tail = body + nv * N;
        const u32x4* vecs = reinterpret_cast<const u32x4*>(xr + body);
        constexpr int step = WPR * 64;
        int at = w * 64;
        const float none = -INFINITY;
        Vec16<T> empty;
        {
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = none;
            empty.set(f);
        }
        auto fetch = [&](int v0) {
            Vec16<T> r = empty;
            const u32x4* p = vecs + v0;
            if (v0 + 64 <= nv || v0 + lane < nv) r.raw = p[lane];
            return r;
        };
        Vec16<T> ahead[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) ahead[u] = fetch(at + u * step);
        {
            float max1 = none, max2 = none;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float f[N];
                if constexpr (WPR == 1) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float x = ahead[u].get(i);
                        max2 = fmaxf(max2, fminf(max1, x));
                        max1 = fmaxf(max1, x);
                    }
                } else {
                    max1 = fmaxf(max1, unpack<T>(ahead[u], f));
                }
            }
            sum.init(uniform(wave_max(max1)), c);
            const uint32_t bound = bound_of_maxima<WPR>(max1, max2, at + lane < nv, k, maxima, w);
            if (bound > order_key(none)) {
                // everything from the bound on: what exceeds the value below it (-0, just below +0, is no less)
                list.tau = key_value(bound - (bound == order_key(0.f) ? 2u : 1u));
                list.open = false;
            }
        }
        // In turn: the elements in front of the first 16-byte vector; the vectors, every WPR-th kilobyte, kAhead of them at a
        // time while as many are on their way; the elements behind the last one.  A group whose candidates
        // do not fit its list (equal values, rising rows), and everything while fewer than k entries are known, goes vector
        // by vector through the careful path, of which there is one copy.
        bool front = w == 0 && head > 0, back = w == 0 && tail < hi;
        while (true) {
            int from = 0, to = 0;      // the single elements of this turn
            bool careful = false;
            if (front) {
                from = lo, to = body, front = false, careful = true;
            } else if (at < nv) {
                if (list.cnt > WaveList<T>::kTrigger) list.shrink(k / 4);
                const int before = list.cnt;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    float f[N];
                    const float vm = unpack<T>(ahead[u], f);
                    ahead[u] = fetch(at + (kAhead + u) * step);
                    sum.add(f, vm, c);
                    if (any_lane(vm > list.tau)) list.push(f, (uint32_t)body + (uint32_t)(at + u * step + lane) * N);
                    __builtin_amdgcn_sched_barrier(0);      // one vector's floats in registers at a time
                }
                if (!list.open && list.cnt <= WaveList<T>::kCap) {
                    at += kAhead * step;
                    continue;
                }
                list.cnt = before;
                careful = true;
            } else if (back) {
                from = tail, to = hi, back = false, careful = true;
            }
            if (!careful) break;
            const bool single = to > from;
            for (int u = 0; u < (single ? 1 : kAhead); ++u) {
                float f[N];
                uint32_t first;      // (of lanes behind the end it may pass 31 bits)
                int valid;
                if (single) {
                    first = (uint32_t)from + lane;
                    valid = lane < to - from ? 1 : 0;
                    f[0] = valid ? to_f32(xr[first]) : none;
#pragma unroll
                    for (int i = 1; i < N; ++i) f[i] = none;
                    sum.add(f, f[0], c);
                } else {
                    const Vec16<T> v = fetch(at + u * step);
                    unpack<T>(v, f);
                    valid = at + u * step + lane < nv ? N : 0;
                    first = (uint32_t)body + (uint32_t)(at + u * step + lane) * N;
                }
                list.push_careful(f, first, valid);
            }
            if (!single) at += kAhead * step;
        }
    }
    LseAcc acc = sum.finish();
    // the k best of the row's candidates: of all waves' at once, or, where there are many, of each wave's best
    u64 mine = 0;
    int found = 0;
    if (WPR == 1) {
        list.shrink(0);
        found = list.cnt;
        mine = (lane < found) ? entry_of(list.buf[lane]) : 0ull;
    } else {
        if (lane == 0) {
            ms[wave] = make_float2(acc.m, acc.s);
            counts[wave] = list.cnt;
        }
        __syncthreads();
        int ends[kWaves], total = 0;
#pragma unroll
        for (int q = 0; q < kWaves; ++q) ends[q] = total += counts[q];
        const bool many = total > 64 * kGather;
        if (many) {
            list.shrink(0);
            __syncthreads();
            if (lane == 0) counts[wave] = list.cnt;
            __syncthreads();
        }
        if (wave != 0) return;
        u64 e[kGather];
#pragma unroll
        for (int r = 0; r < kGather; ++r) {
            if (many) {
                e[r] = (r < kWaves && lane < counts[r % kWaves]) ? entry_of(lists[r % kWaves][lane]) : 0ull;
            } else {
                const int at = r * 64 + lane;
                int q = 0, from = 0;
#pragma unroll
                for (int o = 0; o + 1 < kWaves; ++o)
                    if (at >= ends[o]) q = o + 1, from = ends[o];
                e[r] = at < total ? entry_of(lists[q][at - from]) : 0ull;
            }
        }
        wave_lds_fence();
        acc = join_pairs(ms, kWaves, c);
        const u64 t = select_from<kGather>(e, k, 0);
        found = keep_entries<kGather>(e, t, lists[0]);
        wave_lds_fence();
        mine = (lane < found) ? lists[0][lane] : 0ull;
    }
    if (!live) return;
    if (splits > 1) {
        if (lane < k) part[(row * splits + split) * k + lane] = mine;
        if (lane == 0) part_ms[row * splits + split] = make_float2(acc.m, acc.s);
        return;
    }
    write_top<T>(mine, found, k, values + row * k, idx + row * k);
    if (lane == 0) lse[row] = lse_value(acc, inv_t);
}

// Joins the splits of a row, k entries each.  The largest value of each of the 64 lanes (of a block's sixteen waves together)
// is an entry's, and the k-th largest of them bounds the k-th best entry: some k log k entries reach it, which one
// wave sorts out.  Only if the good ones meet in few lanes, or are equal, are there more than 1024; then every wave
// keeps the k best of its own first.
// One block's latencies bound this, its instructions' way from memory among them.  244 splits of k = 64: 14.4 us, 18.6 with
// every wave's own k best first.
constexpr int kJoinWaves = 16;
constexpr int kJoinR = 16;         // 64 kJoinWaves kJoinR >= kMaxSplits kMaxTop
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void top_logits_join_kernel(int k, float c, float inv_t, int splits, const u64* __restrict__ part,
                                                                          const float2* __restrict__ part_ms,
                                                                          T* __restrict__ values, int* __restrict__ idx,
                                                                          float* __restrict__ lse) {
    __shared__ u64 best[kJoinWaves * 64];
    __shared__ uint32_t keys[kJoinWaves * 64];
    __shared__ int counter;
    const int wave = wave_id(), lane = threadIdx.x & 63;
    const long long row = blockIdx.x;
    const int total = splits * k;
    const u64* src = part + row * total;
    u64 e[kJoinR];
    uint32_t key = 0u;
#pragma unroll
    for (int r = 0; r < kJoinR; ++r) {
        const int at = r * 64 * kJoinWaves + threadIdx.x;
        e[r] = (at < total) ? src[at] : 0ull;
        key = max(key, (uint32_t)(e[r] >> 32));
    }
    keys[threadIdx.x] = key;
    if (threadIdx.x == 0) counter = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) key = max(key, keys[w * 64 + lane]);
    auto count = [&](uint32_t t) { return (int)__popcll(ballot(key >= t)); };
    uint32_t low = 1u;
    bool exact;
    // (of 64 keys for k = 64, the first threshold that all reach is not good enough)
    if (count(1u) >= k) low = search_threshold(1u, 0xffffffffu, k, k < 64 ? 0 : -1, exact, 12, count);
    int mine_count = 0;
#pragma unroll
    for (int r = 0; r < kJoinR; ++r) mine_count += (uint32_t)(e[r] >> 32) >= low ? 1 : 0;
    if (mine_count) {
        int at = atomicAdd(&counter, mine_count);      // (any order: they are ranked in the end)
#pragma unroll
        for (int r = 0; r < kJoinR; ++r)
            if ((uint32_t)(e[r] >> 32) >= low) {
                if (at < kJoinWaves * 64) best[at] = e[r];
                ++at;
            }
    }
    __syncthreads();
    int all = uniform(counter);
    if (all > kJoinWaves * 64) {
        __syncthreads();                 // the list is given up
        const u64 t = select_from<kJoinR>(e, k, 0);
        const int found = keep_entries<kJoinR>(e, t, best + wave * 64);
        if (lane >= found) best[wave * 64 + lane] = 0ull;
        all = kJoinWaves * 64;
        __syncthreads();
    }
    if (wave == 1) {
        LseAcc acc;
        acc.init();
        for (int i = lane; i < splits; i += 64) {
            const float2 p = part_ms[row * splits + i];
            acc.join(p.x, p.y, c);
        }
        acc.join_wave(c);
        if (lane == 0) lse[row] = lse_value(acc, inv_t);
    }
    if (wave != 0) return;
    int found;
    auto pick = [&](auto size) {
        constexpr int R = decltype(size)::value;
        u64 f[R];
#pragma unroll
        for (int r = 0; r < R; ++r) f[r] = (r * 64 + lane < all) ? best[r * 64 + lane] : 0ull;
        const u64 t = select_from<R>(f, k, 0, low);
        found = keep_entries<R>(f, t, best);
    };
    if (all <= 384) pick(std::integral_constant<int, 6>());
    else pick(std::integral_constant<int, kJoinWaves>());
    wave_lds_fence();
    const u64 mine = (lane < found) ? best[lane] : 0ull;
    write_top<T>(mine, found, k, values + row * k, idx + row * k);
}

// ------------------------------------------------------------------ distillation

// What a row's forward pass leaves for its backward pass, and for the loss:
//   x = the student's maximum m,  y = tau / s, so that tau p_j = y exp2((x_j - m) c): -1 for a row without a teacher (or
//   without a class), NaN for a row with an index that is none;
//   z, w: t_i = exp2((a_i - z) ca - w), the teacher's maximum and log of its sum, or its own normaliser and 0
__device__ __forceinline__ float teacher_weight(float a, float ca, float ref, float log_sum) {
    return fast_exp2(fmaf(a - ref, ca, -log_sum));
}

// One wave: the teacher's distribution of a row against the student's log-sum-exp.
template <typename T>
__device__ __forceinline__ void finish_row(const T* __restrict__ xr, long long v, float c, const LseAcc& acc,
                                           const int* __restrict__ idx, const float* __restrict__ top, int k,
                                           const float* __restrict__ teacher_lse, float ca, float teacher_t, long long row,
                                           float* __restrict__ loss, float4* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    const int* ir = idx + row * k;
    const float* ar = top + row * k;
    float top_max = -INFINITY;
    bool bad = false;
    for (int i = lane; i < k; i += 64) {
        const int j = ir[i];
        bad |= j < -1 || j >= v;
        if (j >= 0 && j < v) {
            const float a = ar[i];
            bad |= a != a;
            top_max = fmaxf(top_max, a);
        }
    }
    top_max = wave_max(top_max);
    bad = any_lane(bad);
    const bool empty = top_max == -INFINITY || (acc.m == -INFINITY && acc.s == 0.f);
    float ref = 0.f, log_sum = 0.f, tau = 0.f, part = 0.f;
    if (!empty) {
        if (teacher_lse) {
            ref = teacher_lse[row] * teacher_t;
        } else {
            ref = top_max;
            float s = 0.f;
            for (int i = lane; i < k; i += 64) {
                const int j = ir[i];
                if (j >= 0 && j < v) s += fast_exp2((ar[i] - ref) * ca);
            }
            log_sum = log2f(wave_sum(s));
        }
        // sum t (log t - (x - max)) + tau log(sum): differences from the row's maximum, where little cancels
        for (int i = lane; i < k; i += 64) {
            const int j = ir[i];
            if (j >= 0 && j < v) {
                const float t = teacher_weight(ar[i], ca, ref, log_sum);
                if (!(t <= 0.f)) {
                    part += t * (fmaf(ar[i] - ref, ca, -log_sum) - (to_f32(xr[j]) - acc.r) * c);
                    tau += t;
                }
            }
        }
        tau = wave_sum(tau);
        part = wave_sum(part);
    }
    if (lane == 0) {
        float value = empty ? 0.f : kLn2 * fmaf(tau, log2f(acc.s), part);
        float share = empty ? -1.f : tau / acc.s;
        if (bad || (!empty && acc.s != acc.s)) value = share = NAN;      // (a row without a teacher may hold anything)
        loss[row] = value;
        stats[row] = make_float4(acc.r, share, ref, log_sum);
    }
}

template <typename T, int WPR>
__global__ __launch_bounds__(kThreads) void distill_forward_kernel(const T* __restrict__ x, long long ld, long long n,
                                                                   long long v, float c, int splits, long long split_len,
                                                                   const int* __restrict__ idx, const float* __restrict__ top,
                                                                   int k, const float* __restrict__ teacher_lse, float ca, float teacher_t,
                                                                   float* __restrict__ loss, float4* __restrict__ stats,
                                                                   float2* __restrict__ part_ms) {
    constexpr int N = Vec16<T>::N;
    __shared__ float2 ms[kWaves];
    const int wave = wave_id(), lane = threadIdx.x & 63;
    const int w = wave % WPR;
    const long long row = (long long)blockIdx.x * (kWaves / WPR) + wave / WPR;
    const bool live = row < n;
    const int split = blockIdx.y;
    const long long lo = split * split_len, hi = min(v, lo + split_len);
    const T* xr = x + row * ld;
    LseAcc acc;
    acc.init();
    if (live) {
        stream_row<T>(
            xr, lo, hi, w, WPR,
            [&](const Vec16<T>& vec, long long, bool valid) {
                float f[N];
                const float vm = unpack<T>(vec, f);
                if (valid) {
                    acc.raise(vm, c);
#pragma unroll
                    for (int i = 0; i < N; ++i) acc.add(f[i], c);
                }
            },
            [&](float xv, long long, bool valid) {
                if (valid) {
                    acc.raise(xv, c);
                    acc.add(xv, c);
                }
            });
        acc.join_wave(c);
    }
    if (WPR > 1) {
        if (lane == 0) ms[wave] = make_float2(acc.m, acc.s);
        __syncthreads();
        if (wave != 0) return;
        acc = join_pairs(ms, kWaves, c);
    }
    if (!live) return;
    if (splits > 1) {
        if (lane == 0) part_ms[row * splits + split] = make_float2(acc.m, acc.s);
        return;
    }
    finish_row<T>(xr, v, c, acc, idx, top, k, teacher_lse, ca, teacher_t, row, loss, stats);
}

template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(const T* __restrict__ x, long long ld, long long v, float c, int splits,
                                                          const float2* __restrict__ part_ms, const int* __restrict__ idx,
                                                          const float* __restrict__ top, int k,
                                                          const float* __restrict__ teacher_lse, float ca, float teacher_t,
                                                          float* __restrict__ loss, float4* __restrict__ stats) {
    const long long row = blockIdx.x;
    LseAcc acc;
    acc.init();
    for (int i = threadIdx.x; i < splits; i += 64) {
        const float2 p = part_ms[row * splits + i];
        acc.join(p.x, p.y, c);
    }
    acc.join_wave(c);
    finish_row<T>(x + row * ld, v, c, acc, idx, top, k, teacher_lse, ca, teacher_t, row, loss, stats);
}

// Sum (mean: over the rows that have a teacher) of the rows' losses, in an order that depends on n alone.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(const float* __restrict__ row_loss,
                                                                  const float4* __restrict__ stats, long long n, int mean,
                                                                  float* __restrict__ loss, float* __restrict__ scale) {
    __shared__ double sums[kSumThreads / 64];
    __shared__ int counts[kSumThreads / 64];
    double sum = 0.0;
    int count = 0;
    for (long long i = threadIdx.x; i < n; i += kSumThreads) {
        sum += (double)row_loss[i];
        count += !(stats[i].y < 0.f);
    }
    for (int off = 32; off; off >>= 1) {
        sum += __shfl_xor(sum, off);
        count += __shfl_xor(count, off);
    }
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = sum;
        counts[threadIdx.x >> 6] = count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        count = 0;
        for (int i = 0; i < kSumThreads / 64; ++i) {
            sum += sums[i];
            count += counts[i];
        }
        const double d = (mean && count > 1) ? (double)count : 1.0;
        loss[0] = (float)(sum / d);
        scale[0] = (float)(1.0 / d);
    }
}

// Bound by memory: 8192 x 100 000 bfloat16, k = 64, 720 us, 4.5 TB/s read and written (forward 330 us, 5.0 TB/s read).
// Block (row group, split): the dense part of the split's columns, then the listed classes among them.
// The dense pass has written tau p g / T there; the second write replaces it with the difference, computed
// in float32 from x again, so that nothing is lost where p and t nearly cancel.
template <typename T, int WPR>
__global__ __launch_bounds__(kThreads) void distill_backward_kernel(const T* __restrict__ x, long long ld, long long n,
                                                                    long long v, float c, float inv_t, int splits,
                                                                    long long split_len, const int* __restrict__ idx,
                                                                    const float* __restrict__ top, int k, float ca,
                                                                    const float4* __restrict__ stats,
                                                                    const float* __restrict__ grad, long long grad_stride,
                                                                    const float* __restrict__ scale, T* __restrict__ dx,
                                                                    long long ldd) {
    constexpr int N = Vec16<T>::N;
    extern __shared__ int listed[];       // [kWaves / WPR][k]
    const int wave = wave_id(), lane = threadIdx.x & 63;
    const int w = wave % WPR, group = wave / WPR;
    const long long row = (long long)blockIdx.x * (kWaves / WPR) + group;
    const bool live = row < n;
    const int split = blockIdx.y;
    const long long lo = split * split_len, hi = min(v, lo + split_len);
    const T* xr = x + row * ld;
    T* dr = dx + row * ldd;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    float g = 0.f;
    if (live) {
        st = stats[row];
        g = grad[row * grad_stride] * inv_t;
        if (scale) g *= scale[0];
        int* mine = listed + group * k;
        for (int i = w * 64 + lane; i < k; i += WPR * 64) mine[i] = idx[row * k + i];
        const float f0 = st.y * g;
        const bool empty = st.y < 0.f;
        auto dense = [&](float xv) { return empty ? 0.f : f0 * fast_exp2((xv - st.x) * c); };
        if (((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0) {
            stream_row<T>(
                xr, lo, hi, w, WPR,
                [&](const Vec16<T>& vec, long long first, bool valid) {
                    float f[N];
                    unpack<T>(vec, f);
#pragma unroll
                    for (int i = 0; i < N; ++i) f[i] = dense(f[i]);
                    Vec16<T> out;
                    out.set(f);
                    if (valid) *reinterpret_cast<u32x4*>(dr + first) = out.raw;
                },
                [&](float xv, long long index, bool valid) {
                    if (valid) dr[index] = from_f32<T>(dense(xv));
                });
        } else {      // rows of x and dx that start at different offsets from 16 bytes
            for (long long j = lo + w * 64 + lane; j < hi; j += WPR * 64) dr[j] = from_f32<T>(dense(to_f32(xr[j])));
        }
    }
    __syncthreads();
    if (!live || st.y < 0.f) return;
    const int* mine = listed + group * k;
    const float* ar = top + row * k;
    for (int i = w * 64 + lane; i < k; i += WPR * 64) {
        const int j = mine[i];
        if (j < lo || j >= hi) continue;
        // a class that is listed more than once is written by its first entry, with all of its weight
        bool first = true;
        for (int q = 0; q < i; ++q) first &= mine[q] != j;
        if (!first) continue;
        float t = 0.f;
        for (int q = i; q < k; ++q)
            if (mine[q] == j) t += teacher_weight(ar[q], ca, st.z, st.w);
        dr[j] = from_f32<T>(g * fmaf(st.y, fast_exp2((to_f32(xr[j]) - st.x) * c), -t));
    }
}

// ------------------------------------------------------------------ launch shapes

// Splits of a row: enough blocks for the chip's 256 compute units several times over, none shorter than
// 4096 columns (16 KiB of float32: below that a block's start and end cost more than its columns), no
// more than a join can take.  Top logits of float32 rows, k = 30, with at least 2048 / 4096 / 16384 columns a split:
// 1 x 100 000 15.9 / 16.8 / 20.2 us, 64 x 30 000 19.5 / 18.6 / 20.4, 64 x 100 000 21.2 / 21.5 / 22.3.
constexpr long long kMinSplit = 4096;
constexpr int kMaxSplits = 256;
void plan_splits(long long n, long long v, int esize, int& splits, long long& len) {
    splits = 1;
    len = v;
    if (v <= kShortRow || n < 1) return;
    const long long want = ceil_div(1024, n);
    long long s = want < v / kMinSplit ? want : v / kMinSplit;
    if (s > kMaxSplits) s = kMaxSplits;
    if (s <= 1) return;
    len = round_up(ceil_div(v, s), 64 * (16 / esize));
    splits = (int)ceil_div(v, len);
    if (splits == 1) len = v;
}

inline int esize_of(int dtype) { return dtype == 0 ? 4 : 2; }

template <typename T>
hipError_t top_logits_t(const void* x, long long ld, long long n, long long v, int k, float temperature, void* values,
                        int* idx, float* lse, void* ws, hipStream_t stream) {
    const float c = kLog2e / temperature;
    int splits;
    long long len;
    plan_splits(n, v, sizeof(T), splits, len);
    const T* xt = static_cast<const T*>(x);
    T* vt = static_cast<T*>(values);
    u64* part = static_cast<u64*>(ws);
    float2* part_ms = reinterpret_cast<float2*>(part + (size_t)n * splits * k);
    if (v <= kShortRow || (v <= kShortTopRow && n >= kManyTopRows)) {
        top_logits_kernel<T, 1><<<dim3((unsigned)ceil_div(n, kWaves)), kThreads, 0, stream>>>(xt, ld, n, (int)v, k, c, 1.f / temperature, 1, (int)v, vt, idx,
                                                                                               lse, nullptr, nullptr);
    } else {
        top_logits_kernel<T, kWaves><<<dim3((unsigned)n, splits), kThreads, 0, stream>>>(xt, ld, n, (int)v, k, c, 1.f / temperature, splits, (int)len, vt,
                                                                                        idx, lse, part, part_ms);
        if (splits > 1)
            top_logits_join_kernel<T><<<dim3((unsigned)n), 64 * kJoinWaves, 0, stream>>>(k, c, 1.f / temperature, splits, part, part_ms, vt, idx, lse);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t distill_forward_t(const DistillArgs& a, int reduction, float* loss, float4* stats, float* scale, void* ws,
                             hipStream_t stream) {
    const float c = kLog2e / a.temperature, ca = kLog2e / a.teacher_temperature;
    int splits;
    long long len;
    plan_splits(a.n, a.v, sizeof(T), splits, len);
    const T* x = static_cast<const T*>(a.x);
    float2* part_ms = static_cast<float2*>(ws);
    float* row_loss = reduction == 0 ? loss : reinterpret_cast<float*>(part_ms + (size_t)a.n * splits);
    if (a.n > 0) {
        if (wave_per_row(a.n, a.v)) {
            distill_forward_kernel<T, 1><<<dim3((unsigned)ceil_div(a.n, kWaves)), kThreads, 0, stream>>>(
                x, a.ld, a.n, a.v, c, 1, a.v, a.idx, a.top, a.k, a.teacher_lse, ca, a.teacher_temperature, row_loss, stats, nullptr);
        } else {
            distill_forward_kernel<T, kWaves><<<dim3((unsigned)a.n, splits), kThreads, 0, stream>>>(
                x, a.ld, a.n, a.v, c, splits, len, a.idx, a.top, a.k, a.teacher_lse, ca, a.teacher_temperature, row_loss, stats, part_ms);
            if (splits > 1)
                distill_join_kernel<T><<<dim3((unsigned)a.n), 64, 0, stream>>>(x, a.ld, a.v, c, splits, part_ms, a.idx, a.top,
                                                                              a.k, a.teacher_lse, ca, a.teacher_temperature, row_loss, stats);
        }
    }
    if (reduction != 0)
        distill_sum_kernel<<<1, kSumThreads, 0, stream>>>(row_loss, stats, a.n, reduction == 1, loss, scale);
    return hipGetLastError();
}

template <typename T>
hipError_t distill_backward_t(const DistillArgs& a, const float4* stats, const float* grad, long long grad_stride,
                              const float* scale, void* dx, long long ldd, hipStream_t stream) {
    const float c = kLog2e / a.temperature, ca = kLog2e / a.teacher_temperature;
    int splits;
    long long len;
    plan_splits(a.n, a.v, sizeof(T), splits, len);
    const T* x = static_cast<const T*>(a.x);
    T* d = static_cast<T*>(dx);
    if (wave_per_row(a.n, a.v))
        distill_backward_kernel<T, 1><<<dim3((unsigned)ceil_div(a.n, kWaves)), kThreads, sizeof(int) * kWaves * a.k, stream>>>(
            x, a.ld, a.n, a.v, c, 1.f / a.temperature, 1, a.v, a.idx, a.top, a.k, ca, stats, grad, grad_stride, scale, d, ldd);
    else
        distill_backward_kernel<T, kWaves><<<dim3((unsigned)a.n, splits), kThreads, sizeof(int) * a.k, stream>>>(
            x, a.ld, a.n, a.v, c, 1.f / a.temperature, splits, len, a.idx, a.top, a.k, ca, stats, grad, grad_stride, scale, d,
            ldd);
    return hipGetLastError();
}

}  // namespace

size_t top_logits_workspace_bytes(long long n, long long v, int k, int dtype) {
    int splits;
    long long len;
    plan_splits(n, v, esize_of(dtype), splits, len);
    return splits > 1 ? (size_t)n * splits * ((size_t)k * sizeof(u64) + sizeof(float2)) : 0;
}

size_t distill_workspace_bytes(long long n, long long v, int dtype) {
    if (n == 0) return 0;
    int splits;
    long long len;
    plan_splits(n, v, esize_of(dtype), splits, len);
    return (size_t)n * splits * sizeof(float2) + (size_t)n * sizeof(float);
}

hipError_t launch_top_logits(const void* x, long long ld, long long n, long long v, int dtype, int k, float temperature,
                             void* values, int* idx, float* lse, void* ws, hipStream_t stream) {
    if (n == 0) return hipSuccess;
    switch (dtype) {
        case 0: return top_logits_t<float>(x, ld, n, v, k, temperature, values, idx, lse, ws, stream);
        case 1: return top_logits_t<f16>(x, ld, n, v, k, temperature, values, idx, lse, ws, stream);
        default: return top_logits_t<bf16>(x, ld, n, v, k, temperature, values, idx, lse, ws, stream);
    }
}

hipError_t launch_distill_forward(const DistillArgs& a, int reduction, float* loss, float* row_stats, float* scale,
                                  void* ws, hipStream_t stream) {
    float4* stats = reinterpret_cast<float4*>(row_stats);
    if (a.n == 0 && reduction == 0) return hipSuccess;
    switch (a.dtype) {
        case 0: return distill_forward_t<float>(a, reduction, loss, stats, scale, ws, stream);
        case 1: return distill_forward_t<f16>(a, reduction, loss, stats, scale, ws, stream);
        default: return distill_forward_t<bf16>(a, reduction, loss, stats, scale, ws, stream);
    }
}

hipError_t launch_distill_backward(const DistillArgs& a, const float* row_stats, const float* grad, long long grad_stride,
                                   const float* scale, void* dx, long long ldd, hipStream_t stream) {
    const float4* stats = reinterpret_cast<const float4*>(row_stats);
    if (a.n == 0) return hipSuccess;
    switch (a.dtype) {
        case 0: return distill_backward_t<float>(a, stats, grad, grad_stride, scale, dx, ldd, stream);
        case 1: return distill_backward_t<f16>(a, stats, grad, grad_stride, scale, dx, ldd, stream);
        default: return distill_backward_t<bf16>(a, stats, grad, grad_stride, scale, dx, ldd, stream);
    }
}

}  // namespace scmiac
