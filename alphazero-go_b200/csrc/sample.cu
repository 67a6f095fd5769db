// The move sampler: one index per row of logits.
//
// With l the legal, non-NaN logits above -inf and m their maximum, x = 0
// where l = m and (l - m) / T elsewhere, w = exp(x). In descending order of l
// (ties: lower index first) top-k keeps the first k, top-p of those the
// shortest prefix whose share of their mass reaches p, min-p those with w >=
// min_p; the first is always kept. Among the kept the move is the argmax of
// x - log(-log u): with u uniform that is a draw from the kept w's
// distribution, without a cumulative sum whose rounding would move the
// boundaries between neighbours.
//
// What each filter keeps is a prefix of the descending order, so it is
// written as a threshold: a key (the logit's bits, ordered as unsigned
// integers) and, where several logits equal it, how many of those. The
// threshold is found by halving the range of keys, each time counting and
// weighing the logits at or above the middle, until one logit (or one group
// of equal ones) is left in the range (rows beyond a warp: mostly from a
// histogram). Counts are exact and sums run in a fixed order, so a row's move
// does not depend on the run or on the other rows.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "ops.hpp"
#include "sm100.cuh"

namespace azb {

namespace {

constexpr float kULow = 2.98023223876953125e-08f;    // 2^-25
constexpr float kUHigh = 0.999999940395355224609375f;   // 1 - 2^-24
constexpr uint32_t kKeyLow = 0x00800000u;             // the key of the lowest finite logit

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

// A logit as an unsigned integer of the same order; -inf is below kKeyLow.
// (Adding +0 makes -0 and +0 the same key, as they are the same logit.)
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}

// Noise as the race takes it; a NaN is read as the lowest number.
__device__ __forceinline__ float clamped(float u) { return fminf(fmaxf(u, kULow), kUHigh); }

__device__ __forceinline__ float race(float x, float u) { return x - logf(-logf(clamped(u))); }

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

__device__ __forceinline__ float ex2(float y) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}

__device__ __forceinline__ float lg2(float x) {   // x >= 2^-25
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// w = 2^((l - m) c). The bounds (the least positive number, and what a
// temperature of 5e-39 gives) keep 0 * c and -inf * c what they should be
// whatever the temperature.
__device__ __forceinline__ float log2_scale(float temperature) {
    return fminf(fmaxf(kLog2e / temperature, __uint_as_float(1u)), 3e38f);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// A row's numbers.
struct RowParams {
    float temperature, top_p, min_p;
    int top_k;
    __device__ RowParams(const SampleArgs& a, long long row)
        : temperature(a.temperature_rows ? a.temperature_rows[row] : a.temperature),
          top_p(a.top_p_rows ? a.top_p_rows[row] : a.top_p),
          min_p(a.min_p_rows ? a.min_p_rows[row] : a.min_p),
          top_k(a.top_k_rows ? a.top_k_rows[row] : a.top_k) {}
    __device__ bool greedy() const { return !(temperature > 0.0f); }
    __device__ bool filters_p() const { return top_p < 1.0f; }   // false for a NaN
    // How many the first filter keeps (0 or less: all): top-p 0 keeps one.
    __device__ int first_k() const { return filters_p() && !(top_p > 0.0f) ? 1 : top_k; }
};

// Logits with key > key, and the first `ties` with key == key.
struct Threshold {
    uint32_t key;
    int ties;
};
constexpr int kAllTies = 0x7FFFFFFF;

struct Weighed {
    int count;
    float mass;
};

__device__ __forceinline__ float logit_of_key(uint32_t key) {
    return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}

// A key inside (lo, hi), hi - lo > 1: the middle logit's for the first steps,
// which about halves the logits between where they lie evenly; then the
// middle key, which ends after 32 steps whatever their distribution.
__device__ __forceinline__ uint32_t between(uint32_t lo, uint32_t hi, int step) {
    if (step < 16) {
        const uint32_t mid = key_of(0.5f * logit_of_key(lo) + 0.5f * logit_of_key(hi));
        if (mid > lo && mid < hi) return mid;
    }
    return lo + (hi - lo) / 2;
}

// The threshold of a row's filters. at(k): count and mass of the logits
// with key >= k, the same on every calling thread; count_at(k): the count
// alone. top: the largest key; low_k, low_p: keys at or below which top-k's
// and top-p's cuts should lie (a hint: the lowest key is tried otherwise).
template <class At, class CountAt>
__device__ Threshold find_threshold(const RowParams& rp, uint32_t top, uint32_t low_k, uint32_t low_p, int valid, float mass,
                                    At at, CountAt count_at) {
    Threshold th{kKeyLow, kAllTies};
    const int k = rp.first_k();
    float kept = mass;   // mass of what is kept so far
    if (k > 0 && k < valid) {
        uint32_t lo = max(low_k, kKeyLow), hi = top + 1;   // count(lo) >= k > count(hi)
        int clo = lo > kKeyLow ? count_at(lo) : valid, chi = 0;
        if (clo < k) hi = lo, chi = clo, lo = kKeyLow, clo = valid;
        for (int step = 0; hi - lo > 1 && clo != k; ++step) {
            const uint32_t mid = between(lo, hi, step);
            const int n = count_at(mid);
            if (n >= k) lo = mid, clo = n;
            else hi = mid, chi = n;
        }
        th.key = lo;
        if (clo != k) th.ties = k - chi;   // ties at lo: the first k - count(hi) of them
        if (k == 1 || !rp.filters_p()) return th;
        kept = at(lo).mass;
        if (clo != k) {
            const float above = at(hi).mass;
            kept = above + (kept - above) * (float(th.ties) / float(clo - chi));
        }
    }
    if (rp.filters_p() && k != 1) {   // (a row with one logit, or a top-p of 0 or less, is settled)
        const float target = rp.top_p * kept;
        uint32_t lo = max(low_p, th.key), hi = top + 1;   // mass(lo) >= target > mass(hi)
        Weighed wlo = at(lo), whi{0, 0.0f};
        if (wlo.mass < target && lo > th.key) {
            hi = lo, whi = wlo;
            lo = th.key, wlo = at(lo);
        }
        for (int step = 0; hi - lo > 1 && wlo.count - whi.count > 1; ++step) {
            const uint32_t mid = between(lo, hi, step);
            const Weighed w = at(mid);
            if (w.mass >= target) lo = mid, wlo = w;
            else hi = mid, whi = w;
        }
        const int group = wlo.count - whi.count;   // equal logits unless there is only one
        int ties = kAllTies;
        if (group > 1) {
            const double each = (double(wlo.mass) - double(whi.mass)) / group;
            const double need = each > 0.0 ? ceil((double(rp.top_p) * double(kept) - double(whi.mass)) / each) : double(group);
            ties = need < 1.0 ? 1 : need >= double(group) ? kAllTies : int(need);
        }
        if (lo > th.key) th = Threshold{lo, ties};
        else th.ties = min(th.ties, ties);
    }
    return th;
}

// -------------------------------------------------------- a warp per row
//
// Up to 32 * kPer columns: lane l holds columns l, l + 32, ... in registers.
// One warp has no other to hide its latency behind, so everything is asked
// for at once, the reductions are single instructions where the type allows,
// and the race's two accurate logarithms are taken only for the columns that
// cheap bounds of their keys leave in it.
//
// Bound by the latency of its steps: one row of 362 in 3.0 us, with top-k and
// top-p, whose halvings follow one another, 6.0 us; 1024 rows of 362 with all
// filters 8.7 us, 21% of the issue slots used. (Masses in fixed point, one
// instruction a sum instead of five exchanges: 8.5 us, but 1024 rows of 1000
// 19.4 instead of 18.6.)
template <typename T, int kPer>
__global__ void __launch_bounds__(128) sample_warp_kernel(const SampleArgs a) {
    grid_dependency_wait();     // every earlier launch has completed,
    grid_launch_dependents();   // so the next may start
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 31;
    constexpr uint32_t kFull = 0xFFFFFFFFu;
    const RowParams rp(a, row);
    const T* logits = static_cast<const T*>(a.logits) + size_t(row) * size_t(a.ld);
    const uint8_t* legal = a.legal ? a.legal + size_t(row) * size_t(a.legal_ld) : nullptr;
    const float* noise = a.noise ? a.noise + size_t(row) * size_t(a.noise_ld) : nullptr;
    float l[kPer], u[kPer];   // the numbers are few: asked for before it shows which are needed
    {
        T raw[kPer];
        uint8_t open[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = j * 32 + lane;
            const bool in = i < a.cols;
            raw[j] = in ? logits[i] : T(0.0f);
            open[j] = in ? (legal ? legal[i] : uint8_t(1)) : uint8_t(0);
            u[j] = in && noise ? __ldg(noise + i) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) l[j] = open[j] ? fmaxf(float(raw[j]), neg_inf()) : neg_inf();   // (a NaN: -inf)
    }
    float lane_top = neg_inf();
#pragma unroll
    for (int j = 0; j < kPer; ++j) lane_top = fmaxf(lane_top, l[j]);
    uint32_t top = __reduce_max_sync(kFull, key_of(lane_top));
    float m = logit_of_key(top);
    if (m == neg_inf()) {   // nothing to choose from
        if (lane == 0) {
            a.moves[row] = -1;
            if (a.logprob) a.logprob[row] = neg_inf();
        }
        return;
    }
    if (rp.greedy()) {
        uint32_t first = 0xFFFFFFFFu;
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j)
            if (l[j] == m) first = uint32_t(j * 32 + lane);
        first = __reduce_min_sync(kFull, first);
        if (lane == 0) {
            a.moves[row] = (long long)first;
            if (a.logprob) a.logprob[row] = 0.0f;
        }
        return;
    }
    if (m == __uint_as_float(0x7F800000u)) {   // the infinite logits share everything
#pragma unroll
        for (int j = 0; j < kPer; ++j) l[j] = l[j] == m ? 0.0f : neg_inf();
        lane_top = lane_top == m ? 0.0f : neg_inf();
        m = 0.0f;
        top = key_of(m);
    }
    const float c = log2_scale(rp.temperature);
    float w[kPer], z = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        w[j] = ex2((l[j] - m) * c);
        z += w[j];
    }
    z = warp_sum(z);
    uint32_t in = 0;   // this lane's kept columns, bit j for column j * 32 + lane
    Threshold th{kKeyLow, kAllTies};
    if (rp.first_k() > 0 || rp.filters_p()) {
        const auto count_at = [&](uint32_t at) {
            unsigned n = 0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) n += key_of(l[j]) >= at;
            return int(__reduce_add_sync(kFull, n));
        };
        const auto at = [&](uint32_t key) {
            Weighed s{0, 0.0f};
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (key_of(l[j]) >= key) {
                    ++s.count;
                    s.mass += w[j];
                }
            s.count = int(__reduce_add_sync(kFull, unsigned(s.count)));
            s.mass = warp_sum(s.mass);
            return s;
        };
        // Up to 32, the k-th largest is at least the least of the lanes'
        // largest; beyond, at least the least of all.
        float least = lane_top;
        if (rp.first_k() > 32) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) least = fminf(least, l[j] > neg_inf() ? l[j] : least);
        }
        const uint32_t low_k = __reduce_min_sync(kFull, least > neg_inf() ? key_of(least) : 0xFFFFFFFFu);
        const uint32_t low_p = key_of(m + __log2f((1.0f - rp.top_p) * 0.99f * z / float(a.cols)) / c);
        th = find_threshold(rp, top, low_k, low_p, rp.first_k() > 0 ? count_at(kKeyLow) : 0, z, at, count_at);
    }
    int seen = 0;   // logits equal to the threshold, in columns before
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t key = key_of(l[j]);
        bool keep = key >= th.key && (l[j] == m || !(rp.min_p > 0.0f) || w[j] >= rp.min_p);
        if (th.ties != kAllTies) {
            const uint32_t tied = __ballot_sync(kFull, key == th.key);
            if (key == th.key && seen + __popc(tied & ((1u << lane) - 1u)) >= th.ties) keep = false;
            seen += __popc(tied);
        }
        in |= keep ? 1u << j : 0u;
    }
    // With d = 1 - u: d <= -log u <= d / u, so a column's key x - log(-log u)
    // lies, in log2, between y - lg2(d) + lg2(u) and y - lg2(d). Only those
    // whose upper bound reaches the largest lower one (less the logarithms'
    // error) can win.
    float need = neg_inf();
    const auto upper = [&](int j) { return (l[j] - m) * c - lg2(1.0f - u[j]); };
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        u[j] = clamped(u[j]);
        if (in >> j & 1u) need = fmaxf(need, upper(j) + lg2(u[j]));
    }
    need = logit_of_key(__reduce_max_sync(kFull, key_of(need))) - 2e-3f;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (!(upper(j) >= need)) in &= ~(1u << j);
    uint32_t best = 0, best_i = 0xFFFFFFFFu;   // the largest key of the race, as an ordered integer
    float best_x = 0.0f;
    while (in) {
        const int b = __ffs(int(in)) - 1, i = b * 32 + lane;
        in &= in - 1;
        float lb = 0.0f, ub = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j == b) lb = l[j], ub = u[j];
        const float x = (lb - m) * c * kLn2;
        const uint32_t key = key_of(race(x, ub));
        if (key > best) best = key, best_i = uint32_t(i), best_x = x;   // (columns ascend)
    }
    __syncwarp();
    const uint32_t winner = __reduce_max_sync(kFull, best);
    const uint32_t column = __reduce_min_sync(kFull, best == winner ? best_i : 0xFFFFFFFFu);
    if (best == winner && best_i == column) {
        a.moves[row] = (long long)column;
        if (a.logprob) a.logprob[row] = best_x - logf(z);
    }
}

// ------------------------------------------------------ a cluster per row
//
// More columns: a cluster of CTAs per row, each with a slice of the columns
// in shared memory, so that the logits cross HBM once however many passes
// the filters need. (A slice too long for that is read again from global
// memory: kResident false.) The number of CTAs follows from the columns, and
// beyond 16384 from whether there are many rows: the only way in which the
// order of a row's sums, and with it their last bits, depends on the batch.
//
// A filter's threshold is found from a histogram of the upper logits in
// kBins equal steps of log w, each bin with its count and its mass in fixed
// point (integers: the order of the atomics does not show). The bin in which
// the threshold lies is known from its cumulative sums to within their
// rounding; the logits in it (a list of at most kList) are sorted and the
// exact cut found among them, on top of the exact count and mass of what lies
// above. Where the list would be longer (many equal logits, say) the range of
// keys is halved as in find_threshold, over the listed upper logits.
//
// 512 rows of 131072 (fp32, top-p 0.9) take 270 us: 469 MB from DRAM (the
// kept columns' numbers come in sectors of 32 bytes), a fifth of its rate. A
// CTA lives 25 us, of which the load takes 3.4, the sum 1.9, the first
// exchange 2.2, the list and histogram 5.1 with their exchange, the cut 9
// with four more; three CTAs an SM (their slices fill it) overlap these, the
// barriers of a cluster's eight being what is waited for. Without filters
// 179 us. (One CTA a row, its passes reading L2: 375 us, and one row 76 us
// where a cluster takes 18.)
//
// Up to 64 (a warp each of a cluster) top-k needs no histogram: the k-th
// largest of the warps' maxima bounds the k-th largest logit from below, and
// what lies above it is the list (8 x 50001 with all filters 12.6 -> 11.2 us,
// 512 x 131072 top-k 50 and top-p 211 -> 195 us).
//
// Lower bounds keep most logits out of the histogram: with k <= the number of
// groups of threads that hold a logit, the k-th largest is at least the least
// of the groups' maxima (groups of 1, 2, .. 32 threads: the largest that are
// still enough); and logits with w < (1 - p) Z / cols have together less
// than (1 - p) Z, so the prefix that top-p keeps ends above them.

constexpr int kMaxCluster = 8, kMaxRowWarps = 8;
constexpr int kBins = 512, kList = 256, kUpper = 2048;
// Gumbel noise -log(-log u) lies in [-2.86, 16.64]: a logit with x < -19.6
// loses to the maximum whatever their numbers, which need not be read.
constexpr float kNoChance = -19.6f;

// Descending order of logits, ties by ascending column, as descending numbers.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) { return uint64_t(key) << 32 | uint32_t(~uint32_t(i)); }

constexpr int kGroupSizes = 6;   // groups of 2^0 .. 2^5 threads
struct Part {   // what one CTA knows of its slice
    float top;                // largest logit
    float z;                  // sum of w relative to `top`
    int valid;                // logits above -inf
    float low[kGroupSizes];   // least of its groups' largest logits
    int groups[kGroupSizes];  // groups that hold a logit
};

struct __align__(16) RowShared {
    uint32_t hist_n[kBins], hist_w[kBins];            // this CTA's; then the lists
    union {
        struct {   // a cluster's CTA: its share of the bins, added over the cluster
            uint32_t share_n[kBins / 2], share_w[kBins / 2];
        };
        struct {   // before that: of each warp's groups
            float low[kGroupSizes][kMaxRowWarps];
            int groups[kGroupSizes][kMaxRowWarps];
            alignas(16) float warp_top[kMaxCluster][kMaxRowWarps];   // each CTA's warps' largest logits
        };
    };
    uint16_t upper[kUpper];                           // the slice's upper columns, a part for each warp
    Part part[kMaxCluster];
    float f[2][kMaxCluster];
    int n[2][kMaxCluster];
    unsigned long long best[kMaxCluster];
    float best_x[kMaxCluster];
    float wf[kMaxRowWarps], wg[kMaxRowWarps], wh[kMaxRowWarps];
    int wn[kMaxRowWarps], wm[kMaxRowWarps], wk[kMaxRowWarps];
    unsigned list_n;
    int first, last;
    uint32_t down, above;
    float kept;
    uint64_t cut;
};
static_assert(kList * 2 * 8 <= int(sizeof(uint32_t)) * kBins * 2, "a CTA's list and the merged one take the histogram's place");

// The CTAs that share a row: kThreads each, one of them (kSolo) or a cluster.
template <int kThreads_, bool kSolo_>
struct Team {
    static constexpr int kThreads = kThreads_, kWarps = kThreads / 32;
    static constexpr bool kSolo = kSolo_;
    int rank, ranks;
    // The address of *p in CTA r.
    template <typename P>
    __device__ __forceinline__ uint32_t at(P* p, int r) const {
        return kSolo ? smem_u32(p) : mapa(smem_u32(p), uint32_t(r));
    }
    __device__ __forceinline__ void barrier() const {
        if constexpr (kSolo) {
            __syncthreads();
        } else {
            __syncwarp();
            cluster_sync();
        }
    }
};
__device__ __forceinline__ void put_f(uint32_t a, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ void put_u(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t get_u(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void put_l(uint32_t a, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ unsigned long long get_l(uint32_t a) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

// 16 bytes of logits in shared memory.
template <typename T>
struct Pack {
    static constexpr int kWidth = 16 / int(sizeof(T));
    uint4 q;
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 2) {
            const uint32_t u = reinterpret_cast<const uint32_t*>(&q)[e >> 1];
            return __uint_as_float(e & 1 ? u & 0xFFFF0000u : u << 16);
        } else {
            return reinterpret_cast<const float*>(&q)[e];
        }
    }
    // NaN becomes -inf.
    __device__ __forceinline__ void clean() {
        if constexpr (sizeof(T) == 2) {
            const __nv_bfloat162 low = __floats2bfloat162_rn(neg_inf(), neg_inf());
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                __nv_bfloat162& h = reinterpret_cast<__nv_bfloat162*>(&q)[e];
                h = __hmax2(h, low);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float& f = reinterpret_cast<float*>(&q)[e];
                f = fmaxf(f, neg_inf());
            }
        }
    }
    __device__ __forceinline__ void drop(int e) {
        if constexpr (sizeof(T) == 2) reinterpret_cast<uint16_t*>(&q)[e] = 0xFF80u;
        else reinterpret_cast<uint32_t*>(&q)[e] = 0xFF800000u;
    }
};

template <typename T, bool kResident, int kThreads>
struct Slice {
    using P = Pack<T>;
    enum : int { W = P::kWidth };
    const T* src;            // the slice's first logit
    const uint8_t* legal;    // its legality, or null
    int n;                   // logits in the slice
    int shift;               // src's place in its 16 bytes: logit i is element shift + i of `mem`
    P* mem;                  // resident: the slice, -inf around and where nothing may be chosen
    bool infinite = false;   // the row's maximum is +inf: its infinite logits stand as 0, the rest as -inf

    __device__ __forceinline__ float direct(int i) const {
        float l = float(src[i]);
        if (l != l || (legal && !legal[i])) l = neg_inf();
        if (infinite) l = l == __uint_as_float(0x7F800000u) ? 0.0f : neg_inf();
        return l;
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (kResident) return float(reinterpret_cast<const T*>(mem)[shift + i]);
        else return direct(i);
    }
    __device__ __forceinline__ int packs() const { return (shift + n + W - 1) / W; }

    // Brings the slice in; f(l) for this thread's logits.
    template <class F>
    __device__ __forceinline__ void load(F f) {
        if constexpr (kResident) {
            if (legal) load_as<true>(f);
            else load_as<false>(f);
        } else {
            for (int i = int(threadIdx.x); i < n; i += kThreads) f(direct(i));
        }
    }
    template <bool kLegal, class F>
    __device__ __forceinline__ void load_as(F f) {
        const uint4* base = reinterpret_cast<const uint4*>(src - shift);
        const int np = packs();
        // Packs under way at once, and the words that hold a pack's legality
        // (a byte each, at any place: one more word than their number).
        constexpr int kAhead = kLegal ? 4 : 8, kFours = W / 4;
        const int off = kLegal ? int(reinterpret_cast<uintptr_t>(legal - shift) & 3) : 0;
        for (int v0 = int(threadIdx.x); v0 < np; v0 += kThreads * kAhead) {
            P p[kAhead];
            uint32_t open[kAhead][kFours + 1];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int v = v0 + u * kThreads, i = v * W - shift;
                if (v < np && i >= 0 && i + W <= n) p[u].q = __ldg(base + v);
                if (kLegal && v < np && i >= off && i - off + W + 4 <= n) {
                    const uint32_t* words = reinterpret_cast<const uint32_t*>(legal + i - off);
#pragma unroll
                    for (int w = 0; w <= kFours; ++w) open[u][w] = __ldg(words + w);
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int v = v0 + u * kThreads, i = v * W - shift;
                if (v >= np) continue;
                if (i < 0 || i + W > n) {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        p[u].drop(e);
                        if (i + e >= 0 && i + e < n) reinterpret_cast<T*>(&p[u].q)[e] = src[i + e];
                    }
                }
                p[u].clean();
                if (kLegal && i >= off && i - off + W + 4 <= n) {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const uint32_t four = __funnelshift_r(open[u][e / 4], open[u][e / 4 + 1], 8 * off);
                        if (!(four >> (8 * (e & 3)) & 0xFFu)) p[u].drop(e);
                    }
                } else if (kLegal) {
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        if (i + e >= 0 && i + e < n && !legal[i + e]) p[u].drop(e);
                }
                mem[v] = p[u];
#pragma unroll
                for (int e = 0; e < W; ++e) f(p[u].get(e));
            }
        }
    }
    // f(l, i) for this thread's logits (and some of -inf around the slice).
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (kResident) {
            const int np = packs();
            for (int v = int(threadIdx.x); v < np; v += kThreads) {
                const P p = mem[v];
#pragma unroll
                for (int e = 0; e < W; ++e) f(p.get(e), v * W - shift + e);
            }
        } else {
            for (int i = int(threadIdx.x); i < n; i += kThreads) f(direct(i), i);
        }
    }
    // f(l, i) for this thread's logits of at least l_min, a few of many: they
    // are marked 32 at a time, so that a warp runs f as often as its busiest
    // lane has marks, and not for every place where any lane has one.
    template <class F>
    __device__ __forceinline__ void each_above(float l_min, F f) const {
        if constexpr (kResident) {
            constexpr int kPacks = 32 / P::kWidth;
            const int np = packs();
            for (int v0 = int(threadIdx.x); v0 < np; v0 += kThreads * kPacks) {
                uint32_t marks = 0;
#pragma unroll
                for (int g = 0; g < kPacks; ++g) {
                    const int v = v0 + g * kThreads;
                    if (v >= np) break;
                    const P p = mem[v];
#pragma unroll
                    for (int e = 0; e < P::kWidth; ++e) marks |= p.get(e) >= l_min ? 1u << (g * P::kWidth + e) : 0u;
                }
                while (marks) {
                    const int b = __ffs(int(marks)) - 1;
                    marks &= marks - 1;
                    const int i = (v0 + b / P::kWidth * kThreads) * P::kWidth - shift + b % P::kWidth;
                    f(at(i), i);
                }
            }
        } else {
            for (int i = int(threadIdx.x); i < n; i += kThreads) {
                const float l = direct(i);
                if (l >= l_min) f(l, i);
            }
        }
    }
    // The columns of each_above, in its order, into this warp's part of
    // `upper`; returns their number, or -1 where they do not fit.
    __device__ __forceinline__ int list_above(float l_min, uint16_t* part) const {
        constexpr int kPart = kUpper / (kThreads / 32);
        const int lane = int(threadIdx.x) & 31, first = int(threadIdx.x) & ~31;
        int filled = 0;
        if (n > 65536) return -1;
        const auto put = [&](uint32_t marks, auto column) {   // a warp together
            const int mine = __popc(marks);
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int d = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= o) upto += d;
            }
            const int total = __shfl_sync(0xFFFFFFFFu, upto, 31);
            if (filled + total <= kPart) {
                for (int to = filled + upto - mine; marks; marks &= marks - 1) part[to++] = uint16_t(column(__ffs(int(marks)) - 1));
            }
            filled += total;
        };
        if constexpr (kResident) {
            constexpr int kPacks = 32 / P::kWidth;
            const int np = packs();
            for (int w0 = first; w0 < np && filled <= kPart; w0 += kThreads * kPacks) {
                const int v0 = w0 + lane;
                uint32_t marks = 0;
#pragma unroll
                for (int g = 0; g < kPacks; ++g) {
                    const int v = v0 + g * kThreads;
                    if (v >= np) break;
                    const P p = mem[v];
#pragma unroll
                    for (int e = 0; e < P::kWidth; ++e) marks |= p.get(e) >= l_min ? 1u << (g * P::kWidth + e) : 0u;
                }
                put(marks, [&](int b) { return (v0 + b / P::kWidth * kThreads) * P::kWidth - shift + b % P::kWidth; });
            }
        } else {
            for (int w0 = first; w0 < n && filled <= kPart; w0 += kThreads * 32) {
                uint32_t marks = 0;
                for (int g = 0; g < 32; ++g) {
                    const int i = w0 + lane + g * kThreads;
                    if (i < n && direct(i) >= l_min) marks |= 1u << g;
                }
                put(marks, [&](int b) { return w0 + lane + b * kThreads; });
            }
        }
        __syncwarp();
        return filled <= kPart ? filled : -1;
    }
    // The row's maximum is +inf (every CTA of the cluster learns it at once).
    __device__ void only_infinite() {
        infinite = true;
        if constexpr (kResident) {
            for (int v = int(threadIdx.x); v < packs(); v += kThreads) {
                P p = mem[v];
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    if (p.get(e) != __uint_as_float(0x7F800000u)) p.drop(e);
                    else reinterpret_cast<T*>(&p.q)[e] = T(0.0f);
                }
                mem[v] = p;
            }
        }
    }
};

// Count and mass over the team, in a fixed order; the same everywhere.
// `turn` alternates between two sets of slots: a CTA writes a set again only
// after a barrier that every CTA reaches past its reads of it.
template <class Team>
__device__ __forceinline__ Weighed team_add(const Team& team, Weighed v, RowShared& sh, int& turn) {
    constexpr int kWarps = Team::kWarps;
    const int rank = team.rank, ranks = team.ranks;
    const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31;
    v.count = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(v.count)));
    v.mass = warp_sum(v.mass);
    __syncthreads();
    if (lane == 0) {
        sh.wf[warp] = v.mass;
        sh.wn[warp] = v.count;
    }
    __syncthreads();
    if (warp == 0) {
        Weighed s{lane < kWarps ? sh.wn[lane] : 0, lane < kWarps ? sh.wf[lane] : 0.0f};
        s.count = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(s.count)));
        s.mass = warp_sum(s.mass);
        if (lane < ranks) {
            put_f(team.at(&sh.f[turn][rank], lane), s.mass);
            put_u(team.at(&sh.n[turn][rank], lane), uint32_t(s.count));
        }
    }
    team.barrier();
    Weighed s{0, 0.0f};
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
        if (r < ranks) {
            s.count += sh.n[turn][r];
            s.mass += sh.f[turn][r];
        }
    turn ^= 1;
    return s;
}

struct Inclusive {
    uint32_t n, w;
};
// The team's histogram at this thread's bins, kPer neighbours: a bin's sums
// (in a cluster, from the CTA that added them up) and those up to it.
template <class Team>
struct Sums {
    static constexpr int kPer = kBins / Team::kThreads;
    uint32_t own_n[kPer], n[kPer], w[kPer];
    __device__ __forceinline__ void scan(const Team& team, RowShared& sh) {
        const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31, b0 = int(threadIdx.x) * kPer;
        uint32_t sn = 0, sw = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if constexpr (Team::kSolo) {
                own_n[j] = sh.hist_n[b0 + j];
                w[j] = sh.hist_w[b0 + j];
            } else {
                const int share = kBins / team.ranks, r = (b0 + j) / share, q = (b0 + j) % share;
                own_n[j] = get_u(team.at(&sh.share_n[q], r));
                w[j] = get_u(team.at(&sh.share_w[q], r));
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            n[j] = sn += own_n[j];
            w[j] = sw += w[j];
        }
        const uint32_t mine_n = sn, mine_w = sw;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t un = __shfl_up_sync(0xFFFFFFFFu, sn, o), uw = __shfl_up_sync(0xFFFFFFFFu, sw, o);
            if (lane >= o) sn += un, sw += uw;
        }
        if (lane == 31) sh.wn[warp] = int(sn), sh.wm[warp] = int(sw);
        __syncthreads();   // (the lists may take the histogram's place after this)
        sn -= mine_n;
        sw -= mine_w;
        for (int v = 0; v < warp; ++v) sn += uint32_t(sh.wn[v]), sw += uint32_t(sh.wm[v]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            n[j] += sn;
            w[j] += sw;
        }
    }
};

template <typename T, bool kResident, int kThreads, bool kSolo>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 6 : 3)
    sample_row_kernel(const SampleArgs a, const int ranks, const int per) {
    using Crew = Team<kThreads, kSolo>;
    constexpr int kWarps = Crew::kWarps;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ RowShared sh;
    const int rank = kSolo ? 0 : int(blockIdx.x) % ranks, t = int(threadIdx.x), warp = t >> 5, lane = t & 31;
    const long long row = kSolo ? blockIdx.x : blockIdx.x / unsigned(ranks);
    const Crew crew{rank, ranks};
    if constexpr (!kSolo) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs: its memory may be written
    grid_dependency_wait();
    grid_launch_dependents();
    const RowParams rp(a, row);
    Slice<T, kResident, kThreads> sl;
    const int i0 = min(rank * per, a.cols);
    sl.src = static_cast<const T*>(a.logits) + size_t(row) * size_t(a.ld) + i0;
    sl.legal = a.legal ? a.legal + size_t(row) * size_t(a.legal_ld) + i0 : nullptr;
    sl.n = min(per, a.cols - i0);
    sl.shift = int(reinterpret_cast<uintptr_t>(sl.src) % 16 / sizeof(T));
    sl.mem = reinterpret_cast<Pack<T>*>(smem_raw);
    const float inf = __uint_as_float(0x7F800000u);

    // The slice's largest logit, and the sum of w relative to it.
    float mine = neg_inf();
    sl.load([&](float l) { mine = fmaxf(mine, l); });
    float of_group = mine;
    if (rp.first_k() > 0) {
#pragma unroll
        for (int g = 0; g < kGroupSizes; ++g) {
            if (g) of_group = fmaxf(of_group, __shfl_xor_sync(0xFFFFFFFFu, of_group, 1 << (g ? g - 1 : 0)));
            const bool some = of_group > neg_inf();
            const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, some ? key_of(of_group) : 0xFF800000u);
            const int groups = __popc(__ballot_sync(0xFFFFFFFFu, some)) >> g;
            if (lane == 0) sh.low[g][warp] = logit_of_key(low), sh.groups[g][warp] = groups;
        }
    } else {
        of_group = warp_max(of_group);
    }
    if (lane == 0) sh.wf[warp] = of_group;
    __syncthreads();
    float m = neg_inf();
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sh.wf[w]);
    const bool greedy = rp.greedy();
    const float c = greedy ? 1.0f : log2_scale(rp.temperature);
    {
        Weighed s{0, 0.0f};
        if (!greedy && m > neg_inf()) {
            if (m == inf) sl.each([&](float l, int) { s.mass += l == inf ? 1.0f : 0.0f; });
            else if (rp.first_k() > 0)
                sl.each([&](float l, int) {
                    s.mass += ex2((l - m) * c);
                    s.count += l > neg_inf();
                });
            else sl.each([&](float l, int) { s.mass += ex2((l - m) * c); });
        }
        s.mass = warp_sum(s.mass);
        s.count = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(s.count)));
        if (lane == 0) sh.wh[warp] = s.mass, sh.wk[warp] = s.count;
    }
    __syncwarp();
    if constexpr (!kSolo) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every CTA runs
    __syncthreads();
    Part all;   // (every warp, from its own reads; the sums' order is fixed)
    all.top = m;
    all.z = warp_sum(lane < kWarps ? sh.wh[lane] : 0.0f);
    all.valid = int(__reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? unsigned(sh.wk[lane]) : 0u));
    if (rp.first_k() > 0) {
#pragma unroll
        for (int g = 0; g < kGroupSizes; ++g) {
            all.low[g] = logit_of_key(__reduce_min_sync(0xFFFFFFFFu, lane < kWarps ? key_of(sh.low[g][lane]) : 0xFF800000u));
            all.groups[g] = int(__reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? unsigned(sh.groups[g][lane]) : 0u));
        }
    }
    if constexpr (!kSolo) {   // and of the cluster: lane r takes CTA r's
        if (warp == 0 && lane < ranks) {
            const uint32_t to = crew.at(&sh.part[rank], lane);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(&all);
#pragma unroll
            for (int i = 0; i < int(sizeof(Part) / 4); ++i)
                if (i < 3 || rp.first_k() > 0) put_u(to + uint32_t(i) * 4, words[i]);
            if (rp.first_k() > 0) {
                const uint32_t tops = crew.at(&sh.warp_top[rank][0], lane);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) put_f(tops + uint32_t(w) * 4, sh.wf[w]);
            }
        }
        crew.barrier();
        const Part& p = sh.part[lane < ranks ? lane : 0];
        const bool in = lane < ranks;
        all.top = warp_max(p.top);
        all.z = warp_sum(!in ? 0.0f : p.top == all.top ? p.z : p.z * ex2((p.top - all.top) * c));
        all.valid = int(__reduce_add_sync(0xFFFFFFFFu, in ? unsigned(p.valid) : 0u));
        if (rp.first_k() > 0) {
#pragma unroll
            for (int g = 0; g < kGroupSizes; ++g) {
                all.low[g] = logit_of_key(__reduce_min_sync(0xFFFFFFFFu, key_of(p.low[g])));
                all.groups[g] = int(__reduce_add_sync(0xFFFFFFFFu, in ? unsigned(p.groups[g]) : 0u));
            }
        }
    }
    // The k-th largest of the warps' largest, if k of them hold a logit: a
    // bound of the k-th largest logit, above which about as many lie (50 of 64
    // warps over 50001 columns: 100).
    float kth = neg_inf();
    static_assert(kSolo || (kWarps == kMaxRowWarps && kThreads == 4 * kMaxCluster * kMaxRowWarps), "four threads for each warp of a cluster");
    if (!kSolo && rp.first_k() > 0 && rp.first_k() <= ranks * kWarps) {
        // Four threads count what is above one of them.
        const int tops = ranks * kWarps, v = t >> 2;
        const float* const every = &sh.warp_top[0][0];
        const float mine = v < tops ? every[v] : neg_inf();
        int above = 0;
        for (int j = t & 3; j < tops / 4; j += 4) {
            const float4 f = reinterpret_cast<const float4*>(every)[j];
            above += (f.x > mine) + (f.y > mine) + (f.z > mine) + (f.w > mine);
        }
        above += __shfl_xor_sync(0xFFFFFFFFu, above, 1);
        above += __shfl_xor_sync(0xFFFFFFFFu, above, 2);
        const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, v < tops && above < rp.first_k() ? key_of(mine) : 0xFFFFFFFFu);
        if (lane == 0) sh.wk[warp] = int(low);
        __syncthreads();
        kth = logit_of_key(__reduce_min_sync(0xFFFFFFFFu, lane < kWarps ? uint32_t(sh.wk[lane]) : 0xFFFFFFFFu));
    }
    m = all.top;
    int turn = 0;
    uint64_t best = 0;       // key of the race and the column, as one number: the largest wins
    float best_x = 0.0f;
    const auto run_race = [&](float l, int i, float u) {
        const float x = (l - m) * c * kLn2;
        const uint64_t r = place_of(key_of(race(x, u)), i);
        if (r > best) best = r, best_x = x;
    };

    if (m == neg_inf()) {
        // nothing to choose from
    } else if (greedy) {
        sl.each([&](float l, int i) {
            if (l == m && place_of(1u, i0 + i) > best) best = place_of(1u, i0 + i);
        });
    } else {
        if (m == inf) {
            sl.only_infinite();
            m = 0.0f;
            all.valid = int(all.z);
#pragma unroll
            for (int g = 0; g < kGroupSizes; ++g) all.low[g] = 0.0f;
            kth = neg_inf();
        }
        const float* noise = a.noise + size_t(row) * size_t(a.noise_ld) + i0;
        const int k = rp.first_k();
        const bool by_k = k > 0 && k < all.valid, by_p = rp.filters_p() && rp.top_p > 0.0f && k != 1;
        uint64_t cut = place_of(kKeyLow, 0x7FFFFFFF);   // the last place kept
        bool raced = false;
        // A warp's race of kN columns a lane, those with a bit in `in`. With
        // d = 1 - u, u clamped as the key's is: d <= -log u <= d / u, so that in
        // log2 a column's key lies between reach and reach + lg2(u). The two
        // logarithms (accurate, where the bounds' are approximate: the margins)
        // are taken only where the upper bound reaches the warp's best so far,
        // at first its best lower bound. ok(l, i): whether a column is in the
        // race after all.
        float lead = neg_inf();
        const auto race_some = [&](auto n, const float* l, const float* u, uint32_t in, auto column, auto ok) {
            constexpr int kN = decltype(n)::value;
            const auto reach = [&](int g) { return (l[g] - m) * c - lg2(1.0f - clamped(u[g])); };
            if (lead == neg_inf()) {
                float least = neg_inf();
#pragma unroll
                for (int g = 0; g < (kN < 4 ? kN : 4); ++g)   // (of a few: it is asked of columns that may yet drop out)
                    if ((in >> g & 1u) && ok(l[g], column(g))) least = fmaxf(least, reach(g) + lg2(clamped(u[g])));
                lead = logit_of_key(__reduce_max_sync(0xFFFFFFFFu, key_of(least))) - 2e-3f;
            }
            uint32_t marks = 0;
#pragma unroll
            for (int g = 0; g < kN; ++g) marks |= reach(g) >= lead ? 1u << g : 0u;
            for (marks &= in; marks; marks &= marks - 1) {
                const int b = __ffs(int(marks)) - 1;
                float lb = l[0], ub = u[0];
#pragma unroll
                for (int g = 1; g < kN; ++g)
                    if (g == b) lb = l[g], ub = u[g];
                if (ok(lb, column(b))) run_race(lb, i0 + column(b), ub);
            }
            __syncwarp();
            const uint32_t k = __reduce_max_sync(0xFFFFFFFFu, uint32_t(best >> 32));
            if (k) lead = fmaxf(lead, logit_of_key(k) * kLog2e - 1e-3f);
        };
        const auto passes_min_p = [&](float l) { return l == m || !(rp.min_p > 0.0f) || ex2((l - m) * c) >= rp.min_p; };
        // A little below the logit of log2 w = y (and never -inf, which stands
        // around the slice).
        const auto logit_below = [&](float y) { return fmaxf(m + y / c * 1.00001f - fabsf(m) * 1e-6f, -3.40282347e38f); };
        // This warp's upper columns, while they fit (upper_n is not negative).
        uint16_t* const part = sh.upper + warp * (kUpper / kWarps);
        int upper_n = -1;
        // f(l, i) for this thread's share of the logits of at least l_min.
        const auto each_upper = [&](float l_min, auto f) {
            if (upper_n < 0) {
                sl.each_above(l_min, f);
            } else {
                for (int j = lane; j < upper_n; j += 32) {
                    const int i = part[j];
                    f(sl.at(i), i);
                }
            }
        };
        if (by_k || by_p) {
            float listed = inf;   // every logit of at least this is among the upper ones
            const auto at = [&](uint32_t key) {
                Weighed s{0, 0.0f};
                const auto add = [&](float l, int) {
                    if (key_of(l) >= key) {
                        ++s.count;
                        s.mass += ex2((l - m) * c);
                    }
                };
                if (key >= key_of(listed)) each_upper(listed, add);
                else sl.each(add);
                return team_add(crew, s, sh, turn);
            };
            // What the histogram covers: log2 w from `low` to 0. Any range that
            // holds the cut will do. The bound for top-p takes every logit below
            // to weigh as much as it may, so an eighth of the weight is tried
            // first; should the cut lie below, the bound itself is taken.
            float low, sure;
            if (by_k) {
                float l = neg_inf();
#pragma unroll
                for (int g = 0; g < kGroupSizes; ++g)
                    if (k <= all.groups[g]) l = all.low[g];
                l = fmaxf(l, kth);
                sure = low = fmaxf((l - m) * c, -40.0f);
            } else {
                sure = fmaxf(__log2f((1.0f - rp.top_p) * 0.99f * all.z / float(a.cols)), -40.0f);
                low = sure < -6.0f ? sure + 3.0f : sure;
            }
            const float fixed = 2147483648.0f / all.z;   // all masses together stay below 2^31 + cols / 2
            float steps;                                 // bins per unit of log2 w; the last bin holds `low`
            const auto bin_of = [&](float y) { return int(-y * steps); };
            Sums<Crew> upto;
            const auto count_bins = [&] {
                low = fminf(low, -1e-3f);
                steps = float(kBins - 1) / -low;
                for (int b = t; b < kBins; b += kThreads) sh.hist_n[b] = sh.hist_w[b] = 0;
                if (t == 0) sh.first = sh.last = kBins, sh.list_n = 0;
                listed = logit_below(low);
                upper_n = sl.list_above(listed, part);
                __syncthreads();
                each_upper(listed, [&](float l, int) {
                    const float y = (l - m) * c;
                    if (y >= low) {
                        const int b = bin_of(y);
                        atomicAdd(&sh.hist_n[b], 1u);
                        atomicAdd(&sh.hist_w[b], __float2uint_rn(ex2(y) * fixed));
                    }
                });
                crew.barrier();
                if constexpr (!kSolo) {   // this CTA adds its share of the bins over the cluster
                    const int share = kBins / ranks;
                    for (int q = t; q < share; q += kThreads) {
                        uint32_t n[kMaxCluster], w[kMaxCluster];
#pragma unroll
                        for (int r = 0; r < kMaxCluster; ++r)
                            if (r < ranks) {
                                n[r] = get_u(crew.at(&sh.hist_n[rank * share + q], r));
                                w[r] = get_u(crew.at(&sh.hist_w[rank * share + q], r));
                            }
#pragma unroll
                        for (int r = 1; r < kMaxCluster; ++r)
                            if (r < ranks) n[0] += n[r], w[0] += w[r];
                        sh.share_n[q] = n[0];
                        sh.share_w[q] = w[0];
                    }
                    crew.barrier();
                }
                upto.scan(crew, sh);
            };
            uint64_t* list = reinterpret_cast<uint64_t*>(sh.hist_n);
            uint64_t* merged = list + kList;
            // One filter's cut: the first `count` logits, or the shortest prefix
            // of mass `target`. False: the histogram does not settle it. kept:
            // the mass that the cut is taken from. `final`: the last filter, so
            // that what lies above its cut is raced on the way. (sh.first,
            // sh.last and sh.list_n are at their starts before it.)
            // direct: without a histogram, the logits of at least kth are the list.
            const auto settle = [&](int count, float target, bool final, float* kept, bool direct) -> bool {
                int first = 0, last = kBins;
                bool whole = true;
                if (!direct) {
#pragma unroll
                    for (int j = 0; j < Sums<Crew>::kPer; ++j) {
                        const int b = t * Sums<Crew>::kPer + j;
                        if (count > 0) {
                            if (upto.n[j] >= uint32_t(count) && upto.n[j] - upto.own_n[j] < uint32_t(count)) sh.first = sh.last = b;
                        } else {
                            // A fixed-point sum is off by half a unit a logit, and by
                            // the masses' own rounding, a few 2^-22 of it.
                            const float goal = target * fixed, slack = 0.5f * float(upto.n[j]) + 4096.0f, w = float(upto.w[j]);
                            if (w + slack >= goal) atomicMin(&sh.first, b);
                            if (w - slack >= goal) atomicMin(&sh.last, b);
                        }
                    }
                    __syncthreads();
                    first = sh.first;
                    last = sh.last;
                    if (last >= kBins) return false;
#pragma unroll
                    for (int j = 0; j < Sums<Crew>::kPer; ++j) {
                        const int b = t * Sums<Crew>::kPer + j;
                        if (b == last) sh.down = upto.n[j];
                        if (b == first) sh.above = upto.n[j] - upto.own_n[j];
                    }
                    __syncthreads();
                    // Few enough down to the cut: all of them are listed, and raced there.
                    whole = sh.down <= uint32_t(kList);
                    if (!whole && sh.down - sh.above > uint32_t(kList)) return false;
                    if (whole) first = 0;
                }
                Weighed s{0, 0.0f};
                // A column's bin against the cut's: above it is kept for certain
                // (and raced if no filter follows).
                const auto place_in = [&](float l, int i) -> bool {
                    if (direct) {
                        const unsigned to = atomicAdd(&sh.list_n, 1u);
                        if (to < unsigned(kList)) list[to] = place_of(key_of(l), i0 + i);
                        return false;
                    }
                    const float y = (l - m) * c;
                    if (!(y >= low)) return false;
                    const int b = bin_of(y);
                    if (b < first) {
                        ++s.count;
                        s.mass += ex2(y);
                        return final && passes_min_p(l);
                    }
                    if (b <= last) list[atomicAdd(&sh.list_n, 1u)] = place_of(key_of(l), i0 + i);
                    return false;
                };
                if (upper_n < 0) {
                    sl.each_above(direct ? kth : logit_below(fmaxf(low, -float(last + 2) / steps)), [&](float l, int i) {
                        if (place_in(l, i)) run_race(l, i0 + i, __ldg(noise + i));
                    });
                } else {
                    constexpr int kAhead = 4;   // numbers asked for before the first is used
                    for (int b0 = 0; b0 < upper_n; b0 += 32 * kAhead) {
                        const int j0 = b0 + lane;
                        int i[kAhead];
                        float l[kAhead], u[kAhead];
                        uint32_t in = 0;
#pragma unroll
                        for (int g = 0; g < kAhead; ++g) {
                            i[g] = 0, l[g] = neg_inf(), u[g] = 0.0f;
                            if (j0 + 32 * g >= upper_n) continue;
                            i[g] = part[j0 + 32 * g];
                            l[g] = sl.at(i[g]);
                            if (place_in(l[g], i[g])) {
                                in |= 1u << g;
                                u[g] = __ldg(noise + i[g]);
                            }
                        }
                        if (final)
                            race_some(std::integral_constant<int, kAhead>(), l, u, in, [&](int b) { return int(part[j0 + 32 * b]); },
                                      [](float, int) { return true; });
                    }
                }
                s = team_add(crew, s, sh, turn);   // (also: every list is written)
                // All lists here, then in order.
                constexpr int kSlots = kList / kThreads;
                int n = 0;
                uint64_t place[kSlots] = {};
                int of_rank[kMaxCluster];
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r)
                    if (r < ranks) of_rank[r] = int(get_u(crew.at(&sh.list_n, r)));
                if (direct) {
                    int all_lists = 0;
#pragma unroll
                    for (int r = 0; r < kMaxCluster; ++r)
                        if (r < ranks) all_lists += min(of_rank[r], kList + 1);
                    if (all_lists > kList) return false;
                }
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r)
                    if (r < ranks) {
#pragma unroll
                        for (int j = 0; j < kSlots; ++j) {
                            const int at = t + j * kThreads - n;
                            if (at >= 0 && at < of_rank[r]) place[j] = get_l(crew.at(&list[at], r));
                        }
                        n += of_rank[r];
                    }
#pragma unroll
                for (int j = 0; j < kSlots; ++j)
                    if (t + j * kThreads < n) merged[t + j * kThreads] = place[j];
                __syncthreads();
                int before[kSlots] = {};
                if (t < n) {
                    const ulonglong2* two = reinterpret_cast<const ulonglong2*>(merged);
#pragma unroll 4
                    for (int q = 0; q < n; q += 2) {
                        const ulonglong2 other = two[q >> 1];
#pragma unroll
                        for (int j = 0; j < kSlots; ++j) before[j] += (other.x > place[j]) + (other.y > place[j] && q + 1 < n);
                    }
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < kSlots; ++j)
                    if (t + j * kThreads < n) merged[before[j]] = place[j];
                __syncthreads();
                // The sums run down the sorted list: the same for every CTA and
                // run. A lane takes `each` neighbours.
                const auto cut_list = [&](auto each_most) {
                    constexpr int kEach = decltype(each_most)::value;
                    const int each = (n + 31) / 32;
                    const int live = count > 0 ? min(n, count - s.count) : n;   // of the list, what top-k keeps
                    float w[kEach], sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const int q = lane * each + j;
                        w[j] = j < each && q < live ? ex2((logit_of_key(uint32_t(merged[q] >> 32)) - m) * c) : 0.0f;
                        sum += w[j];
                    }
                    float ahead = sum;   // up to and with this lane's
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const float d = __shfl_up_sync(0xFFFFFFFFu, ahead, o);
                        if (lane >= o) ahead += d;
                    }
                    const float total = s.mass + __shfl_sync(0xFFFFFFFFu, ahead, 31);
                    float ahead_of_me = __shfl_up_sync(0xFFFFFFFFu, ahead, 1);
                    ahead_of_me = s.mass + (lane ? ahead_of_me : 0.0f);
                    int stay = live;
                    if (count == 0 || (whole && by_p)) {
                        const float goal = count > 0 ? rp.top_p * total : target;
                        int here = 0;
#pragma unroll
                        for (int j = 0; j < kEach; ++j) {
                            here += j < each && lane * each + j < live && ahead_of_me < goal;
                            ahead_of_me += w[j];
                        }
                        stay = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(here)));
                    }
                    if (lane == 0) {
                        sh.cut = stay > 0 ? merged[stay - 1] : merged[0] + 1;
                        sh.kept = total;
                    }
                };
                if (warp == 0) {
                    if (n <= 64) cut_list(std::integral_constant<int, 2>());
                    else cut_list(std::integral_constant<int, kList / 32>());
                }
                __syncthreads();
                *kept = sh.kept;
                if (sh.cut > cut) cut = sh.cut;
                // Whole: rank 0 has them all in order. Else every CTA has its own.
                if (whole ? rank == 0 : final) {
                    const uint64_t* from = whole ? merged : list;
                    const int those = whole ? n : int(sh.list_n);
                    for (int j = t; j < those; j += kThreads) {
                        const uint64_t at = from[j];
                        const float l = logit_of_key(uint32_t(at >> 32));
                        const int i = int(~uint32_t(at)) - i0;
                        if (at >= cut && passes_min_p(l)) run_race(l, i0 + i, __ldg(noise + i));
                    }
                }
                raced = whole || final;
                return true;
            };
            float kept = all.z;
            bool settled = false, count_now = true, k_stage = by_k;
            if (!kSolo && by_k && kth > neg_inf()) {
                if (t == 0) sh.list_n = 0;
                upper_n = sl.list_above(kth, part);
                __syncthreads();
                settled = settle(k, 0.0f, true, &kept, true);
                if (!settled) crew.barrier();   // every CTA is past its reads of this one's count
            }
            while (!settled) {
                if (count_now) count_bins();
                count_now = false;
                settled = settle(k_stage ? k : 0, rp.top_p * kept, !k_stage || !by_p, &kept, false);
                if (!settled) {
                    if (k_stage || !(low > sure) || sh.last < kBins) break;
                    low = sure;   // the cut lies lower than was tried
                    count_now = true;
                } else {
                    if (!k_stage || !by_p || raced) break;
                    settled = k_stage = false;
                }
                crew.barrier();   // every CTA is past its reads of this one's lists
                if (t == 0) sh.first = sh.last = kBins, sh.list_n = 0;
                __syncthreads();
            }
            if (!settled) {
                const Weighed every = at(kKeyLow);
                const uint32_t hint = key_of(logit_below(sure));
                const Threshold th = find_threshold(rp, key_of(m), hint, hint, every.count, every.mass, at,
                                                    [&](uint32_t key) { return at(key).count; });
                int end = a.cols;   // the column after the threshold's last tie kept
                if (th.ties != kAllTies) {
                    int lo = 0;     // ties before lo < th.ties <= ties before end
                    while (end - lo > 1) {
                        const int mid = lo + (end - lo) / 2;
                        Weighed s{0, 0.0f};
                        const auto add = [&](float l, int i) { s.count += i0 + i < mid && key_of(l) == th.key; };
                        if (th.key >= key_of(listed)) each_upper(listed, add);
                        else sl.each(add);
                        if (team_add(crew, s, sh, turn).count >= th.ties) end = mid;
                        else lo = mid;
                    }
                }
                cut = place_of(th.key, end - 1);
            }
        }
        if (!raced) {
            const float cut_l = logit_of_key(uint32_t(cut >> 32));
            float low = kNoChance * kLog2e;
            if (rp.min_p > 0.0f) low = fmaxf(low, fminf(__log2f(rp.min_p) - 1e-3f, 0.0f));
            const auto stays = [&](float l, int i) {
                const float y = (l - m) * c;
                return y >= low && place_of(key_of(l), i0 + i) >= cut && passes_min_p(l);
            };
            // Where a filter leaves few columns they are listed first and raced
            // from the list.
            if (by_k || by_p || rp.min_p > 0.0f) {
                const float l_min = fmaxf(cut_l, logit_below(low));
                upper_n = sl.list_above(l_min, part);
                if (upper_n >= 0)
                    each_upper(l_min, [&](float l, int i) {
                        if (stays(l, i)) run_race(l, i0 + i, __ldg(noise + i));
                    });
            }
            if (upper_n < 0) {
                if constexpr (kResident) {
                    using P = Pack<T>;
                    constexpr int W = P::kWidth, kAhead = 16 / W, kN = kAhead * W;
                    const int np = sl.packs();
                    const bool wide = (reinterpret_cast<uintptr_t>(noise) - 4u * unsigned(sl.shift)) % 16 == 0;
                    for (int w0 = t & ~31; w0 < np; w0 += kThreads * kAhead) {   // a warp's lanes stay together
                        float l[kN], u[kN];
#pragma unroll
                        for (int g = 0; g < kAhead; ++g) {
                            const int v = w0 + lane + g * kThreads, i = v * W - sl.shift;
                            if (v < np && i >= 0 && i + W <= sl.n && wide) {
#pragma unroll
                                for (int e = 0; e < W; e += 4) {
                                    const float4 f = __ldg(reinterpret_cast<const float4*>(noise + i + e));
                                    u[g * W + e] = f.x, u[g * W + e + 1] = f.y, u[g * W + e + 2] = f.z, u[g * W + e + 3] = f.w;
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < W; ++e)
                                    u[g * W + e] = v < np && i + e >= 0 && i + e < sl.n ? __ldg(noise + i + e) : 0.0f;
                            }
                        }
                        uint32_t in = 0;
#pragma unroll
                        for (int g = 0; g < kAhead; ++g) {
                            const int v = w0 + lane + g * kThreads;
                            P p;
                            if (v < np) {
                                p = sl.mem[v];
                                in |= ((1u << W) - 1u) << (g * W);
                            }
#pragma unroll
                            for (int e = 0; e < W; ++e) l[g * W + e] = v < np ? p.get(e) : neg_inf();
                        }
                        const auto column = [&](int b) { return (w0 + lane + b / W * kThreads) * W - sl.shift + b % W; };
                        race_some(std::integral_constant<int, kN>(), l, u, in, column, stays);
                    }
                } else {
                    for (int w0 = t & ~31; w0 < sl.n; w0 += kThreads) {
                        const int i = w0 + lane;
                        const bool there = i < sl.n;
                        const float l = there ? sl.direct(i) : neg_inf(), u = there ? __ldg(noise + i) : 0.0f;
                        race_some(std::integral_constant<int, 1>(), &l, &u, there, [&](int) { return i; }, stays);
                    }
                }
            }
        }
    }

    // The cluster's winner.
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t b = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        const float x = __shfl_xor_sync(0xFFFFFFFFu, best_x, o);
        if (b > best) best = b, best_x = x;
    }
    __shared__ uint64_t warp_best[kWarps];
    if (lane == 0) warp_best[warp] = best, sh.wg[warp] = best_x;
    __syncthreads();
    if (t == 0) {
        for (int w = 0; w < kWarps; ++w)
            if (warp_best[w] > best) best = warp_best[w], best_x = sh.wg[w];
        put_l(crew.at(&sh.best[rank], 0), best);
        put_f(crew.at(&sh.best_x[rank], 0), best_x);
    }
    crew.barrier();
    if (rank == 0 && t == 0) {
        for (int r = 0; r < ranks; ++r)
            if (sh.best[r] > best) best = sh.best[r], best_x = sh.best_x[r];
        a.moves[row] = best ? (long long)uint32_t(~uint32_t(best)) : -1;
        if (a.logprob) a.logprob[row] = !best ? neg_inf() : greedy ? 0.0f : best_x - logf(all.z);
    }
}

template <typename T, bool kResident, int kThreads, bool kSolo>
cudaError_t launch_rows(const SampleArgs& a, int ranks, int per, size_t smem, cudaStream_t s) {
    constexpr auto kernel = sample_row_kernel<T, kResident, kThreads, kSolo>;
    if (const cudaError_t e = open_smem<kernel>(smem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {unsigned(ranks), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = kSolo ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kernel, a, ranks, per);
}

constexpr int kRowCtas = 384;   // that run at once: 48 clusters of eight

template <typename T>
cudaError_t launch_sample_t(const SampleArgs& a, cudaStream_t s) {
    const int grid = int((a.rows + 3) / 4);
    if (a.cols <= 1024) {
        if (a.cols <= 128) return launch_pdl(sample_warp_kernel<T, 4>, dim3(unsigned(grid)), dim3(128), 0, s, a);
        if (a.cols <= 384) return launch_pdl(sample_warp_kernel<T, 12>, dim3(unsigned(grid)), dim3(128), 0, s, a);
        return launch_pdl(sample_warp_kernel<T, 32>, dim3(unsigned(grid)), dim3(128), 0, s, a);
    }
    // Up to 16384 columns one CTA has the row (512 rows of 16384, top-p: 27 us,
    // with two of 8192 each 42 us); beyond, slices of at most 8192 while eight
    // CTAs can hold the row so (8 rows of 50001, top-p: 14 us, with 16384 16 us). Where
    // not all of those run at once, up to 65536 columns, a row has half as many
    // CTAs (512 rows of 50001: 174 us with eight, 101 us with four; 64 rows 30
    // and 19), and its sums another order.
    int ranks = a.cols <= 16384 ? 1 : a.cols <= 32768 ? 4 : kMaxCluster;
    if (ranks > 1 && a.cols <= 65536 && a.rows * ranks > kRowCtas) ranks /= 2;
    const int per = (a.cols + ranks - 1) / ranks;
    const size_t smem = size_t(per) * sizeof(T) + 32;   // up to 16 bytes of alignment at either end
    if (a.cols <= 8192) return launch_rows<T, true, 128, true>(a, 1, per, smem, s);
    if (ranks == 1) return launch_rows<T, true, 256, true>(a, 1, per, smem, s);
    return smem <= (size_t(200) << 10) ? launch_rows<T, true, 256, false>(a, ranks, per, smem, s)
                                       : launch_rows<T, false, 256, false>(a, ranks, per, 0, s);
}

}  // namespace

cudaError_t launch_sample_moves(const SampleArgs& a, cudaStream_t s) {
    return a.type == kElemBF16 ? launch_sample_t<__nv_bfloat16>(a, s) : launch_sample_t<float>(a, s);
}

}  // namespace azb
