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
// of equal ones) is left in the range. Counts are exact and sums run in a
// fixed order, so a row's move does not depend on the batch or the run.
#include <cuda_bf16.h>

#include <algorithm>

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

template <typename T>
__device__ __forceinline__ float logit_at(const SampleArgs& a, const T* row, const uint8_t* legal, int i) {
    float l = float(row[i]);
    if ((legal && !legal[i]) || l != l) l = neg_inf();
    return l;
}

__device__ __forceinline__ float scaled(float l, float m, float inv_t) {
    const float x = (l - m) * inv_t;
    return l == m ? 0.0f : x == x ? x : neg_inf();   // (an infinite m over an infinite T)
}

__device__ __forceinline__ float race(float x, float u) {
    // fmaxf reads a NaN as the lowest number.
    return x - logf(-logf(fminf(fmaxf(u, kULow), kUHigh)));
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

// The threshold of a row's filters. at(k): count and mass of the logits
// with key >= k, the same on every calling thread. top: the largest key.
template <class At>
__device__ Threshold find_threshold(const RowParams& rp, uint32_t top, int valid, float mass, At at) {
    Threshold th{kKeyLow, kAllTies};
    const int k = rp.filters_p() && !(rp.top_p > 0.0f) ? 1 : rp.top_k;
    float kept = mass;   // mass of what is kept so far
    if (k > 0 && k < valid) {
        uint32_t lo = kKeyLow, hi = top + 1;   // count(lo) >= k > count(hi)
        Weighed wlo{valid, mass}, whi{0, 0.0f};
        while (hi - lo > 1 && wlo.count != k) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const Weighed w = at(mid);
            if (w.count >= k) lo = mid, wlo = w;
            else hi = mid, whi = w;
        }
        th.key = lo;
        kept = wlo.mass;
        if (wlo.count != k) {   // ties at lo: the first k - count(hi) of them
            th.ties = k - whi.count;
            kept = whi.mass + (wlo.mass - whi.mass) * (float(th.ties) / float(wlo.count - whi.count));
        }
        if (k == 1) return th;
    }
    if (rp.filters_p()) {
        const double target = double(rp.top_p) * double(kept);
        uint32_t lo = th.key, hi = top + 1;   // mass(lo) >= target > mass(hi)
        Weighed wlo = at(lo), whi{0, 0.0f};
        while (hi - lo > 1 && wlo.count - whi.count > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const Weighed w = at(mid);
            if (double(w.mass) >= target) lo = mid, wlo = w;
            else hi = mid, whi = w;
        }
        const int group = wlo.count - whi.count;   // equal logits unless there is only one
        int ties = kAllTies;
        if (group > 1) {
            const double each = (double(wlo.mass) - double(whi.mass)) / group;
            const double need = each > 0.0 ? ceil((target - double(whi.mass)) / each) : double(group);
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
template <typename T, int kPer>
__global__ void __launch_bounds__(128) sample_warp_kernel(const SampleArgs a) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const int lane = threadIdx.x & 31;
    constexpr uint32_t kFull = 0xFFFFFFFFu;
    const RowParams rp(a, row);
    const T* logits = static_cast<const T*>(a.logits) + size_t(row) * size_t(a.ld);
    const uint8_t* legal = a.legal ? a.legal + size_t(row) * size_t(a.legal_ld) : nullptr;
    float l[kPer];
    float m = neg_inf();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * 32 + lane;
        l[j] = i < a.cols ? logit_at(a, logits, legal, i) : neg_inf();
        m = fmaxf(m, l[j]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
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
    const float inv_t = 1.0f / rp.temperature;
    uint32_t key[kPer];
    float x[kPer], w[kPer];
    float z = 0.0f;
    int valid = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        key[j] = key_of(l[j]);
        x[j] = scaled(l[j], m, inv_t);
        w[j] = key[j] >= kKeyLow ? expf(x[j]) : 0.0f;
        z += w[j];
        valid += key[j] >= kKeyLow;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(kFull, z, o);
    valid = int(__reduce_add_sync(kFull, unsigned(valid)));
    const Threshold th = find_threshold(rp, key_of(m), valid, z, [&](uint32_t at) {
        Weighed s{0, 0.0f};
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (key[j] >= at) {
                ++s.count;
                s.mass += w[j];
            }
        s.count = int(__reduce_add_sync(kFull, unsigned(s.count)));
#pragma unroll
        for (int o = 16; o; o >>= 1) s.mass += __shfl_xor_sync(kFull, s.mass, o);
        return s;
    });
    const float* noise = a.noise + size_t(row) * size_t(a.noise_ld);
    float best = neg_inf(), best_x = 0.0f;
    uint32_t best_i = 0xFFFFFFFFu;
    int seen = 0;   // logits equal to the threshold, in columns before
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * 32 + lane;
        bool keep = key[j] >= th.key && (w[j] >= rp.min_p || l[j] == m || !(rp.min_p > 0.0f));
        if (th.ties != kAllTies) {
            const uint32_t tied = __ballot_sync(kFull, key[j] == th.key);
            if (key[j] == th.key && seen + __popc(tied & ((1u << lane) - 1u)) >= th.ties) keep = false;
            seen += __popc(tied);
        }
        if (keep) {
            const float r = race(x[j], noise[i]);
            if (r > best) best = r, best_i = uint32_t(i), best_x = x[j];
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float r = __shfl_xor_sync(kFull, best, o);
        const uint32_t i = __shfl_xor_sync(kFull, best_i, o);
        const float bx = __shfl_xor_sync(kFull, best_x, o);
        if (r > best || (r == best && i < best_i)) best = r, best_i = i, best_x = bx;
    }
    if (lane == 0) {
        a.moves[row] = (long long)best_i;
        if (a.logprob) a.logprob[row] = best_x - logf(z);
    }
}

// -------------------------------------------------------- a block per row

constexpr int kWideThreads = 1024;

struct WideShared {
    float f[32];
    int n[32];
};

// Every thread's value reduced over the block, in a fixed order.
__device__ __forceinline__ float block_max(float v, WideShared& sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.f[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.f[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

__device__ __forceinline__ Weighed block_add(Weighed v, WideShared& sh) {
    v.count = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(v.count)));
#pragma unroll
    for (int o = 16; o; o >>= 1) v.mass += __shfl_xor_sync(0xFFFFFFFFu, v.mass, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        sh.f[threadIdx.x >> 5] = v.mass;
        sh.n[threadIdx.x >> 5] = v.count;
    }
    __syncthreads();
    v.count = int(__reduce_add_sync(0xFFFFFFFFu, unsigned(sh.n[threadIdx.x & 31])));
    v.mass = sh.f[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v.mass += __shfl_xor_sync(0xFFFFFFFFu, v.mass, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) sample_block_kernel(const SampleArgs a) {
    __shared__ WideShared sh;
    const long long row = blockIdx.x;
    const RowParams rp(a, row);
    const T* logits = static_cast<const T*>(a.logits) + size_t(row) * size_t(a.ld);
    const uint8_t* legal = a.legal ? a.legal + size_t(row) * size_t(a.legal_ld) : nullptr;
    const int t = int(threadIdx.x), step = kWideThreads;
    float m = neg_inf();
    for (int i = t; i < a.cols; i += step) m = fmaxf(m, logit_at(a, logits, legal, i));
    m = block_max(m, sh);
    if (m == neg_inf()) {
        if (t == 0) {
            a.moves[row] = -1;
            if (a.logprob) a.logprob[row] = neg_inf();
        }
        return;
    }
    const bool greedy = rp.greedy();
    const float inv_t = greedy ? 1.0f : 1.0f / rp.temperature;
    float z = 0.0f;
    Threshold th{key_of(m), kAllTies};
    int cut = 0x7FFFFFFF;   // columns from here on keep none of the threshold's ties
    if (!greedy) {
        auto at = [&](uint32_t key) {
            Weighed s{0, 0.0f};
            for (int i = t; i < a.cols; i += step) {
                const float l = logit_at(a, logits, legal, i);
                if (key_of(l) >= key) {
                    ++s.count;
                    s.mass += expf(scaled(l, m, inv_t));
                }
            }
            return block_add(s, sh);
        };
        const Weighed all = at(kKeyLow);
        z = all.mass;
        th = find_threshold(rp, key_of(m), all.count, all.mass, at);
        if (th.ties != kAllTies) {   // the column after the last tie kept
            int lo = 0, hi = a.cols;   // ties before lo < th.ties <= ties before hi
            while (hi - lo > 1) {
                const int mid = lo + (hi - lo) / 2;
                Weighed s{0, 0.0f};
                for (int i = t; i < mid; i += step) s.count += key_of(logit_at(a, logits, legal, i)) == th.key;
                if (block_add(s, sh).count >= th.ties) hi = mid;
                else lo = mid;
            }
            cut = hi;
        }
    }
    const float* noise = greedy ? nullptr : a.noise + size_t(row) * size_t(a.noise_ld);
    float best = neg_inf(), best_x = 0.0f;
    uint32_t best_i = 0xFFFFFFFFu;
    for (int i = t; i < a.cols; i += step) {
        const float l = logit_at(a, logits, legal, i);
        const uint32_t key = key_of(l);
        if (key < th.key || (key == th.key && i >= cut)) continue;
        const float x = scaled(l, m, inv_t);
        if (l != m && rp.min_p > 0.0f && !greedy && !(expf(x) >= rp.min_p)) continue;
        const float r = greedy ? 0.0f : race(x, noise[i]);
        if (r > best) best = r, best_i = uint32_t(i), best_x = x;
    }
    // The winner: the largest key's lowest index.
    __shared__ uint32_t first;
    __shared__ float first_x;
    const float top = block_max(best, sh);
    if (t == 0) first = 0xFFFFFFFFu;
    __syncthreads();
    if (best == top) atomicMin(&first, best_i);
    __syncthreads();
    if (best == top && best_i == first) first_x = best_x;
    __syncthreads();
    if (t == 0) {
        a.moves[row] = (long long)first;
        if (a.logprob) a.logprob[row] = greedy ? 0.0f : first_x - logf(z);
    }
}

template <typename T>
cudaError_t launch_sample_t(const SampleArgs& a, cudaStream_t s) {
    const int grid = int((a.rows + 3) / 4);
    if (a.cols <= 128) sample_warp_kernel<T, 4><<<grid, 128, 0, s>>>(a);
    else if (a.cols <= 384) sample_warp_kernel<T, 12><<<grid, 128, 0, s>>>(a);
    else if (a.cols <= 1024) sample_warp_kernel<T, 32><<<grid, 128, 0, s>>>(a);
    else sample_block_kernel<T><<<int(a.rows), kWideThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_sample_moves(const SampleArgs& a, int sms, cudaStream_t s) {
    (void)sms;
    return a.type == kElemBF16 ? launch_sample_t<__nv_bfloat16>(a, s) : launch_sample_t<float>(a, s);
}

}  // namespace azb
