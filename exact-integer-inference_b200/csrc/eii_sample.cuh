// Drawing tokens from integer logits (eii_sample).
//
// Weight of logit l in a row of maximum M, exponent 16, inverse temperature beta (Q16):
//   x = (M - l) b2, b2 = (beta 24204406 + 2^15) >> 16 (beta log2(e) in Q24), n = x >> 40, f = bits 16..39 of x,
//   w = RS(2^30 - f (C1 - f (C2 - f (C3 - f C4))), n) for n <= 30, else 0:
// 2^30 exp(-(M - l) / T) to 3.4e-6 of its value and half a unit.  The C are a minimax fit of 2^-f on [0, 1] (this
// project's own; exact at both ends), each product floored to Q30.  With 24 bits of f the steps of the
// polynomial outweigh its roundings, so w never rises with the distance: the order of the weights is
// the order of the logits.  Every sum of weights is exact in 64 bits, so the result does not depend on
// the order of the threads.
#pragma once
#include <cstdint>

#include "eii_int.cuh"

namespace eii {

constexpr uint32_t SAMPLE_C1 = 744163075, SAMPLE_C2 = 257059888, SAMPLE_C3 = 57045411, SAMPLE_C4 = 7277686;
constexpr int64_t SAMPLE_LOG2E_Q24 = 24204406;
constexpr int32_t SAMPLE_MASKED = INT32_MIN;
constexpr int SAMPLE_MAX_VOCAB = 262144;  // 2^30 x 2^18 weights: sums stay below 2^48
constexpr int32_t SAMPLE_MAX_INV_TEMP = 1 << 22;

enum : int { ERR_SAMPLE_PARAM = 311 };

struct SampleParams {
    const int32_t* logits;
    int64_t ld;
    int n_rows, vocab;
    const int32_t *inv_temp, *top_k, *top_p, *min_p;
    const uint32_t* u;
    int64_t* token;
    int32_t *kept, *prob;
    int* err;
};

// One row's parameters; ok is false when one lies outside its range.
struct SampleRow {
    uint32_t b2;
    int k, p, mp;
    bool ok;
};

__device__ __forceinline__ SampleRow sample_row(const SampleParams& p, int r) {
    SampleRow o;
    const int beta = p.inv_temp ? p.inv_temp[r] : 65536;
    o.k = p.top_k ? p.top_k[r] : 0;
    o.p = p.top_p ? p.top_p[r] : 65536;
    o.mp = p.min_p ? p.min_p[r] : 0;
    o.ok = beta >= 1 && beta <= SAMPLE_MAX_INV_TEMP && o.k >= 0 && o.p >= 0 && o.p <= 65536 && o.mp >= 0 && o.mp <= 65536;
    o.b2 = static_cast<uint32_t>((beta * SAMPLE_LOG2E_Q24 + (1 << 15)) >> 16);
    return o;
}

// floor(y f / 2^31) of the 31-bit fraction f is umulhi(y, 2 f).
__device__ __forceinline__ uint32_t sample_weight(int32_t l, int32_t row_max, uint32_t b2) {
    if (l == SAMPLE_MASKED) return 0;
    const uint64_t x = static_cast<uint64_t>(static_cast<uint32_t>(row_max) - static_cast<uint32_t>(l)) * b2;
    const uint32_t n = static_cast<uint32_t>(x >> 40);
    if (n > 30) return 0;
    const uint32_t f2 = static_cast<uint32_t>(x >> 8) & 0xFFFFFF00u;
    uint32_t y = SAMPLE_C3 - __umulhi(SAMPLE_C4, f2);
    y = SAMPLE_C2 - __umulhi(y, f2);
    y = SAMPLE_C1 - __umulhi(y, f2);
    y = (1u << 30) - __umulhi(y, f2);
    return (y + ((1u << n) >> 1)) >> n;
}

// ceil(p mass / 2^16), at least 1.
__device__ __forceinline__ uint64_t sample_goal(uint64_t mass, int p) {
    const uint64_t g = p * (mass >> 16) + ((p * (mass & 0xFFFF) + 0xFFFF) >> 16);
    return g ? g : 1;
}
// floor(u mass / 2^32).
__device__ __forceinline__ uint64_t sample_target(uint64_t mass, uint32_t u) {
    return (u * (mass >> 24) + ((u * (mass & 0xFFFFFF)) >> 24)) >> 8;
}

constexpr int SAMPLE_THREADS = 256;

__device__ __forceinline__ uint64_t block_sum(uint64_t v, unsigned long long* s) {
    __syncthreads();
    if (threadIdx.x == 0) *s = 0;
    __syncthreads();
    atomicAdd(s, static_cast<unsigned long long>(v));
    __syncthreads();
    return *s;
}

// One block per row.  The kept tokens are a prefix of the order (weight descending, index ascending):
// all weights above theta and the first `quota` of those equal to it.  Both cuts are found by bisection.
__global__ void __launch_bounds__(SAMPLE_THREADS) k_sample(const SampleParams p) {
    __shared__ unsigned long long sum_s;
    __shared__ int32_t max_s;
    __shared__ unsigned long long mass_t[SAMPLE_THREADS];
    __shared__ int ties_t[SAMPLE_THREADS];
    const int r = blockIdx.x, tid = threadIdx.x, V = p.vocab;
    const int32_t* row = p.logits + r * p.ld;
    const SampleRow q = sample_row(p, r);
    if (tid == 0) max_s = SAMPLE_MASKED;
    __syncthreads();
    int32_t mx = SAMPLE_MASKED;
    for (int i = tid; i < V; i += SAMPLE_THREADS) mx = max(mx, row[i]);
    atomicMax(&max_s, mx);
    __syncthreads();
    mx = max_s;
    if (!q.ok || mx == SAMPLE_MASKED) {
        if (tid == 0) {
            if (!q.ok) atomicCAS(p.err, 0, ERR_SAMPLE_PARAM);
            p.token[r] = -1;
            if (p.kept) p.kept[r] = 0;
            if (p.prob) p.prob[r] = 0;
        }
        return;
    }
    auto count_from = [&](uint32_t th) {
        uint64_t c = 0;
        for (int i = tid; i < V; i += SAMPLE_THREADS) c += sample_weight(row[i], mx, q.b2) >= th;
        return block_sum(c, &sum_s);
    };
    auto mass_from = [&](uint32_t th) {
        uint64_t c = 0;
        for (int i = tid; i < V; i += SAMPLE_THREADS) {
            const uint32_t w = sample_weight(row[i], mx, q.b2);
            c += w >= th ? w : 0;
        }
        return block_sum(c, &sum_s);
    };
    uint32_t theta = 1;
    uint64_t quota = UINT32_MAX;
    if (q.k > 0 && count_from(1) > q.k) {
        uint32_t lo = 1, hi = (1u << 30) + 1;  // count_from(lo) >= k > count_from(hi)
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (count_from(mid) >= q.k) lo = mid;
            else hi = mid;
        }
        theta = lo;
        quota = q.k - count_from(theta + 1);
    }
    if ((static_cast<uint32_t>(q.mp) << 14) > theta) {
        theta = static_cast<uint32_t>(q.mp) << 14;
        quota = UINT32_MAX;
    }
    uint64_t above = mass_from(theta + 1);
    uint64_t equal = count_from(theta) - count_from(theta + 1);
    if (quota > equal) quota = equal;
    if (q.p < 65536) {
        const uint64_t goal = sample_goal(above + quota * theta, q.p);
        if (above >= goal) {
            uint32_t lo = theta, hi = (1u << 30) + 1;  // mass_from(lo + 1) or its part >= goal > mass_from(hi)
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (mass_from(mid) >= goal) lo = mid;
                else hi = mid;
            }
            theta = lo;
            above = mass_from(theta + 1);
        }
        quota = (goal - above + theta - 1) / theta;
    }
    const uint64_t mass = above + quota * theta, target = sample_target(mass, p.u[r]);
    const uint64_t above_n = count_from(theta + 1);
    // index order: thread t owns a contiguous part
    const int part = (V + SAMPLE_THREADS - 1) / SAMPLE_THREADS, i0 = min(tid * part, V), i1 = min(i0 + part, V);
    uint64_t m = 0;
    int ties = 0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t w = sample_weight(row[i], mx, q.b2);
        m += w > theta ? w : 0;
        ties += w == theta;
    }
    mass_t[tid] = m;
    ties_t[tid] = ties;
    __syncthreads();
    uint64_t run = 0, tied = 0;
    for (int t = 0; t < tid; ++t) {
        const uint64_t take = tied >= quota ? 0 : min(static_cast<uint64_t>(ties_t[t]), quota - tied);
        run += mass_t[t] + take * theta;
        tied += ties_t[t];
    }
    const uint64_t take = tied >= quota ? 0 : min(static_cast<uint64_t>(ties), quota - tied);
    if (run <= target && target < run + m + take * theta) {
        for (int i = i0; i < i1; ++i) {
            const uint32_t w = sample_weight(row[i], mx, q.b2);
            const bool in = w > theta || (w == theta && tied < quota);
            tied += w == theta;
            run += in ? w : 0;
            if (in && run > target) {
                p.token[r] = i;
                if (p.kept) p.kept[r] = static_cast<int32_t>(above_n + quota);
                if (p.prob) p.prob[r] = static_cast<int32_t>(((static_cast<uint64_t>(w) << 30) + (mass >> 1)) / mass);
                break;
            }
        }
    }
}

}  // namespace eii
