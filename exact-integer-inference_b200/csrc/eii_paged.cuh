// Paged K/V cache: layout and kernels of eii_paged_append and eii_paged_attention.
//
// A pool holds n_pages pages; a page holds `page` consecutive positions of one sequence for every kv
// head, one slab per head:  pool[page][kv head][slab].  A slab of a 16-bit cache is int16
// [page][hd].  A slab of a 4-bit cache is uint8 [page][hd / 2] followed by uint32 [page][hd / 64]:
// every 64 dimensions of a row form a group of 32 bytes, byte j holding dimension j in its low nibble
// and dimension j + 32 in its high nibble, and one scale word m | (z & 0xffff) << 16 (m in [1, 4369]
// unsigned, z signed); nibble n stands for z + m n.  Page sizes are powers of two >= 16, so every
// slab, and the scale block in it, starts on a 16-byte boundary.
#pragma once
#include <cstdint>

#include "eii_int.cuh"
#include "eii_ptx.cuh"

namespace eii {

constexpr int PAGED_DMAX = 1536;  // exp table entries 0..1536 (a distance beyond it has weight zero)

enum : int {
    ERR_PAGED_SEQ = 301,    // sequence index >= n_seq
    ERR_PAGED_POS = 302,    // position outside the rope table or the page table's columns
    ERR_PAGED_PAGE = 303,   // page index outside [0, n_pages)
    ERR_PAGED_LEN = 304,    // visible length above max_len or the page table's columns
    ERR_PAGED_INPUT = 305,  // int32 input outside the int16 range
};

// What every kernel needs of the cache and of one call's pages.
struct PagedGeom {
    int n_heads, n_kv, hd, group;  // group = n_heads / n_kv
    int page_shift, bits;
    int64_t slab;                  // bytes of one page of one kv head
    uint8_t *k_pool, *v_pool;
    int64_t n_pages;
    const int32_t* table;
    int64_t ld_table;
    int n_seq;
    const int32_t* exp_tab;        // [PAGED_DMAX + 1], Q30
    int* err;
};

__device__ __forceinline__ int64_t slab_offset(const PagedGeom& g, int page_id, int head) {
    return (static_cast<int64_t>(page_id) * g.n_kv + head) * g.slab;
}

__host__ __device__ __forceinline__ int paged_row_bytes(int hd, int bits) {
    return bits == 16 ? hd * 2 : hd / 2 + hd / 16;
}

// ------------------------------------------------------------------------------------------ append
// o[d] = SAT16(RS(a[d] C - a[d + hd/2] S, shift)), o[d + hd/2] = SAT16(RS(a[d + hd/2] C + a[d] S, shift))
// with the Q30 row of the token's position; v rows keep their values.
struct AppendParams {
    PagedGeom g;
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;
    int n_rows;
    const int32_t *seq, *pos;
    const int32_t *rope_c, *rope_s;  // [n_pos][hd / 2]
    int n_pos;
    int shift_q, shift_k;
    int16_t* q_out;
    int64_t ldqo;
    int32_t* kv_out;
};

// Writes one lane's HD / 32 values of a cached row: x[i] is dimension lane + 32 i.
template <int HD, int BITS>
__device__ __forceinline__ void store_row(const PagedGeom& g, uint8_t* slab, int slot, int lane, int32_t (&x)[HD / 32]) {
    if constexpr (BITS == 16) {
        int16_t* row = reinterpret_cast<int16_t*>(slab) + slot * HD;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) row[lane + 32 * i] = static_cast<int16_t>(x[i]);
    } else {
        uint8_t* row = slab + slot * (HD / 2);
        uint32_t* scale = reinterpret_cast<uint32_t*>(slab + (HD / 2 << g.page_shift)) + slot * (HD / 64);
#pragma unroll
        for (int a = 0; a < HD / 64; ++a) {
            const int32_t lo = __reduce_min_sync(~0u, min(x[2 * a], x[2 * a + 1]));
            const int32_t hi = __reduce_max_sync(~0u, max(x[2 * a], x[2 * a + 1]));
            const uint32_t m = max(1u, static_cast<uint32_t>(hi - lo + 14) / 15u);
            // n = floor((2 (x - z) + m) / (2 m)) <= 15: (hi - z) / m <= 15
            const uint32_t n0 = (2u * static_cast<uint32_t>(x[2 * a] - lo) + m) / (2u * m);
            const uint32_t n1 = (2u * static_cast<uint32_t>(x[2 * a + 1] - lo) + m) / (2u * m);
            row[32 * a + lane] = static_cast<uint8_t>(n0 | (n1 << 4));
            if (lane == 0) scale[a] = m | (static_cast<uint32_t>(lo) << 16);
            x[2 * a] = lo + static_cast<int32_t>(m * n0);
            x[2 * a + 1] = lo + static_cast<int32_t>(m * n1);
        }
    }
}

// One warp per (row, head of q | k | v).
template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(256) k_paged_append(const AppendParams p) {
    constexpr int N = HD / 32;
    const PagedGeom& g = p.g;
    const int lane = threadIdx.x & 31;
    const int nq = p.q ? g.n_heads : 0, heads = nq + 2 * g.n_kv;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (item >= static_cast<int64_t>(p.n_rows) * heads) return;
    const int r = static_cast<int>(item / heads), h = static_cast<int>(item % heads);
    const int seq = p.seq ? p.seq[r] : r, pos = p.pos[r];
    if (seq < 0 || pos < 0) return;  // a padding row
    if (seq >= g.n_seq || pos >= p.n_pos || (pos >> g.page_shift) >= g.ld_table) {
        if (lane == 0) atomicCAS(g.err, 0, seq >= g.n_seq ? ERR_PAGED_SEQ : ERR_PAGED_POS);
        return;
    }
    const bool is_q = h < nq, is_v = h >= nq + g.n_kv;
    const int head = is_q ? h : is_v ? h - nq - g.n_kv : h - nq;
    const T* src = is_q ? static_cast<const T*>(p.q) + r * p.ldq
                        : is_v ? static_cast<const T*>(p.v) + r * p.ldv : static_cast<const T*>(p.k) + r * p.ldk;
    int page_id = 0;
    if (!is_q) {
        page_id = g.table[seq * g.ld_table + (pos >> g.page_shift)];
        if (page_id < 0 || page_id >= g.n_pages) {
            if (lane == 0) atomicCAS(g.err, 0, ERR_PAGED_PAGE);
            return;
        }
    }
    int32_t x[N];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = src[head * HD + lane + 32 * i];
        bad |= x[i] != static_cast<int16_t>(x[i]);
    }
    if (__any_sync(~0u, bad)) {
        if (lane == 0) atomicCAS(g.err, 0, ERR_PAGED_INPUT);
        return;
    }
    if (!is_v) {
        const int shift = is_q ? p.shift_q : p.shift_k;
        const int64_t half = HD / 2;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const int64_t c = p.rope_c[pos * half + lane + 32 * i], s = p.rope_s[pos * half + lane + 32 * i];
            const int64_t a = x[i], b = x[i + N / 2];
            x[i] = static_cast<int32_t>(sat64(rs64(a * c - b * s, shift), 16));
            x[i + N / 2] = static_cast<int32_t>(sat64(rs64(b * c + a * s, shift), 16));
        }
    }
    if (is_q) {
#pragma unroll
        for (int i = 0; i < N; ++i) p.q_out[r * p.ldqo + head * HD + lane + 32 * i] = static_cast<int16_t>(x[i]);
        return;
    }
    store_row<HD, BITS>(g, (is_v ? g.v_pool : g.k_pool) + slab_offset(g, page_id, head), pos & ((1 << g.page_shift) - 1),
                        lane, x);
    if (p.kv_out) {
        int32_t* o = p.kv_out + ((static_cast<int64_t>(r) * 2 + is_v) * g.n_kv + head) * HD + lane;
#pragma unroll
        for (int i = 0; i < N; ++i) o[32 * i] = x[i];
    }
}

// --------------------------------------------------------------------------------------- attention
//   s_j = SAT16(RS(sum_d q_d k_jd, shift_s)), e_j = E[max s - s_j], Z = sum e_j,
//   P_j = floor((e_j 2^pb + floor(Z / 2)) / Z), ctx_d = SAT(RS(sum_j P_j v_jd, shift_c), bits_c)
struct PagedAttnParams {
    PagedGeom g;
    const int16_t* q;
    int64_t ldq;
    int n_rows;
    const int32_t *seq, *len;
    int max_len;
    int shift_s, prob_bits, shift_c, bits_c;
    int32_t* ctx;
    int64_t ldc;
};

// Value d of the cached row (slot) of a slab.
__device__ __forceinline__ int32_t cached_value(const PagedGeom& g, const uint8_t* slab, int slot, int d) {
    if (g.bits == 16) return reinterpret_cast<const int16_t*>(slab)[slot * g.hd + d];
    const int a = d >> 6, b = d & 63;
    const uint32_t w = reinterpret_cast<const uint32_t*>(slab + (g.hd / 2 << g.page_shift))[slot * (g.hd / 64) + a];
    const uint32_t n = (slab[slot * (g.hd / 2) + 32 * a + (b & 31)] >> (b >> 5 << 2)) & 15u;
    return (static_cast<int32_t>(w) >> 16) + static_cast<int32_t>((w & 0xffffu) * n);
}

// One block of 128 threads per (row, query head): three passes over the keys (maximum, sum, weights),
// each recomputing the scores.
__global__ void __launch_bounds__(128) k_paged_attention(const PagedAttnParams p) {
    const PagedGeom& g = p.g;
    __shared__ int32_t q_s[128], p_s[128], red_max;
    __shared__ unsigned long long red_sum;
    const int r = blockIdx.x / g.n_heads, head = blockIdx.x % g.n_heads, kv = head / g.group, tid = threadIdx.x;
    const int seq = p.seq ? p.seq[r] : r, len = p.len[r];
    if (seq < 0) return;  // a padding row
    const int64_t cols = (static_cast<int64_t>(len) + (1 << g.page_shift) - 1) >> g.page_shift;
    if (seq >= g.n_seq || len > p.max_len || cols > g.ld_table) {
        if (tid == 0) atomicCAS(g.err, 0, seq >= g.n_seq ? ERR_PAGED_SEQ : ERR_PAGED_LEN);
        return;
    }
    const int32_t* table = g.table + seq * g.ld_table;
    if (tid < g.hd) q_s[tid] = p.q[r * p.ldq + head * g.hd + tid];
    if (tid == 0) {
        red_max = -32768;
        red_sum = 0;
    }
    __syncthreads();
    auto slab_of = [&](const uint8_t* pool, int j) -> const uint8_t* {
        int id = table[j >> g.page_shift];
        if (id < 0 || id >= g.n_pages) {
            atomicCAS(g.err, 0, ERR_PAGED_PAGE);
            id = 0;
        }
        return pool + slab_offset(g, id, kv);
    };
    auto score = [&](int j) -> int32_t {
        const uint8_t* slab = slab_of(g.k_pool, j);
        const int slot = j & ((1 << g.page_shift) - 1);
        int64_t acc = 0;
        for (int d = 0; d < g.hd; ++d) acc += static_cast<int64_t>(q_s[d]) * cached_value(g, slab, slot, d);
        return static_cast<int32_t>(sat64(rs64(acc, p.shift_s), 16));
    };
    int32_t m = -32768;
    for (int j = tid; j < len; j += 128) m = max(m, score(j));
    atomicMax(&red_max, m);
    __syncthreads();
    m = red_max;
    auto weight = [&](int j) -> int64_t {
        const int d = m - score(j);
        return d > PAGED_DMAX ? 0 : g.exp_tab[d];
    };
    unsigned long long z = 0;
    for (int j = tid; j < len; j += 128) z += weight(j);
    atomicAdd(&red_sum, z);
    __syncthreads();
    z = red_sum;
    int64_t acc = 0;
    for (int j0 = 0; j0 < len; j0 += 128) {
        if (j0 + tid < len) p_s[tid] = static_cast<int32_t>(((static_cast<unsigned long long>(weight(j0 + tid)) << p.prob_bits) + (z >> 1)) / z);
        __syncthreads();
        if (tid < g.hd)
            for (int j = j0; j < len && j < j0 + 128; ++j)
                acc += static_cast<int64_t>(p_s[j - j0]) *
                       cached_value(g, slab_of(g.v_pool, j), j & ((1 << g.page_shift) - 1), tid);
        __syncthreads();
    }
    if (tid < g.hd)
        p.ctx[r * p.ldc + head * g.hd + tid] = static_cast<int32_t>(sat64(rs64(acc, p.shift_c), p.bits_c));
}

}  // namespace eii
