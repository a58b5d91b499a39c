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

// Geometry of the kernel below.  A tile is 32 keys of one warp; a block holds the scores of one part of
// the keys for up to four query heads in shared memory.
constexpr int PATTN_HEADS = 4;          // query heads of one block (they share a kv head)
constexpr int PATTN_MAX_PART = 8192;    // keys of one block: 64 KB of scores
constexpr int PATTN_MAX_CLUSTER = 16;
constexpr int PATTN_EXP_BYTES = (PAGED_DMAX + 1 + 3) / 4 * 16;

template <int HD, int BITS>
struct PattnCfg {
    static constexpr int A = HD / 64;                        // scale groups of a row
    static constexpr int KS = HD / 32;                       // 32-wide steps of the score product
    static constexpr int SWEEPS = BITS == 4 ? 1 : A;         // passes over V (64 accumulators at most per thread)
    static constexpr int GPS = A / SWEEPS;                   // 64-dim groups per sweep
    static constexpr int NT = BITS == 4 ? 8 * GPS : 16;      // 8-column accumulator tiles
    static constexpr int RAW_ROW = BITS == 4 ? 40 : 36;      // padded row of 32 raw scores
    static constexpr int RAW_BYTES = PATTN_HEADS * RAW_ROW * (BITS == 4 ? 4 * A : 8);
    static constexpr int PLANE_BYTES = 16 * 32 * (BITS == 4 ? A : 1);
    static constexpr int WARP_BYTES = RAW_BYTES > PLANE_BYTES ? RAW_BYTES : PLANE_BYTES;  // the two uses do not overlap in time
    static constexpr int ACC_COLS = BITS == 4 ? 64 * GPS : 128;  // columns of the block's accumulator rows
    static constexpr int ACC_LD = ACC_COLS + 8;
    static constexpr int ACC_BYTES = 16 * ACC_LD * 4;
    static constexpr int CTX_BYTES = PATTN_HEADS * HD * 8;
    static constexpr int smem(int warps, int part) {
        return PATTN_EXP_BYTES + ACC_BYTES + CTX_BYTES + warps * WARP_BYTES + PATTN_HEADS * part * 2;
    }
};

// D += A B on 16 x 8 x 32 bytes: A rows are query heads (scores) or head x weight plane (context), B
// columns are keys or dimensions.  A decoding step has a handful of rows, so the 128-row tcgen05 tile
// would be empty: the warp-level instruction takes its operands from registers, straight from the loads.
template <bool A_SIGNED, bool B_SIGNED>
__device__ __forceinline__ void mma_m16n8k32(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    if constexpr (A_SIGNED && B_SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else if constexpr (A_SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else if constexpr (B_SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Byte j of x0..x3 -> r_j (x0's byte lowest).
__device__ __forceinline__ void transpose4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t (&r)[4]) {
    const uint32_t t0 = __byte_perm(x0, x1, 0x5140), t1 = __byte_perm(x2, x3, 0x5140);
    const uint32_t t2 = __byte_perm(x0, x1, 0x7362), t3 = __byte_perm(x2, x3, 0x7362);
    r[0] = __byte_perm(t0, t1, 0x5410);
    r[1] = __byte_perm(t0, t1, 0x7632);
    r[2] = __byte_perm(t2, t3, 0x5410);
    r[3] = __byte_perm(t2, t3, 0x7632);
}

// floor((e 2^pb + floor(z / 2)) / z): the float estimate is off by at most one (e 2^pb / z <= 2^19 with
// three roundings of 2^-24), which the exact remainder corrects.
__device__ __forceinline__ uint32_t prob_of(uint32_t e, int pb, uint64_t z, float scale) {
    const uint64_t num = (static_cast<uint64_t>(e) << pb) + (z >> 1);
    uint32_t est = static_cast<uint32_t>(__fmaf_rz(static_cast<float>(e), scale, 0.5f));
    const int64_t rem = static_cast<int64_t>(num - est * z);
    if (rem < 0) --est;
    else if (rem >= static_cast<int64_t>(z)) ++est;
    return est;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t remote_smem(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int32_t ld_remote32(uint32_t a) {
    int32_t v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ int64_t ld_remote64(uint32_t a) {
    int64_t v;
    asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

// One cluster of `cs` blocks per (row, kv head, tile of four query heads); block `rank` takes a contiguous
// part of the keys, its warps every NW-th tile of 32 of them.  K and V are read once: pass 1 writes
// SAT16 scores to shared memory and finds the maximum (joined over the cluster), pass 2 sums the
// exponentials from the scores, pass 3 turns them into probabilities and multiplies V.  All sums are
// exact integers, so neither the split nor the order changes a result.
//   scores: q = 256 qh + ql (s8, u8 rows of A); keys are B columns.  4 bits: nibbles are B bytes as they
//     lie (byte j of a group holds dimensions j and j + 32), s = sum_a m_a (q . n)_a + z_a sum(q_a).
//     16 bits: k = 256 kh + kl split by byte permutes.
//   context: 4 bits: W = P m <= 2^19 4369 + 4369 < 2^32 as four u8 planes, sum_j P_j z_j apart; 16 bits:
//     P as three planes.  Keys run along the product's K: four keys' words are transposed in registers.
template <int HD, int BITS>
__global__ void __launch_bounds__(256, BITS == 4 && HD == 64 ? 3 : 2) k_paged_attention(const PagedAttnParams p, const int cs, const int part_cap) {
    using C = PattnCfg<HD, BITS>;
    constexpr int H = PATTN_HEADS, A = C::A;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int32_t max_s[H];
    __shared__ unsigned long long z_s[H];
    __shared__ uint32_t zlo_s[H * A];  // 8 warps x 32 lanes x 2^24
    __shared__ int32_t zhi_s[H * A];
    const PagedGeom& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    int32_t* exp_s = reinterpret_cast<int32_t*>(smem);
    int32_t* acc_s = reinterpret_cast<int32_t*>(smem + PATTN_EXP_BYTES);
    int64_t* ctx_s = reinterpret_cast<int64_t*>(smem + PATTN_EXP_BYTES + C::ACC_BYTES);
    uint8_t* stage = smem + PATTN_EXP_BYTES + C::ACC_BYTES + C::CTX_BYTES + warp * C::WARP_BYTES;
    int16_t* score_s = reinterpret_cast<int16_t*>(smem + PATTN_EXP_BYTES + C::ACC_BYTES + C::CTX_BYTES + nw * C::WARP_BYTES);

    const int rank = cs > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int head_tiles = (g.group + H - 1) / H;
    int item = blockIdx.x / cs;
    const int ht = item % head_tiles;
    item /= head_tiles;
    const int kv = item % g.n_kv, r = item / g.n_kv;
    const int head0 = kv * g.group + ht * H, nh = min(H, g.group - ht * H);
    const int seq = p.seq ? p.seq[r] : r;
    if (seq < 0) return;  // a padding row (the whole cluster agrees)
    const int len = max(p.len[r], 0);
    if (seq >= g.n_seq || len > p.max_len || ((static_cast<int64_t>(len) + (1 << g.page_shift) - 1) >> g.page_shift) > g.ld_table) {
        if (tid == 0) atomicCAS(g.err, 0, seq >= g.n_seq ? ERR_PAGED_SEQ : ERR_PAGED_LEN);
        return;
    }
    int32_t* ctx = p.ctx + r * p.ldc + head0 * HD;
    if (len == 0) {
        if (rank == 0)
            for (int i = tid; i < nh * HD; i += blockDim.x) ctx[i] = 0;
        return;
    }
    const int32_t* table = g.table + seq * g.ld_table;
    const int tiles = (len + 31) >> 5;
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * rank / cs);
    const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / cs);

    for (int i = tid; i <= PAGED_DMAX; i += blockDim.x) exp_s[i] = g.exp_tab[i];
    for (int i = tid; i < C::ACC_BYTES / 4; i += blockDim.x) acc_s[i] = 0;
    if (tid < H) {
        max_s[tid] = -32768;
        z_s[tid] = 0;
    }
    if (tid < H * A) {
        zlo_s[tid] = 0;
        zhi_s[tid] = 0;
    }

    const int gid = lane >> 2, tig = lane & 3;
    // q fragments: step i of row gid holds dimensions 32 i + 8 tig .. + 7 (two words of each plane)
    uint32_t qh[C::KS][2], ql[C::KS][2];
    int32_t qsum[A];
#pragma unroll
    for (int a = 0; a < A; ++a) qsum[a] = 0;
#pragma unroll
    for (int i = 0; i < C::KS; ++i) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t hi = 0, lo = 0;
            if (gid < nh) {
                const int16_t* src = p.q + r * p.ldq + (head0 + gid) * HD + 32 * i + 8 * tig + 4 * w;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int32_t x = src[b];
                    hi |= (static_cast<uint32_t>(x >> 8) & 0xFFu) << (8 * b);
                    lo |= (static_cast<uint32_t>(x) & 0xFFu) << (8 * b);
                    qsum[i >> 1] += x;
                }
            }
            qh[i][w] = hi;
            ql[i][w] = lo;
        }
    }
    int32_t qs[H][A];  // sum of each head's q over each group, in every lane
#pragma unroll
    for (int a = 0; a < A; ++a) {
        qsum[a] += __shfl_xor_sync(~0u, qsum[a], 1);
        qsum[a] += __shfl_xor_sync(~0u, qsum[a], 2);
#pragma unroll
        for (int h = 0; h < H; ++h) qs[h][a] = __shfl_sync(~0u, qsum[a], 4 * h);
    }

    // the two pages of a tile (pages hold at least 16 keys); entries behind the last key are not followed
    auto page_ids = [&](int t, int (&id)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = 32 * t + 16 * h;
            id[h] = j < len ? table[j >> g.page_shift] : -2;
        }
    };
    auto slabs = [&](const uint8_t* pool, const int (&id)[2], int t, const uint8_t* (&s)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int x = id[h] == -2 ? id[0] : id[h];
            if (x < 0 || x >= g.n_pages) {
                if (lane == 0) atomicCAS(g.err, 0, ERR_PAGED_PAGE);
                x = 0;
            }
            s[h] = pool + slab_offset(g, x, kv);
        }
    };
    const int slot_mask = (1 << g.page_shift) - 1;
    const int scale_at = (HD / 2) << g.page_shift;

    // ---------------------------------------------------------------- pass 1: scores and their maximum
    int32_t mx[H];
#pragma unroll
    for (int h = 0; h < H; ++h) mx[h] = -32768;
    for (int t = t0 + warp; t < t1; t += nw) {
        int id[2];
        const uint8_t* sl[2];
        page_ids(t, id);
        slabs(g.k_pool, id, t, sl);
        const int slot0 = (32 * t) & slot_mask, slot1 = (32 * t + 16) & slot_mask;
        if constexpr (BITS == 4) {
            uint2 kw[A][4];
            uint32_t sw[A];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint8_t* row = sl[n >> 1] + ((n >> 1 ? slot1 : slot0) + 8 * (n & 1) + gid) * (HD / 2);
#pragma unroll
                for (int a = 0; a < A; ++a) kw[a][n] = *reinterpret_cast<const uint2*>(row + 32 * a + 8 * tig);
            }
            {
                const uint32_t* w = reinterpret_cast<const uint32_t*>((lane < 16 ? sl[0] : sl[1]) + scale_at) +
                                    ((lane < 16 ? slot0 : slot1) + (lane & 15)) * A;
#pragma unroll
                for (int a = 0; a < A; ++a) sw[a] = w[a];
            }
            int32_t* raw = reinterpret_cast<int32_t*>(stage);
#pragma unroll
            for (int a = 0; a < A; ++a)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    int32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
                    const uint32_t l0 = kw[a][n].x & 0x0F0F0F0Fu, l1 = kw[a][n].y & 0x0F0F0F0Fu;
                    const uint32_t h0 = (kw[a][n].x >> 4) & 0x0F0F0F0Fu, h1 = (kw[a][n].y >> 4) & 0x0F0F0F0Fu;
                    mma_m16n8k32<true, false>(hi, qh[2 * a][0], 0, qh[2 * a][1], 0, l0, l1);
                    mma_m16n8k32<false, false>(lo, ql[2 * a][0], 0, ql[2 * a][1], 0, l0, l1);
                    mma_m16n8k32<true, false>(hi, qh[2 * a + 1][0], 0, qh[2 * a + 1][1], 0, h0, h1);
                    mma_m16n8k32<false, false>(lo, ql[2 * a + 1][0], 0, ql[2 * a + 1][1], 0, h0, h1);
                    if (gid < nh)
                        *reinterpret_cast<int2*>(raw + (a * H + gid) * C::RAW_ROW + 8 * n + 2 * tig) =
                            make_int2(hi[0] * 256 + lo[0], hi[1] * 256 + lo[1]);
                }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (h >= nh) break;
                int64_t acc = 0;
#pragma unroll
                for (int a = 0; a < A; ++a)
                    acc += static_cast<int64_t>(raw[(a * H + h) * C::RAW_ROW + lane]) * static_cast<int32_t>(sw[a] & 0xFFFFu) +
                           static_cast<int64_t>(qs[h][a]) * (static_cast<int32_t>(sw[a]) >> 16);
                const int32_t s = static_cast<int32_t>(sat64(rs64(acc, p.shift_s), 16));
                score_s[h * part_cap + 32 * (t - t0) + lane] = static_cast<int16_t>(s);
                if (32 * t + lane < len) mx[h] = max(mx[h], s);
            }
        } else {
            int64_t* raw = reinterpret_cast<int64_t*>(stage);
            uint4 kw[C::KS][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint8_t* row = sl[n >> 1] + ((n >> 1 ? slot1 : slot0) + 8 * (n & 1) + gid) * (HD * 2);
#pragma unroll
                for (int i = 0; i < C::KS; ++i) kw[i][n] = *reinterpret_cast<const uint4*>(row + 64 * i + 16 * tig);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                int32_t hh[4] = {0, 0, 0, 0}, mid[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < C::KS; ++i) {
                    const uint4 w = kw[i][n];
                    const uint32_t l0 = __byte_perm(w.x, w.y, 0x6420), l1 = __byte_perm(w.z, w.w, 0x6420);
                    const uint32_t h0 = __byte_perm(w.x, w.y, 0x7531), h1 = __byte_perm(w.z, w.w, 0x7531);
                    mma_m16n8k32<true, true>(hh, qh[i][0], 0, qh[i][1], 0, h0, h1);
                    mma_m16n8k32<true, false>(mid, qh[i][0], 0, qh[i][1], 0, l0, l1);
                    mma_m16n8k32<false, true>(mid, ql[i][0], 0, ql[i][1], 0, h0, h1);
                    mma_m16n8k32<false, false>(ll, ql[i][0], 0, ql[i][1], 0, l0, l1);
                }
                if (gid < nh) {
                    int64_t* o = raw + gid * C::RAW_ROW + 8 * n + 2 * tig;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        o[c] = static_cast<int64_t>(hh[c]) * 65536 + static_cast<int64_t>(mid[c]) * 256 + ll[c];
                }
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (h >= nh) break;
                const int32_t s = static_cast<int32_t>(sat64(rs64(raw[h * C::RAW_ROW + lane], p.shift_s), 16));
                score_s[h * part_cap + 32 * (t - t0) + lane] = static_cast<int16_t>(s);
                if (32 * t + lane < len) mx[h] = max(mx[h], s);
            }
        }
        __syncwarp();
    }
    __syncthreads();  // the block's tables and reduction words are set
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int32_t m = __reduce_max_sync(~0u, mx[h]);
        if (lane == 0) atomicMax(&max_s[h], m);
    }
    if (cs > 1) {
        cluster_barrier();
#pragma unroll
        for (int h = 0; h < H; ++h)
            mx[h] = __reduce_max_sync(~0u, lane < cs ? ld_remote32(remote_smem(&max_s[h], lane)) : -32768);
    } else {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < H; ++h) mx[h] = max_s[h];
    }

    // ---------------------------------------------------------------- pass 2: sum of the exponentials
    {
        unsigned long long z[H];
#pragma unroll
        for (int h = 0; h < H; ++h) z[h] = 0;
        for (int t = t0 + warp; t < t1; t += nw)
            if (32 * t + lane < len)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    if (h >= nh) break;
                    const int32_t d = mx[h] - score_s[h * part_cap + 32 * (t - t0) + lane];
                    z[h] += d > PAGED_DMAX ? 0 : exp_s[d];
                }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            // in pieces of 24 and 32 bits: 32 lanes of 2^24 and of 2^47 / 2^24 stay in 32 bits
            const uint32_t lo = __reduce_add_sync(~0u, static_cast<uint32_t>(z[h]) & 0xFFFFFFu);
            const uint32_t hi = __reduce_add_sync(~0u, static_cast<uint32_t>(z[h] >> 24));
            if (lane == 0) atomicAdd(&z_s[h], (static_cast<unsigned long long>(hi) << 24) + lo);
        }
    }
    uint64_t z[H];
    if (cs > 1) {
        cluster_barrier();
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint64_t v = lane < cs ? static_cast<uint64_t>(ld_remote64(remote_smem(&z_s[h], lane))) : 0;
            const uint32_t lo = __reduce_add_sync(~0u, static_cast<uint32_t>(v) & 0xFFFFFFu);
            const uint32_t hi = __reduce_add_sync(~0u, static_cast<uint32_t>(v >> 24));
            z[h] = (static_cast<uint64_t>(hi) << 24) + lo;
        }
    } else {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < H; ++h) z[h] = z_s[h];
    }

    // ---------------------------------------------------------------- pass 3: probabilities times V
    float zscale[H];
#pragma unroll
    for (int h = 0; h < H; ++h) zscale[h] = __fdiv_rn(static_cast<float>(1 << p.prob_bits), static_cast<float>(z[h]));
    // key lane of a tile -> its byte of a plane row, so that a thread's 8 bytes are keys tig + 4 i + 16 h
    const int plane_at = 8 * (lane & 3) + 4 * (lane >> 4) + ((lane >> 2) & 3);
    for (int sweep = 0; sweep < C::SWEEPS; ++sweep) {
        int32_t acc[C::NT][4];
#pragma unroll
        for (int i = 0; i < C::NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
        int64_t pz[H][A];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int a = 0; a < A; ++a) pz[h][a] = 0;
        if (nh < H)
            for (int i = lane; i < C::PLANE_BYTES / 4; i += 32) reinterpret_cast<uint32_t*>(stage)[i] = 0;  // absent heads
        __syncwarp();
        for (int t = t0 + warp; t < t1; t += nw) {
            int id[2];
            const uint8_t* sl[2];
            page_ids(t, id);
            slabs(g.v_pool, id, t, sl);
            const int slot0 = (32 * t) & slot_mask, slot1 = (32 * t + 16) & slot_mask;
            uint32_t vw[BITS == 4 ? A : 4][8];  // [group or word][key tig + 4 i (+ 16)]
            uint32_t sw[A];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int slot = (i < 4 ? slot0 : slot1) + tig + 4 * (i & 3);
                if constexpr (BITS == 4) {
#pragma unroll
                    for (int a = 0; a < A; ++a)
                        vw[a][i] = *reinterpret_cast<const uint32_t*>(sl[i >> 2] + slot * (HD / 2) + 32 * a + 4 * gid);
                } else {
                    const uint4 w = *reinterpret_cast<const uint4*>(sl[i >> 2] + slot * (HD * 2) + 128 * sweep + 16 * gid);
                    vw[0][i] = w.x; vw[1][i] = w.y; vw[2][i] = w.z; vw[3][i] = w.w;
                }
            }
            if constexpr (BITS == 4) {
                const uint32_t* w = reinterpret_cast<const uint32_t*>((lane < 16 ? sl[0] : sl[1]) + scale_at) +
                                    ((lane < 16 ? slot0 : slot1) + (lane & 15)) * A;
#pragma unroll
                for (int a = 0; a < A; ++a) sw[a] = w[a];
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (h >= nh) break;
                uint32_t pr = 0;
                if (32 * t + lane < len) {
                    const int32_t d = mx[h] - score_s[h * part_cap + 32 * (t - t0) + lane];
                    if (d <= PAGED_DMAX) pr = prob_of(exp_s[d], p.prob_bits, z[h], zscale[h]);
                }
                if constexpr (BITS == 4) {
#pragma unroll
                    for (int a = 0; a < A; ++a) {
                        const uint32_t w = pr * (sw[a] & 0xFFFFu);
                        pz[h][a] += static_cast<int64_t>(static_cast<int32_t>(pr)) * (static_cast<int32_t>(sw[a]) >> 16);
#pragma unroll
                        for (int b = 0; b < 4; ++b) stage[a * 512 + (h * 4 + b) * 32 + plane_at] = static_cast<uint8_t>(w >> (8 * b));
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b) stage[(h * 4 + b) * 32 + plane_at] = static_cast<uint8_t>(pr >> (8 * b));
                }
            }
            __syncwarp();
#pragma unroll
            for (int a = 0; a < C::GPS; ++a) {
                const uint2 x = *reinterpret_cast<const uint2*>(stage + (BITS == 4 ? a * 512 : 0) + gid * 32 + 8 * tig);
                const uint2 y = *reinterpret_cast<const uint2*>(stage + (BITS == 4 ? a * 512 : 0) + (gid + 8) * 32 + 8 * tig);
                if constexpr (BITS == 4) {
                    uint32_t b0[4], b1[4];
                    transpose4(vw[a][0], vw[a][1], vw[a][2], vw[a][3], b0);
                    transpose4(vw[a][4], vw[a][5], vw[a][6], vw[a][7], b1);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_m16n8k32<false, false>(acc[8 * a + 2 * j], x.x, y.x, x.y, y.y, b0[j] & 0x0F0F0F0Fu, b1[j] & 0x0F0F0F0Fu);
                        mma_m16n8k32<false, false>(acc[8 * a + 2 * j + 1], x.x, y.x, x.y, y.y, (b0[j] >> 4) & 0x0F0F0F0Fu,
                                                   (b1[j] >> 4) & 0x0F0F0F0Fu);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t b0[4], b1[4];
                        transpose4(vw[j][0], vw[j][1], vw[j][2], vw[j][3], b0);
                        transpose4(vw[j][4], vw[j][5], vw[j][6], vw[j][7], b1);
                        mma_m16n8k32<false, false>(acc[4 * j + 0], x.x, y.x, x.y, y.y, b0[0], b1[0]);
                        mma_m16n8k32<false, true>(acc[4 * j + 1], x.x, y.x, x.y, y.y, b0[1], b1[1]);
                        mma_m16n8k32<false, false>(acc[4 * j + 2], x.x, y.x, x.y, y.y, b0[2], b1[2]);
                        mma_m16n8k32<false, true>(acc[4 * j + 3], x.x, y.x, x.y, y.y, b0[3], b1[3]);
                    }
                }
            }
            __syncwarp();
        }
        // join the warps: 255 x 255 x PATTN_MAX_PART stays in 32 bits
        if (t0 + warp < t1) {
#pragma unroll
            for (int i = 0; i < C::NT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int col = 2 * tig + (c & 1);
                    const int at = BITS == 4 ? 64 * (i >> 3) + 4 * col + ((i & 7) >> 1) + 32 * (i & 1)
                                             : 64 * (i & 1) + 8 * col + 2 * (i >> 2) + ((i >> 1) & 1);
                    if ((gid + 8 * (c >> 1)) < 4 * nh) atomicAdd(&acc_s[(gid + 8 * (c >> 1)) * C::ACC_LD + at], acc[i][c]);
                }
            if constexpr (BITS == 4) {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int a = 0; a < A; ++a) {
                        const uint32_t lo = __reduce_add_sync(~0u, static_cast<uint32_t>(pz[h][a]) & 0xFFFFFFu);
                        const int32_t hi = __reduce_add_sync(~0u, static_cast<int32_t>(pz[h][a] >> 24));
                        if (lane == 0) {
                            atomicAdd(&zlo_s[h * A + a], lo);
                            atomicAdd(&zhi_s[h * A + a], hi);
                        }
                    }
            }
        }
        __syncthreads();
        for (int i = tid; i < nh * 64 * C::GPS; i += blockDim.x) {
            const int h = i / (64 * C::GPS), d = i % (64 * C::GPS);
            int64_t v = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                int32_t* x = acc_s + (4 * h + b) * C::ACC_LD + d;
                int64_t y = x[0];
                if constexpr (BITS == 16) {
                    y += static_cast<int64_t>(x[64]) * 256;
                    if (sweep + 1 < C::SWEEPS) x[0] = x[64] = 0;
                }
                v += y << (8 * b);
            }
            if constexpr (BITS == 4)
                v += static_cast<int64_t>(zlo_s[h * A + (d >> 6)]) + (static_cast<int64_t>(zhi_s[h * A + (d >> 6)]) << 24);
            if (cs > 1) ctx_s[h * HD + 64 * sweep + d] = v;
            else ctx[h * HD + 64 * sweep + d] = static_cast<int32_t>(sat64(rs64(v, p.shift_c), p.bits_c));
        }
        if (sweep + 1 < C::SWEEPS) __syncthreads();
    }
    if (cs > 1) {
        cluster_barrier();
        for (int i = rank * blockDim.x + tid; i < nh * HD; i += cs * blockDim.x) {
            int64_t v = 0;
            for (int c = 0; c < cs; ++c) v += ld_remote64(remote_smem(ctx_s + i, c));
            ctx[i] = static_cast<int32_t>(sat64(rs64(v, p.shift_c), p.bits_c));
        }
        cluster_barrier();  // no block leaves while its words are read
    }
}

}  // namespace eii
