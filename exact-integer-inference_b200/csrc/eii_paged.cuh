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

#include "eii_cluster.cuh"
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
    const int32_t* exp_tab;        // [PAGED_DMAX + 1], Q30, and zeros to a multiple of four words
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

// SAT16(x >> shift) with the rounding half already added to x, |x| >> `fits` below 2^31.  From a shift of
// `fits` to 31 the low word is the answer, one above is taken in two steps; below `fits` (at most 16) x is
// clamped to 2^30 first, which changes only values that saturate.
struct Requant16 {
    int down, rest;
    bool clamp;
    int64_t half;
    __device__ Requant16(int shift, int fits)
        : down(min(shift, 32)), rest(max(shift - 32, 0)), clamp(shift < fits), half(int64_t(1) << (shift - 1)) {}
    __device__ __forceinline__ int32_t operator()(int64_t x) const {
        if (clamp) x = max(min(x, (int64_t(1) << 30) - 1), -(int64_t(1) << 30));
        const int32_t s = static_cast<int32_t>(__funnelshift_rc(static_cast<uint32_t>(x), static_cast<uint32_t>(x >> 32), down)) >> rest;
        return max(min(s, 32767), -32768);
    }
};

// The lanes of a head: each has dimensions 4 l .. 4 l + 3 and the same of the other half.
template <int HD>
struct AppendLanes {
    static constexpr int LANES = HD / 8, HEADS = 32 / LANES;  // of one warp
};

template <typename T>
__device__ __forceinline__ void load4(const T* src, bool vec, int32_t (&x)[4]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = src[i];
    } else if constexpr (sizeof(T) == 4) {
        const int4 w = *reinterpret_cast<const int4*>(src);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    } else {
        const int2 w = *reinterpret_cast<const int2*>(src);
        x[0] = static_cast<int16_t>(w.x); x[1] = w.x >> 16; x[2] = static_cast<int16_t>(w.y); x[3] = w.y >> 16;
    }
}

// Nibbles of a group's values x (each lane's four of a or b) for a span of `lanes` lanes that share the group;
// x becomes what the nibbles stand for.  floor(n / d) for n < 2^18, d = 2 m <= 2^13.1 is umulhi(n, floor((2^32 -
// 1) / d) + 1): the reciprocal's error adds less than 2^-14 to a quotient whose fraction is a multiple of 1 / d.
template <int LANES, int N>
__device__ __forceinline__ uint32_t quantise4(int32_t (&x)[N], uint32_t (&nib)[N]) {
    int32_t lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) {
        lo = min(lo, x[i]);
        hi = max(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) {
        lo = min(lo, __shfl_xor_sync(~0u, lo, o));
        hi = max(hi, __shfl_xor_sync(~0u, hi, o));
    }
    const uint32_t m = max(1u, static_cast<uint32_t>(hi - lo + 14) / 15u), rcp = 0xFFFFFFFFu / (2 * m) + 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        nib[i] = __umulhi(2 * static_cast<uint32_t>(x[i] - lo) + m, rcp);
        x[i] = lo + static_cast<int32_t>(m * nib[i]);
    }
    return m | (static_cast<uint32_t>(lo) << 16);
}

// `wpr` warps per row take turns at its steps: four (two) heads of q, then of k, then of v, HD / 8 lanes each; the
// row's position, page and each lane's four cosines and sines stay in registers.  16-byte loads of int32
// inputs, 8-byte ones of int16, element by element where alignment does not allow them.  65536 rows of 15
// heads to 16 bits take 100 us (0.73 of the copy rate), one warp per head and row 226.  Bound by the latency of its
// loads, for which a warp waits more than half of its time, with the 34 warps that an SM holds at 48 registers (issue
// slots 52% busy, integer pipe 39%); 20011 rows of 48 heads of 128 to 4 bits 152 us (0.61), 28 warps at 62 (49%, 39%).
template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(256) k_paged_append(const AppendParams p, const int wpr, const int vec_in, const int vec_out) {
    constexpr int LANES = AppendLanes<HD>::LANES, HEADS = AppendLanes<HD>::HEADS, HALF = HD / 2;
    const PagedGeom& g = p.g;
    const int lane = threadIdx.x & 31, l = lane % LANES, sub = lane / LANES;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int r = static_cast<int>(index / wpr);
    if (r >= p.n_rows) return;
    const int seq = p.seq ? p.seq[r] : r, pos = p.pos[r];
    if (seq < 0 || pos < 0) return;  // a padding row
    if (seq >= g.n_seq || pos >= p.n_pos || (pos >> g.page_shift) >= g.ld_table) {
        if (lane == 0) atomicCAS(g.err, 0, seq >= g.n_seq ? ERR_PAGED_SEQ : ERR_PAGED_POS);
        return;
    }
    const int page_id = g.table[seq * g.ld_table + (pos >> g.page_shift)];
    // (q's loads and rotation need not wait for it; n_pages is below 2^31)
    auto in_pool = [&]() { return static_cast<uint32_t>(page_id) < static_cast<uint32_t>(g.n_pages); };
    const int4 c4 = *reinterpret_cast<const int4*>(p.rope_c + static_cast<int64_t>(pos) * HALF + 4 * l);
    const int4 s4 = *reinterpret_cast<const int4*>(p.rope_s + static_cast<int64_t>(pos) * HALF + 4 * l);
    const int32_t cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
    const int steps_q = p.q ? (g.n_heads + HEADS - 1) / HEADS : 0, steps_kv = (g.n_kv + HEADS - 1) / HEADS;

    // this lane's eight values of a head; true when all of the head's lie in the int16 range
    auto load8 = [&](const T* src, int32_t (&x)[8]) {
        int32_t a[4], b[4];
        load4(src + 4 * l, vec_in, a);
        load4(src + HALF + 4 * l, vec_in, b);
        uint32_t over = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
            over |= static_cast<uint32_t>(a[i] + 32768) | static_cast<uint32_t>(b[i] + 32768);
        }
        if constexpr (sizeof(T) == 2) return true;
        const uint32_t mine = ((1ull << LANES) - 1) << (sub * LANES);
        if ((__ballot_sync(~0u, over >> 16 != 0) & mine) == 0) return true;
        if (l == 0) atomicCAS(g.err, 0, ERR_PAGED_INPUT);
        return false;
    };
    // |sum| <= 2^46: a shift of 16 to 31 leaves 32 bits, which the caller saturates
    auto rotate8 = [&](int32_t (&x)[8], int shift) {
        const Requant16 down(shift, 16);
        const bool plain = shift >= 16 && shift <= 31;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t u = static_cast<int64_t>(x[i]) * cv[i] + down.half - static_cast<int64_t>(x[4 + i]) * sv[i];
            const int64_t w = static_cast<int64_t>(x[4 + i]) * cv[i] + down.half + static_cast<int64_t>(x[i]) * sv[i];
            if (plain) {
                x[i] = static_cast<int32_t>(__funnelshift_r(static_cast<uint32_t>(u), static_cast<uint32_t>(u >> 32), shift));
                x[4 + i] = static_cast<int32_t>(__funnelshift_r(static_cast<uint32_t>(w), static_cast<uint32_t>(w >> 32), shift));
            } else {
                x[i] = down(u);
                x[4 + i] = down(w);
            }
        }
    };
    auto store8 = [&](int16_t* o, const int32_t (&x)[8], bool vec) {
        const uint2 a = make_uint2(pack_sat_s16(x[1], x[0]), pack_sat_s16(x[3], x[2]));
        const uint2 b = make_uint2(pack_sat_s16(x[5], x[4]), pack_sat_s16(x[7], x[6]));
        o += 4 * l;
        if (vec) {
            *reinterpret_cast<uint2*>(o) = a;
            *reinterpret_cast<uint2*>(o + HALF) = b;
        } else {
            o[0] = a.x; o[1] = a.x >> 16; o[2] = a.y; o[3] = a.y >> 16;
            o[HALF] = b.x; o[HALF + 1] = b.x >> 16; o[HALF + 2] = b.y; o[HALF + 3] = b.y >> 16;
        }
    };

    int step = static_cast<int>(index % wpr);
#pragma unroll 2
    for (; step < steps_q; step += wpr) {
        const int head = step * HEADS + sub, from = min(head, g.n_heads - 1);  // (lanes behind the last head repeat it)
        int32_t x[8];
        const bool good = load8(static_cast<const T*>(p.q) + r * p.ldq + from * HD, x);
        rotate8(x, p.shift_q);
        if (good && head < g.n_heads && in_pool()) store8(p.q_out + r * p.ldqo + head * HD, x, vec_out & 1);
    }
    if (step >= steps_q + 2 * steps_kv) return;
    if (!in_pool()) {
        if (lane == 0) atomicCAS(g.err, 0, ERR_PAGED_PAGE);
        return;
    }
    const int slot = pos & ((1 << g.page_shift) - 1);
#pragma unroll 1
    for (; step < steps_q + 2 * steps_kv; step += wpr) {
        const bool is_v = step >= steps_q + steps_kv;
        const int head = (step - steps_q - (is_v ? steps_kv : 0)) * HEADS + sub, from = min(head, g.n_kv - 1);
        int32_t x[8];
        bool good = load8((is_v ? static_cast<const T*>(p.v) + r * p.ldv : static_cast<const T*>(p.k) + r * p.ldk) + from * HD, x);
        if (!is_v) {
            rotate8(x, p.shift_k);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = max(min(x[i], 32767), -32768);
        }
        uint32_t bytes[HD / 64] = {}, scale[HD / 64] = {};
        if constexpr (BITS == 4 && HD == 64) {
            uint32_t nib[8];
            scale[0] = quantise4<LANES>(x, nib);
            bytes[0] = nib[0] | nib[4] << 4 | nib[1] << 8 | nib[5] << 12 | nib[2] << 16 | nib[6] << 20 | nib[3] << 24 | nib[7] << 28;
        } else if constexpr (BITS == 4) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                int32_t z[4] = {x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]};
                uint32_t n[4];
                scale[a] = quantise4<LANES>(z, n);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * a + i] = z[i];
                // lanes 0 .. 7 have the low nibbles, 8 .. 15 the high ones of the same bytes
                const uint32_t own = n[0] | n[1] << 8 | n[2] << 16 | n[3] << 24, other = __shfl_xor_sync(~0u, own, 8);
                bytes[a] = l < 8 ? own | other << 4 : other | own << 4;
            }
        }
        if (!good || head >= g.n_kv) continue;
        uint8_t* slab = (is_v ? g.v_pool : g.k_pool) + slab_offset(g, page_id, head);
        if constexpr (BITS == 16) store8(reinterpret_cast<int16_t*>(slab) + slot * HD, x, true);
        else {
            uint32_t* sc = reinterpret_cast<uint32_t*>(slab + (HALF << g.page_shift)) + slot * (HD / 64);
            // (head_dim 128: lanes 8 .. 15 hold the second group's words)
            reinterpret_cast<uint32_t*>(slab + slot * HALF)[l] = HD == 64 || l < 8 ? bytes[0] : bytes[HD / 64 - 1];
            if (l == 0) {
                if constexpr (HD == 64) sc[0] = scale[0];
                else *reinterpret_cast<uint2*>(sc) = make_uint2(scale[0], scale[1]);
            }
        }
        if (p.kv_out) {
            int32_t* o = p.kv_out + ((static_cast<int64_t>(r) * 2 + is_v) * g.n_kv + head) * HD + 4 * l;
            if (vec_out & 2) {
                *reinterpret_cast<int4*>(o) = make_int4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<int4*>(o + HALF) = make_int4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = x[i];
                    o[HALF + i] = x[4 + i];
                }
            }
        }
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
    int len_add;             // a row sees len[r] + len_add keys (len holds positions where this is 1)
    int max_len;
    int shift_s, prob_bits, shift_c, bits_c;
    int32_t* ctx;
    int64_t ldc;
    // instead of ctx: the engine's row-blocked byte planes of n_rows rows (blocked_off), in offset binary if so
    uint8_t* planes;
    int n_planes, offset;
};

// Context value `col` (of all query heads) of row r from its exact sum.
__device__ __forceinline__ void store_context(const PagedAttnParams& p, int r, int col, int64_t sum) {
    const int64_t c = sat64(rs64(sum, p.shift_c), p.bits_c);
    if (!p.planes) {
        p.ctx[r * p.ldc + col] = static_cast<int32_t>(c);
        return;
    }
    const int K = p.g.n_heads * p.g.hd;
    uint8_t* at = p.planes + blocked_off(r, col, K);
    const int64_t x = c + (p.offset ? int64_t(1) << (8 * p.n_planes - 1) : 0);
    for (int i = 0; i < p.n_planes; ++i) at[i * blocked_plane_stride(p.n_rows, K)] = plane_byte(x, i);
}

// Geometry of the kernel below.  A tile is 32 keys of one warp.
constexpr int PATTN_MAX_HEADS = 4;      // query heads of one item (they share a kv head)
constexpr int PATTN_MAX_PART = 8192;    // keys of one block: 64 KB of scores
constexpr int PATTN_MAX_WARPS = 16;     // of one block
constexpr int PATTN_MAX_CLUSTER = 16;
constexpr int PATTN_EXP_BYTES = (PAGED_DMAX + 2 + 3) / 4 * 16;  // one entry more at least: zeros, in g.exp_tab too

template <int HD, int BITS, int NH>
struct PattnCfg {
    static constexpr int A = HD / 64;                        // scale groups of a row
    static constexpr int KS = HD / 32;                       // 32-wide steps of the score product
    static constexpr int SWEEPS = BITS == 4 ? 1 : A;         // passes over V (64 accumulators at most per thread)
    static constexpr int GPS = A / SWEEPS;                   // 64-dim groups per sweep
    static constexpr int NT = BITS == 4 ? 8 * GPS : 16;      // 8-column accumulator tiles
    static constexpr int RR = NH > 2 ? 2 : 1;                // halves of the 16 product rows in use by the context
    static constexpr int ROW = BITS == 4 ? HD / 2 : HD * 2;  // bytes of a cached row without its scales
    static constexpr int TILE = 32 * ROW + (BITS == 4 ? 128 * A : 0);
    static constexpr int STAGES = BITS == 4 && HD == 64 ? 3 : 2;  // tiles of the warp's ring
    static constexpr int RAW_ROW = BITS == 4 ? 40 : 36;      // padded row of 32 raw scores
    static constexpr int RAW_BYTES = (NH + 1) * RAW_ROW * (BITS == 4 ? 4 * A : 8);
    static constexpr int WGT_BYTES = 2 * RR * 32 * 4 * (BITS == 4 ? A : 1);
    static constexpr int TEMP_BYTES = RAW_BYTES > WGT_BYTES ? RAW_BYTES : WGT_BYTES;  // never in use at once
    static constexpr int WARP_BYTES = STAGES * TILE + TEMP_BYTES;
    static constexpr int ACC_LD = 8 * NT + 8;
    static constexpr int ACC_BYTES = (8 * RR * ACC_LD + 4) * 4;  // four rows further on, one word further on
    static constexpr int CTX_BYTES = NH * HD * 8;
    // A warp on its own puts its accumulators over its ring and scores, unless another sweep needs those:
    // then behind them.
    __host__ __device__ static constexpr int warp_bytes(int part) {
        const int used = WARP_BYTES + NH * part * 2, acc = (ACC_BYTES + 15) / 16 * 16;
        return SWEEPS > 1 ? used + acc : used > acc ? used : acc;
    }
    static constexpr int smem_warp(int warps, int part) { return PATTN_EXP_BYTES + warps * warp_bytes(part); }
    static constexpr int smem_block(int warps, int part) {
        return PATTN_EXP_BYTES + ACC_BYTES + CTX_BYTES + warps * WARP_BYTES + NH * part * 2;
    }
};

// D = A B (+ D) on 16 x 8 x 32 bytes: A rows are query heads (scores) or head x weight byte (context), B
// columns are keys or dimensions.  A decoding step has a handful of rows, so the 128-row tcgen05 tile
// would be empty: the warp-level instruction takes its operands from registers, straight from the loads.
__device__ __forceinline__ void mma_s8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8s8_first(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma_u8u8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// floor((e 2^pb + floor(z / 2)) / z) for e <= 2^30 <= z, with rcp = floor(2^61 / z) <= 2^31: e rcp / 2^(61 - pb)
// + 1/2 lies above the quotient by at most 1 / (2 z) and below it by less than 2^30 / 2^(61 - pb) <= 2^-12, so
// its floor is the answer unless its fraction's leading 29 - pb bits are all ones or all zeros
// (`unsure`, one key in 2^12 at pb = 16); then prob_exact decides by the remainder.
__device__ __forceinline__ uint32_t prob_of(uint32_t e, int pb, uint32_t rcp, bool& unsure) {
    const uint32_t hi = static_cast<uint32_t>((static_cast<uint64_t>(e) * rcp + (1ull << (60 - pb))) >> 32);
    unsure |= ((hi + 1) & ((1u << (29 - pb)) - 1)) <= 1;
    return hi >> (29 - pb);
}
__device__ __forceinline__ uint32_t prob_exact(uint32_t q, uint32_t e, int pb, uint64_t z) {
    const int64_t rem = static_cast<int64_t>((static_cast<uint64_t>(e) << pb) + (z >> 1) - q * z);
    return rem < 0 ? q - 1 : rem >= static_cast<int64_t>(z) ? q + 1 : q;
}

// An item is (row, kv head, up to NH query heads).  WARP: one warp works on an item by itself (many
// short sequences).  Otherwise a cluster of `cs` blocks does: block `rank` takes a contiguous part of the
// keys, its warps every nw-th tile of 32 of them.
// K and V are read once, as one stream of tiles that each warp copies ahead of itself into a ring in
// shared memory: pass 1 writes SAT16 scores to shared memory and finds the maximum (joined over the
// cluster), pass 2 sums the exponentials from the scores, pass 3 turns them into probabilities and
// multiplies V.  All sums are exact integers, so neither the split nor the order changes a result.
//   scores: q = 256 qh + 128 + ql with s8 bytes; A holds qh in rows 0..3, ql in rows 8..11 and ones in row
//     15, keys are B columns, so one product gives qh . k, ql . k and sum(k).  4 bits: nibbles are B bytes as
//     they lie (byte j of a group holds dimensions j and j + 32), s = sum_a m_a (q . n)_a + z_a sum(q_a).
//     16 bits: k = 256 kh + 128 + kl split by byte permutes, two products.
//   context: A holds byte b of head h's weights in row 4 h + b, keys run along the product's K (four keys'
//     words are transposed in registers), dimensions are columns.  4 bits: W = P m <= 2^19 4369 < 2^32, and
//     sum_j P_j z_j apart; 16 bits: W = P, the bytes of v in separate columns.
// An item with fewer heads than NH computes the absent ones from zeros and drops them.
// Bound by instruction latency, not by memory: a tile of 32 keys and three heads is about 700 instructions of its warp,
// mostly in one dependent chain, and 7 to 16 warps on an SM (registers, ring; for want of items) keep 37 to 53% of the
// issue slots busy.  4096 sequences of 128 keys at 16 bits take 88 us (0.61 of the copy rate; 227 without the ring and
// with four warps per item), 512 of up to 512 keys at 4 bits 27, one of 65521 at 4 bits 24.
// The bounds give a thread 128 registers; with room for 24 warps per SM instead of 16 (80 registers at 4 bits and
// head_dim 64) 512 of up to 512 keys took 32.
template <int HD, int BITS, int NH, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512, WARP ? 4 : 1)
    k_paged_attention(const PagedAttnParams p, const int cs, const int part_cap, const int n_items) {
    using C = PattnCfg<HD, BITS, NH>;
    constexpr int A = C::A, S = C::STAGES;
    extern __shared__ __align__(16) uint8_t smem[];
    // each warp's part of a joined value, and (word PATTN_MAX_WARPS) the block's for its cluster; 64-bit shared
    // atomics are loops and cost 16 warps 7 us
    constexpr int PARTS = WARP ? 1 : PATTN_MAX_WARPS + 1;
    __shared__ int32_t max_s[NH][PARTS];
    __shared__ uint64_t z_s[NH][PARTS];
    __shared__ int64_t pz_s[NH * A][PARTS];
    const PagedGeom& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    int32_t* exp_s = reinterpret_cast<int32_t*>(smem);
    // block: accumulators, context, ring and temporaries of each warp, scores; warp: ring, temporaries, scores
    uint8_t* own = smem + PATTN_EXP_BYTES + (WARP ? warp * C::warp_bytes(part_cap) : 0);
    int32_t* acc_s = reinterpret_cast<int32_t*>(own);
    int64_t* ctx_s = reinterpret_cast<int64_t*>(own + C::ACC_BYTES);
    uint8_t* ring = WARP ? own : own + C::ACC_BYTES + C::CTX_BYTES + warp * C::WARP_BYTES;
    uint8_t* temp = ring + S * C::TILE;
    int16_t* score_s = reinterpret_cast<int16_t*>(WARP ? own + C::WARP_BYTES
                                                       : own + C::ACC_BYTES + C::CTX_BYTES + (blockDim.x >> 5) * C::WARP_BYTES);

    for (int i = tid; i < PATTN_EXP_BYTES / 16; i += blockDim.x) cp_async16(exp_s + 4 * i, g.exp_tab + 4 * i);
    cp_async_commit();
    if constexpr (!WARP) {
        for (int i = tid; i < C::ACC_BYTES / 16; i += blockDim.x) reinterpret_cast<int4*>(acc_s)[i] = make_int4(0, 0, 0, 0);
    }
    const int nw = blockDim.x >> 5;

    const int rank = !WARP && cs > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int head_tiles = (g.group + NH - 1) / NH;
    const int index = WARP ? blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x / cs;
    const int item = WARP ? min(index, n_items - 1) : index;
    const int ht = item % head_tiles, kv = item / head_tiles % g.n_kv, r = item / head_tiles / g.n_kv;
    const int head0 = kv * g.group + ht * NH, nh = min(NH, g.group - ht * NH);
    const int seq = p.seq ? p.seq[r] : r;
    int len = max(min(p.len[r], INT32_MAX - 1) + p.len_add, 0);
    // a padding row, or one that is refused: all threads of the item agree
    bool skip = seq < 0 || (WARP && index >= n_items);
    if (!skip && (seq >= g.n_seq || len > p.max_len ||
                  ((static_cast<int64_t>(len) + (1 << g.page_shift) - 1) >> g.page_shift) > g.ld_table)) {
        if (lane == 0) atomicCAS(g.err, 0, seq >= g.n_seq ? ERR_PAGED_SEQ : ERR_PAGED_LEN);
        skip = true;
    }
    if (skip) len = 0;
    const int me = WARP ? lane : tid, team = WARP ? 32 : blockDim.x;
    const int32_t* table = g.table + seq * g.ld_table;
    const int tiles = (len + 31) >> 5;
    const int t0 = WARP ? 0 : static_cast<int>(static_cast<int64_t>(tiles) * rank / cs);
    const int t1 = WARP ? tiles : static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / cs);
    const int stride_log2 = WARP ? 0 : 26 - __clz(blockDim.x);  // (a power of two of warps)
    const int first = WARP ? 0 : t0 + warp;
    const int n = first < t1 ? ((t1 - 1 - first) >> stride_log2) + 1 : 0;  // this warp's tiles

    // ------------------------------------------------------------ the stream of tiles: K 0..n-1, V 0..n-1 (per sweep)
    // Lane l holds the page ids of the first (l < 16) or second half of tile number ids_base + (l & 15); pages
    // hold at least 16 keys, and a half behind the last key repeats the first.
    const uint32_t page_pitch = static_cast<uint32_t>(g.slab) * g.n_kv;
    const int slot_mask = (1 << g.page_shift) - 1;
    int ids = 0, ids_base = 0, tile_i = 0, at_s = 0;  // the next tile to copy and its place in the ring
    const uint8_t* pool = g.k_pool + kv * g.slab;
    int sweep_i = -1;                                 // -1: K
    auto fetch_ids = [&]() {
        const int i = tile_i + (lane & 15), j = 32 * (first + (i << stride_log2)) + (lane & 16);
        int x = i < n && j < len ? table[j >> g.page_shift] : 0;
        const int x0 = __shfl_sync(~0u, x, lane & 15);
        if (j >= len) x = x0;
        if (x < 0 || x >= g.n_pages) {
            atomicCAS(g.err, 0, ERR_PAGED_PAGE);
            x = 0;
        }
        ids = x;
        ids_base = tile_i;
    };
    auto copy_next = [&]() {
        if (tile_i == n) {
            tile_i = 0;
            pool = g.v_pool + kv * g.slab;
            if (++sweep_i == C::SWEEPS) tile_i = n + 1;  // the stream has ended
            else if (ids_base != 0) fetch_ids();
        }
        if (tile_i < n) {
            if (tile_i == ids_base + 16) fetch_ids();
            const int key = 32 * (first + (tile_i << stride_log2));
            uint8_t* dst = ring + at_s * C::TILE;
            // 16-byte chunks of rows, 32 at a time; a row's chunk c lands in chunk c ^ f(row), against bank conflicts.  What
            // depends on the lane alone is the same for every tile, the rest are constants and the halves' slots.
            const uint8_t* half[2];
            int slot[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                slot[h] = (key + 16 * h) & slot_mask;
                half[h] = pool + static_cast<uint64_t>(static_cast<uint32_t>(__shfl_sync(~0u, ids, tile_i - ids_base + 16 * h))) * page_pitch;
            }
            constexpr int CH = C::ROW / 16, VCH = BITS == 4 ? CH : CH / C::SWEEPS;
            const uint8_t* from[2] = {half[0] + slot[0] * C::ROW, half[1] + slot[1] * C::ROW};
            if (BITS == 16 && sweep_i >= 0) {
                const int row = lane / VCH, c = lane % VCH, at = row * C::ROW + 16 * (c + VCH * sweep_i);
                uint8_t* to = dst + row * (16 * VCH) + 16 * (c ^ 2 * (row & 3));
#pragma unroll
                for (int i = 0; i < VCH; ++i)
                    cp_async16(to + i * 512, from[i >= VCH / 2] + at + (i % (VCH / 2)) * (32 / VCH * C::ROW));
            } else {
                const int row = lane / CH, c = lane % CH, at = row * C::ROW + 16 * c;
                const int f = BITS == 16 ? (row & 1) * 4 : HD == 128 ? (row >> 1 & 1) * 2 : 0;
                uint8_t* to = dst + row * C::ROW + 16 * (c ^ f);
#pragma unroll
                for (int i = 0; i < CH; ++i)
                    cp_async16(to + i * 512, from[i >= CH / 2] + at + (i % (CH / 2)) * (32 / CH * C::ROW));
            }
            if (BITS == 4 && lane < 8 * A) {
                const int h = lane >= 4 * A;
                cp_async16(dst + 32 * C::ROW + 16 * lane,
                           (h ? half[1] : half[0]) + (C::ROW << g.page_shift) + (h ? slot[1] : slot[0]) * (4 * A) + 16 * (lane - 4 * A * h));
            }
            ++tile_i;
            at_s = at_s + 1 == S ? 0 : at_s + 1;
        }
        cp_async_commit();
    };
    if (n > 0) fetch_ids();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
        if (n > 0) copy_next();
        else cp_async_commit();
    }
    cp_async_wait<S - 1>();  // the exp table
    __syncthreads();
    if (len == 0) {
        if (!skip && rank == 0)
            for (int i = me; i < nh * HD; i += team) store_context(p, r, head0 * HD + i, 0);
        return;
    }
    int use_s = 0;  // the ring's next tile to use
    // Waits for that tile, and puts the copy of a later one into the place of the tile used before.
    auto next_tile = [&]() -> const uint8_t* {
        cp_async_wait<S - 2>();
        __syncwarp();
        copy_next();
        const uint8_t* x = ring + use_s * C::TILE;
        use_s = use_s + 1 == S ? 0 : use_s + 1;
        return x;
    };

    // q fragments: step i of rows gid and gid + 8 holds dimensions 32 i + 8 tig .. + 7
    uint32_t qa[C::KS][4];
    int32_t qc[NH][A];  // sum of a head's q over each group
    {
        int32_t v[A];
#pragma unroll
        for (int a = 0; a < A; ++a) v[a] = 0;
        const int16_t* src = p.q + r * p.ldq + (head0 + min(gid, nh - 1)) * HD + 8 * tig;
        const bool vec = ((reinterpret_cast<uintptr_t>(p.q) | (p.ldq * 2)) & 15) == 0, on = gid < nh;
#pragma unroll
        for (int i = 0; i < C::KS; ++i) {
            uint4 w;
            if (vec) w = *reinterpret_cast<const uint4*>(src + 32 * i);
            else {
                const uint16_t* x = reinterpret_cast<const uint16_t*>(src + 32 * i);
                w = make_uint4(x[0] | uint32_t(x[1]) << 16, x[2] | uint32_t(x[3]) << 16, x[4] | uint32_t(x[5]) << 16,
                               x[6] | uint32_t(x[7]) << 16);
            }
            const uint32_t none = gid == 7 ? 0x01010101u : 0;
            qa[i][0] = on ? __byte_perm(w.x, w.y, 0x7531) : 0;
            qa[i][2] = on ? __byte_perm(w.z, w.w, 0x7531) : 0;
            qa[i][1] = on ? __byte_perm(w.x, w.y, 0x6420) ^ 0x80808080u : none;
            qa[i][3] = on ? __byte_perm(w.z, w.w, 0x6420) ^ 0x80808080u : none;
            // q sum = 256 sum(qh) + sum(ql) + 128 per dimension
            const int32_t hi = __dp4a(static_cast<int>(qa[i][0]), 0x01010101, __dp4a(static_cast<int>(qa[i][2]), 0x01010101, 0));
            const int32_t lo = __dp4a(static_cast<int>(qa[i][1]), 0x01010101, __dp4a(static_cast<int>(qa[i][3]), 0x01010101, 0));
            v[i >> 1] += 256 * hi + lo;
        }
#pragma unroll
        for (int a = 0; a < A; ++a) {
            v[a] += __shfl_xor_sync(~0u, v[a], 1);
            v[a] += __shfl_xor_sync(~0u, v[a], 2);
#pragma unroll
            for (int h = 0; h < NH; ++h) qc[h][a] = __shfl_sync(~0u, v[a], 4 * h) + 128 * 64;
        }
    }

    // ---------------------------------------------------------------- pass 1: scores and their maximum
    const Requant16 shift(p.shift_s, 8);  // (|scores| < 2^38 for every valid cache)
    int32_t mx[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) mx[h] = -32768;
    int16_t* my_scores = score_s + 32 * (first - t0) + lane;
    const bool keeps = gid < NH || gid == 7;  // rows of heads and the row of ones
    const int raw_row = gid < NH ? gid : NH;
    int64_t cq[NH];
    if constexpr (BITS == 16) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            int32_t s = 0;
#pragma unroll
            for (int a = 0; a < A; ++a) s += qc[h][a];
            cq[h] = static_cast<int64_t>(s) * 128 + shift.half;
        }
    }
    for (int i = 0; i < n; ++i) {
        const uint8_t* tile = next_tile();
        const int key = 32 * (first + (i << stride_log2)) + lane;
        const bool in = key < len;
        int16_t* sc = my_scores + (32 * i << stride_log2);
        if constexpr (BITS == 4) {
            int32_t* raw = reinterpret_cast<int32_t*>(temp);
#pragma unroll
            for (int a = 0; a < A; ++a)
#pragma unroll
                for (int nn = 0; nn < 4; ++nn) {
                    const int at = (8 * nn + gid) * C::ROW + (HD == 128 ? 32 * (a ^ (gid >> 1 & 1)) : 0) + 8 * tig;
                    const uint2 w = *reinterpret_cast<const uint2*>(tile + at);
                    int32_t c[4];
                    mma_s8s8_first(c, qa[2 * a], w.x & 0x0F0F0F0Fu, w.y & 0x0F0F0F0Fu);
                    mma_s8s8(c, qa[2 * a + 1], (w.x >> 4) & 0x0F0F0F0Fu, (w.y >> 4) & 0x0F0F0F0Fu);
                    // (the row of ones has zeros in its first half)
                    if (keeps)
                        *reinterpret_cast<int2*>(raw + (a * (NH + 1) + raw_row) * C::RAW_ROW + 8 * nn + 2 * tig) =
                            make_int2(c[0] * 256 + c[2], c[1] * 256 + c[3]);
                }
            __syncwarp();
            int64_t base = shift.half;
            int32_t m[A], z[A];
#pragma unroll
            for (int a = 0; a < A; ++a) {
                const uint32_t sw = *reinterpret_cast<const uint32_t*>(tile + 32 * C::ROW + 4 * (A * lane + a));
                m[a] = static_cast<int32_t>(sw & 0xFFFFu);
                z[a] = static_cast<int32_t>(sw) >> 16;
                base += static_cast<int64_t>(m[a]) * (128 * raw[(a * (NH + 1) + NH) * C::RAW_ROW + lane]);
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                int64_t acc = base;
#pragma unroll
                for (int a = 0; a < A; ++a)
                    acc += static_cast<int64_t>(m[a]) * raw[(a * (NH + 1) + h) * C::RAW_ROW + lane] + static_cast<int64_t>(z[a]) * qc[h][a];
                const int32_t s = shift(acc);
                sc[h * part_cap] = static_cast<int16_t>(s);
                mx[h] = max(mx[h], in ? s : -32768);
            }
        } else {
            int64_t* raw = reinterpret_cast<int64_t*>(temp);
#pragma unroll
            for (int nn = 0; nn < 4; ++nn) {
                int32_t ch[4], cl[4];
#pragma unroll
                for (int k = 0; k < C::KS; ++k) {
                    const uint4 w = *reinterpret_cast<const uint4*>(tile + (8 * nn + gid) * C::ROW + 16 * ((4 * k + tig) ^ (gid & 1) * 4));
                    const uint32_t h0 = __byte_perm(w.x, w.y, 0x7531), h1 = __byte_perm(w.z, w.w, 0x7531);
                    const uint32_t l0 = __byte_perm(w.x, w.y, 0x6420) ^ 0x80808080u, l1 = __byte_perm(w.z, w.w, 0x6420) ^ 0x80808080u;
                    if (k == 0) {
                        mma_s8s8_first(ch, qa[k], h0, h1);
                        mma_s8s8_first(cl, qa[k], l0, l1);
                    } else {
                        mma_s8s8(ch, qa[k], h0, h1);
                        mma_s8s8(cl, qa[k], l0, l1);
                    }
                }
                // heads: 65536 qh.kh + 256 (ql.kh + qh.kl) + ql.kl; ones: 256 sum(kh) + sum(kl)
                if (keeps)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        raw[raw_row * C::RAW_ROW + 8 * nn + 2 * tig + c] =
                            static_cast<int64_t>(ch[c]) * 65536 + (static_cast<int64_t>(ch[2 + c] + cl[c]) * 256 + cl[2 + c]);
            }
            __syncwarp();
            const int64_t ck = raw[NH * C::RAW_ROW + lane] * 128;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int32_t s = shift(raw[h * C::RAW_ROW + lane] + ck + cq[h]);
                sc[h * part_cap] = static_cast<int16_t>(s);
                mx[h] = max(mx[h], in ? s : -32768);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) mx[h] = __reduce_max_sync(~0u, mx[h]);
    if constexpr (!WARP) {
        if (lane == 0)
#pragma unroll
            for (int h = 0; h < NH; ++h) max_s[h][warp] = mx[h];
        __syncthreads();
#pragma unroll
        for (int h = 0; h < NH; ++h) mx[h] = __reduce_max_sync(~0u, lane < nw ? max_s[h][lane] : -32768);
        if (cs > 1) {
            if (tid == 0)
#pragma unroll
                for (int h = 0; h < NH; ++h) max_s[h][PATTN_MAX_WARPS] = mx[h];
            cluster_barrier();
#pragma unroll
            for (int h = 0; h < NH; ++h)
                mx[h] = __reduce_max_sync(~0u, lane < cs ? ld_remote32(remote_smem(&max_s[h][PATTN_MAX_WARPS], lane)) : -32768);
        }
    }

    // ---------------------------------------------------------------- pass 2: sum of the exponentials
    uint64_t z[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) z[h] = 0;
    for (int i = 0; i < n; ++i) {
        const bool in = 32 * (first + (i << stride_log2)) + lane < len;
        const int16_t* sc = my_scores + (32 * i << stride_log2);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const int d = in ? min(mx[h] - sc[h * part_cap], PAGED_DMAX + 1) : PAGED_DMAX + 1;
            z[h] += static_cast<uint32_t>(exp_s[d]);
        }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) z[h] = warp_sum47(z[h]);
    if constexpr (!WARP) {
        if (lane == 0)
#pragma unroll
            for (int h = 0; h < NH; ++h) z_s[h][warp] = z[h];
        __syncthreads();
#pragma unroll
        for (int h = 0; h < NH; ++h) z[h] = warp_sum47(lane < nw ? z_s[h][lane] : 0);
        if (cs > 1) {
            if (tid == 0)
#pragma unroll
                for (int h = 0; h < NH; ++h) z_s[h][PATTN_MAX_WARPS] = z[h];
            cluster_barrier();
#pragma unroll
            for (int h = 0; h < NH; ++h)
                z[h] = warp_sum47(lane < cs ? static_cast<uint64_t>(ld_remote64(remote_smem(&z_s[h][PATTN_MAX_WARPS], lane))) : 0);
        }
    }

    // ---------------------------------------------------------------- pass 3: probabilities times V
    uint32_t rcp[NH];
    {
        uint64_t d = z[0];
#pragma unroll
        for (int h = 1; h < NH; ++h) d = lane == h ? z[h] : d;
        const uint32_t q = static_cast<uint32_t>((1ull << 61) / d);
#pragma unroll
        for (int h = 0; h < NH; ++h) rcp[h] = __shfl_sync(~0u, q, h);
    }
    // key lane of a tile -> its word of a weight row, so that a thread's 8 words are keys tig + 4 i + 16 k
    uint32_t* wgt = reinterpret_cast<uint32_t*>(temp);
    uint32_t* my_wgt = wgt + 8 * (lane & 3) + 4 * (lane >> 4) + ((lane >> 2) & 3);
    const uint32_t byte_sel = (gid & 3) * 0x11 + 0x40;
    if (NH < 2 * C::RR) {  // rows of heads that are never there
        __syncwarp();
        for (int i = lane; i < C::WGT_BYTES / 4; i += 32) wgt[i] = 0;
    }
#pragma unroll 1
    for (int sweep = 0; sweep < C::SWEEPS; ++sweep) {
        int32_t acc[C::NT][4];
#pragma unroll
        for (int i = 0; i < C::NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
        int64_t pz[NH][A];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int a = 0; a < A; ++a) pz[h][a] = 0;
        for (int i = 0; i < n; ++i) {
            const uint8_t* tile = next_tile();
            const bool in = 32 * (first + (i << stride_log2)) + lane < len;
            const int16_t* sc = my_scores + (32 * i << stride_log2);
            uint32_t e[NH], pr[NH];
            bool unsure = false;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const int d = in ? min(mx[h] - sc[h * part_cap], PAGED_DMAX + 1) : PAGED_DMAX + 1;
                e[h] = static_cast<uint32_t>(exp_s[d]);
                pr[h] = prob_of(e[h], p.prob_bits, rcp[h], unsure);
            }
            if (unsure)
#pragma unroll
                for (int h = 0; h < NH; ++h) pr[h] = prob_exact(pr[h], e[h], p.prob_bits, z[h]);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int a = 0; a < A; ++a) {
                    const uint32_t sw = *reinterpret_cast<const uint32_t*>(tile + 32 * C::ROW + 4 * (A * lane + a));
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        pz[h][a] += static_cast<int64_t>(static_cast<int32_t>(pr[h])) * (static_cast<int32_t>(sw) >> 16);
                        my_wgt[(a * 2 * C::RR + h) * 32] = pr[h] * (sw & 0xFFFFu);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < NH; ++h) my_wgt[h * 32] = pr[h];
            }
            __syncwarp();
#pragma unroll
            for (int a = 0; a < C::GPS; ++a) {
                uint32_t x[4] = {0, 0, 0, 0};  // rows gid and gid + 8: one byte of eight keys' weights
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int rr = 0; rr < C::RR; ++rr) {
                        const uint4 w = *reinterpret_cast<const uint4*>(wgt + (a * 2 * C::RR + (gid >> 2) + 2 * rr) * 32 + 8 * tig + 4 * k);
                        x[rr + 2 * k] = __byte_perm(__byte_perm(w.x, w.y, byte_sel), __byte_perm(w.z, w.w, byte_sel), 0x5410);
                    }
                if constexpr (BITS == 4) {
                    uint32_t w[8], b0[4], b1[4];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int row = tig + 4 * k;  // (keys tig + 4 i and, from k = 4, 16 further on)
                        w[k] = *reinterpret_cast<const uint32_t*>(tile + row * C::ROW + (HD == 128 ? 32 * (a ^ (row >> 1 & 1)) : 0) + 4 * gid);
                    }
                    transpose4(w[0], w[1], w[2], w[3], b0);
                    transpose4(w[4], w[5], w[6], w[7], b1);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_u8u8(acc[8 * a + 2 * j], x, b0[j] & 0x0F0F0F0Fu, b1[j] & 0x0F0F0F0Fu);
                        mma_u8u8(acc[8 * a + 2 * j + 1], x, (b0[j] >> 4) & 0x0F0F0F0Fu, (b1[j] >> 4) & 0x0F0F0F0Fu);
                    }
                } else {
                    uint4 w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int row = tig + 4 * k;
                        w[k] = *reinterpret_cast<const uint4*>(tile + row * 128 + 16 * (gid ^ 2 * tig));
                    }
                    auto four = [&](int j, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t w4, uint32_t w5, uint32_t w6, uint32_t w7) {
                        uint32_t b0[4], b1[4];
                        transpose4(w0, w1, w2, w3, b0);
                        transpose4(w4, w5, w6, w7, b1);
                        mma_u8u8(acc[4 * j + 0], x, b0[0], b1[0]);
                        mma_u8s8(acc[4 * j + 1], x, b0[1], b1[1]);
                        mma_u8u8(acc[4 * j + 2], x, b0[2], b1[2]);
                        mma_u8s8(acc[4 * j + 3], x, b0[3], b1[3]);
                    };
                    four(0, w[0].x, w[1].x, w[2].x, w[3].x, w[4].x, w[5].x, w[6].x, w[7].x);
                    four(1, w[0].y, w[1].y, w[2].y, w[3].y, w[4].y, w[5].y, w[6].y, w[7].y);
                    four(2, w[0].z, w[1].z, w[2].z, w[3].z, w[4].z, w[5].z, w[6].z, w[7].z);
                    four(3, w[0].w, w[1].w, w[2].w, w[3].w, w[4].w, w[5].w, w[6].w, w[7].w);
                }
            }
        }
        // Accumulators to shared memory: word 8 i + column of row 4 h + b, joined over the block's warps (255 x
        // 255 x PATTN_MAX_PART stays in 32 bits).  Four rows are skewed by a word against bank conflicts.
        if constexpr (WARP) {
            if (sweep + 1 == C::SWEEPS) cp_async_wait<0>();  // (the ring's copies have ended; the last ones are empty)
            __syncwarp();
        }
        int32_t* warp_acc = WARP && C::SWEEPS > 1 ? nullptr : acc_s;
        if (WARP && C::SWEEPS > 1) warp_acc = reinterpret_cast<int32_t*>(score_s + NH * part_cap);
        if (n > 0) {
            int32_t* at = warp_acc + gid * C::ACC_LD + (gid >> 2) + 2 * tig;
#pragma unroll
            for (int rr = 0; rr < C::RR; ++rr)
#pragma unroll
                for (int i = 0; i < C::NT; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        int32_t* o = at + rr * (8 * C::ACC_LD + 2) + 8 * i + c;
                        if constexpr (WARP) *o = acc[i][2 * rr + c];
                        else atomicAdd(o, acc[i][2 * rr + c]);
                    }
        }
        if constexpr (BITS == 4) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int a = 0; a < A; ++a) {
                    pz[h][a] = warp_sum_signed(pz[h][a]);
                    if (!WARP && lane == 0) pz_s[h * A + a][warp] = pz[h][a];
                }
        }
        if constexpr (WARP) __syncwarp();
        else __syncthreads();
        if constexpr (BITS == 4 && !WARP) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int a = 0; a < A; ++a) pz[h][a] = warp_sum_signed(lane < nw ? pz_s[h * A + a][lane] : 0);
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            if (h >= nh) break;
            for (int d = me; d < 64 * C::GPS; d += team) {
                // 4 bits: dimension 32 k + 4 n + j of a group is column n of tile 2 j + k; 16 bits: dimension 8 n + d'
                // has its bytes in column n of tiles 2 d' and 2 d' + 1
                const int word = BITS == 4 ? 64 * (d >> 6) + 16 * (d & 3) + 8 * ((d >> 5) & 1) + ((d >> 2) & 7) : 16 * (d & 7) + (d >> 3);
                int64_t v = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    int32_t* x = warp_acc + (4 * h + b) * C::ACC_LD + h + word;
                    int64_t y = x[0];
                    if constexpr (BITS == 16) {
                        y += static_cast<int64_t>(x[8]) * 256;
                        if (!WARP && sweep + 1 < C::SWEEPS) x[0] = x[8] = 0;
                    }
                    v += y << (8 * b);
                }
                if constexpr (BITS == 4) v += A == 1 || d < 64 ? pz[h][0] : pz[h][A - 1];
                if (!WARP && cs > 1) ctx_s[h * HD + 64 * sweep + d] = v;
                else store_context(p, r, (head0 + h) * HD + 64 * sweep + d, v);
            }
        }
        if (!WARP && sweep + 1 < C::SWEEPS) __syncthreads();
        if (WARP && sweep + 1 < C::SWEEPS) __syncwarp();
    }
    if constexpr (!WARP) {
        if (cs > 1) {
            cluster_barrier();
            for (int i = rank * blockDim.x + tid; i < nh * HD; i += cs * blockDim.x) {
                int64_t v = 0;
                for (int c = 0; c < cs; ++c) v += ld_remote64(remote_smem(ctx_s + i, c));
                store_context(p, r, head0 * HD + i, v);
            }
            cluster_barrier();  // no block leaves while its words are read
        }
    }
}

}  // namespace eii
