// C ABI of the paged K/V cache (eii_paged_*): argument checks, handle, launches.
#include <cuda_runtime.h>

#include <cstdint>
#include <new>
#include <vector>

#include "eii.h"
#include "eii_host.h"
#include "eii_paged.cuh"
#include "eii_paged.h"

using namespace eii;

struct eii_paged {
    int device = 0, num_sms = 0;
    int n_heads = 0, n_kv = 0, hd = 0, page_shift = 0, bits = 0, n_pos = 0;
    int32_t *exp_tab = nullptr, *rope_c = nullptr, *rope_s = nullptr;
    int* err = nullptr;
    uint8_t* mem = nullptr;  // the four above, one allocation
};

namespace {

int64_t slab_bytes(const eii_paged* p) {
    return static_cast<int64_t>(paged_row_bytes(p->hd, p->bits)) << p->page_shift;
}

int check_pages(const eii_pages* pg) {
    if (!pg) return fail(EII_ERR_ARG, "pages is null");
    if (!pg->k_pool || !pg->v_pool || !pg->table) return fail(EII_ERR_ARG, "a pool or the page table is null");
    if ((reinterpret_cast<uintptr_t>(pg->k_pool) | reinterpret_cast<uintptr_t>(pg->v_pool)) & 15)
        return fail(EII_ERR_ARG, "the pools must be 16-byte aligned");
    TRY(check_aligned("table", pg->table, 4));
    if (pg->n_pages < 1 || pg->n_pages > INT32_MAX)
        return fail(EII_ERR_ARG, "n_pages must be in [1, 2^31) (got %lld)", (long long)pg->n_pages);
    if (pg->n_seq < 1) return fail(EII_ERR_ARG, "n_seq must be >= 1 (got %d)", pg->n_seq);
    if (pg->ld_table < 1) return fail(EII_ERR_ARG, "ld_table must be >= 1 (got %lld)", (long long)pg->ld_table);
    return EII_OK;
}

PagedGeom geometry(const eii_paged* p, const eii_pages* pg) {
    PagedGeom g{};
    g.n_heads = p->n_heads; g.n_kv = p->n_kv; g.hd = p->hd; g.group = p->n_heads / p->n_kv;
    g.page_shift = p->page_shift; g.bits = p->bits; g.slab = slab_bytes(p);
    g.k_pool = static_cast<uint8_t*>(pg->k_pool); g.v_pool = static_cast<uint8_t*>(pg->v_pool);
    g.n_pages = pg->n_pages; g.table = pg->table; g.ld_table = pg->ld_table; g.n_seq = pg->n_seq;
    g.exp_tab = p->exp_tab; g.err = p->err;
    return g;
}

int check_shift(const char* name, int s) {
    if (s < 1 || s > 62) return fail(EII_ERR_ARG, "%s must be in [1, 62] (got %d)", name, s);
    return EII_OK;
}

int check_ld(const char* name, int64_t ld, int64_t least) {
    if (ld < least) return fail(EII_ERR_ARG, "%s must be >= %lld (got %lld)", name, (long long)least, (long long)ld);
    return EII_OK;
}

// Launches in clusters of `cs` blocks and returns this launch's own status (cudaGetLastError may hold an earlier call's).
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), int64_t grid, int block, size_t smem, int cs, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.stream = st;
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cs;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

template <int HD, int BITS>
int launch_append(const AppendParams& ap, int in_bits, int num_sms, cudaStream_t st) {
    // one warp per row, more while that leaves the SMs short of warps and there are heads to share
    constexpr int at_once = AppendLanes<HD>::HEADS;
    const int steps = (ap.q ? (ap.g.n_heads + at_once - 1) / at_once : 0) + 2 * ((ap.g.n_kv + at_once - 1) / at_once);
    int wpr = 1;
    while (wpr < steps && static_cast<int64_t>(ap.n_rows) * wpr < 32 * num_sms) ++wpr;
    const int64_t blocks = (static_cast<int64_t>(ap.n_rows) * wpr + 7) / 8;
    if (blocks > INT32_MAX) return fail(EII_ERR_ARG, "n_rows %d is too large", ap.n_rows);
    const int64_t e = in_bits / 8;
    const uintptr_t in = reinterpret_cast<uintptr_t>(ap.q) | reinterpret_cast<uintptr_t>(ap.k) | reinterpret_cast<uintptr_t>(ap.v) |
                         static_cast<uintptr_t>((ap.q ? ap.ldq : 0) * e | ap.ldk * e | ap.ldv * e);
    const int vec_in = (in & (4 * e - 1)) == 0;
    const int vec_out = (((reinterpret_cast<uintptr_t>(ap.q_out) | static_cast<uintptr_t>(ap.ldqo * 2)) & 7) == 0) |
                        ((reinterpret_cast<uintptr_t>(ap.kv_out) & 15) == 0) << 1;
    if (in_bits == 16) CK(launch(k_paged_append<HD, BITS, int16_t>, blocks, 256, 0, 1, st, ap, wpr, vec_in, vec_out));
    else CK(launch(k_paged_append<HD, BITS, int32_t>, blocks, 256, 0, 1, st, ap, wpr, vec_in, vec_out));
    return EII_OK;
}

constexpr int kSmemOptin = 224 * 1024;  // dynamic shared memory of one block beside the static words

// How the work of one attention call is laid out.
struct AttnShape {
    bool warp;      // one warp per item
    int warps, cs;  // warps per block, blocks per cluster
};

// Measured in captured graphs (sequences x keys, 9 query heads on 3 kv heads, head_dim 64, 4 bits unless said, us):
//  - one warp per item once items fill the SMs and none is long: 4096 x 128 keys 58 (two warps per item 90,
//    eight 193), at 16 bits 88 (140), 512 x 512 at 16 bits 46 (four 60), 400 x 1000 45.8 (four 39.9).  A warp's fixed
//    cost is about two tiles' work.  At 16 bits and head_dim 128 the warps' rings (8 KB a tile) leave few on an SM:
//    1000 x 64 of 32 heads on 8 96 (two warps 142), x 128 221 (194), 160 x 500 142 (99).
//  - otherwise as few warps per block as give eight warps per SM, two at least and from 17 tiles on four: 64 x 512 9.5
//    with eight (four 10.6), 200 x 512 17.3 with two (four 19.7, eight 23.2), 160 x 1000 of 32 heads on 8 of head_dim
//    128 83 with four (two 100, eight 94);
//  - for longer items blocks of four warps, of which more fit an SM, where clusters of eight reach that: 64 x 4096
//    31.1 (eight warps 34.4), at 16 bits 46.6 (63.5), 512 x 2000 92.6 (107.5), 16 x 16384 32.0 (36.6); eight warps for
//    fewer items and for head_dim 128: 64 x 4096 of 32 heads on 8 119 (four 146);
//  - clusters until there are eight warps per SM, as long as a warp keeps two tiles: 8 x 4096 13.1 with eight blocks
//    (sixteen 25.5), 8 x 32768 37 (of sixteen warps 46); and until a block's scores (nh int16 per key) leave room for a second
//    block on the SM: 128 rows x 6000 keys of 32 heads on 8 of head_dim 128 271 with two blocks, 370 with one;
//  - sixteen warps for the longest of a few sequences: 1 x 65521 24 (eight 27), at 16 bits 30 (35), 2 x 65521 27 (31);
//    not with two tiles a warp: 1 x 16384 of 32 heads on 8 of head_dim 128 44 (eight 27).
AttnShape attn_shape(int64_t items, int tiles, int nh, int hd, int bits, int sms) {
    const int64_t enough = 8 * static_cast<int64_t>(sms);
    if (tiles <= (hd == 128 && bits == 16 ? 3 : 16) && items >= enough) return {true, 4, 1};
    int warps = 1, cs = 1;
    while (warps < 8 && warps < tiles) warps *= 2;
    if (tiles <= 32) {
        const int least = tiles <= 16 ? 2 : 4;
        while (warps > least && items * (warps / 2) >= enough) warps /= 2;
    } else if (hd == 64 && items * 8 * 4 >= enough) {
        warps = 4;
    }
    while (cs < PATTN_MAX_CLUSTER &&
           ((tiles + cs - 1) / cs * 32 > PATTN_MAX_PART || (items * cs * warps < enough && 4 * cs * warps <= tiles) ||
            (cs < 4 && nh * ((tiles + cs - 1) / cs) > 600)))
        cs *= 2;
    if (cs >= 8 && items * cs <= sms && 8 * cs * warps <= tiles) warps = 16;
    return {false, warps, cs};
}

int attn_tiles(const PagedAttnParams& ap) { return ap.max_len > 0 ? (ap.max_len + 31) / 32 : 1; }
int64_t attn_items(const PagedAttnParams& ap, int nh) {
    return static_cast<int64_t>(ap.n_rows) * ap.g.n_kv * ((ap.g.group + nh - 1) / nh);
}

// Query heads of one item.  All that share a kv head (up to four) take its keys apart once; but where the blocks of
// items with one or two heads leave SMs idle all the same, a block with less to do is done sooner.  Measured as above,
// one, two and three heads: 1 x 200 keys 5.4, 6.0, 7.0 (at 16 bits 6.6, 7.0, 7.8), 16 x 512 6.4, 7.5, 8.4, 1 x 4096
// 8.4, 9.3, 10.5; but with more blocks than SMs 8 x 4096 20.6, 14.7, 13.1; from 17 tiles on two thirds of the SMs
// are as much as pays, as clusters have to fit: 16 x 1000 at 16 bits 14.9, 12.9, 12.1.
int attn_heads(const PagedAttnParams& ap, int hd, int bits, int sms) {
    const int most = ap.g.group < PATTN_MAX_HEADS ? ap.g.group : PATTN_MAX_HEADS, tiles = attn_tiles(ap);
    for (int nh = 1; nh <= 2 && nh < most; ++nh) {
        const AttnShape s = attn_shape(attn_items(ap, nh), tiles, nh, hd, bits, sms);
        const int64_t blocks = attn_items(ap, nh) * s.cs;
        if (!s.warp && (tiles <= 16 ? blocks <= sms : 3 * blocks <= 2 * sms)) return nh;
    }
    return most;
}

template <int HD, int BITS, int NH>
int launch_attention_nh(const eii_paged* p, const PagedAttnParams& ap, cudaStream_t st) {
    using C = PattnCfg<HD, BITS, NH>;
    const int tiles = attn_tiles(ap);
    const int64_t items = attn_items(ap, NH);
    if (items > INT32_MAX / PATTN_MAX_CLUSTER) return fail(EII_ERR_ARG, "n_rows %d is too large", ap.n_rows);
    AttnShape s = attn_shape(items, tiles, NH, HD, BITS, p->num_sms);
    if (s.warp) {
        CK(launch(k_paged_attention<HD, BITS, NH, true>, (items + s.warps - 1) / s.warps, 32 * s.warps,
                  C::smem_warp(s.warps, tiles * 32), 1, st, ap, 1, tiles * 32, static_cast<int>(items)));
        return EII_OK;
    }
    const int part = (tiles + s.cs - 1) / s.cs * 32;
    if (C::smem_block(s.warps, part) > kSmemOptin) s.warps = 8;
    CK(launch(k_paged_attention<HD, BITS, NH, false>, items * s.cs, 32 * s.warps, C::smem_block(s.warps, part), s.cs, st, ap,
              s.cs, part, static_cast<int>(items)));
    return EII_OK;
}

template <int HD, int BITS>
int launch_attention(const eii_paged* p, const PagedAttnParams& ap, cudaStream_t st) {
    switch (attn_heads(ap, HD, BITS, p->num_sms)) {
        case 1: return launch_attention_nh<HD, BITS, 1>(p, ap, st);
        case 2: return launch_attention_nh<HD, BITS, 2>(p, ap, st);
        case 3: return launch_attention_nh<HD, BITS, 3>(p, ap, st);
    }
    return launch_attention_nh<HD, BITS, 4>(p, ap, st);
}

// Once per handle: the attention kernels' shared memory and cluster limits on the current device.
template <int HD, int BITS, int NH>
int allow_attention() {
    static_assert(PattnCfg<HD, BITS, NH>::smem_block(8, PATTN_MAX_PART) <= kSmemOptin && PattnCfg<HD, BITS, NH>::smem_warp(4, 1024) <= kSmemOptin, "shared memory");
    CK(cudaFuncSetAttribute(k_paged_attention<HD, BITS, NH, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOptin));
    CK(cudaFuncSetAttribute(k_paged_attention<HD, BITS, NH, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemOptin));
    CK(cudaFuncSetAttribute(k_paged_attention<HD, BITS, NH, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return EII_OK;
}
template <int HD, int BITS>
int allow_attention() {
    TRY((allow_attention<HD, BITS, 1>()));
    TRY((allow_attention<HD, BITS, 2>()));
    TRY((allow_attention<HD, BITS, 3>()));
    return allow_attention<HD, BITS, 4>();
}

}  // namespace

extern "C" {

int eii_paged_open(int device, int n_heads, int n_kv, int head_dim, int page_size, int cache_bits, int n_pos,
                   const int64_t* rope_cos, const int64_t* rope_sin, eii_paged** out) {
    if (!out) return fail(EII_ERR_ARG, "out is null");
    *out = nullptr;
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv != 0 || n_heads > 1024)
        return fail(EII_ERR_ARG, "n_heads must be a multiple of n_kv in [1, 1024] (got %d and %d)", n_heads, n_kv);
    if (head_dim != 64 && head_dim != 128) return fail(EII_ERR_ARG, "head_dim must be 64 or 128 (got %d)", head_dim);
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
        return fail(EII_ERR_ARG, "page_size must be a power of two in [16, 1024] (got %d)", page_size);
    if (cache_bits != 4 && cache_bits != 16) return fail(EII_ERR_ARG, "cache_bits must be 4 or 16 (got %d)", cache_bits);
    if (n_pos < 1 || n_pos > EII_PAGED_MAX_LEN)
        return fail(EII_ERR_ARG, "n_pos must be in [1, %d] (got %d)", EII_PAGED_MAX_LEN, n_pos);
    if (!rope_cos != !rope_sin) return fail(EII_ERR_ARG, "rope_cos and rope_sin come together");
    if (!rope_cos && head_dim != 64)
        return fail(EII_ERR_ARG, "head_dim %d needs rope tables (they are generated for head_dim 64 only)", head_dim);
    const size_t n = static_cast<size_t>(n_pos) * (head_dim / 2);
    std::vector<int64_t> e, c, s;
    std::vector<int32_t> h;
    try {
        e.resize(PAGED_DMAX + 1);
        if (!rope_cos) {
            c.resize(n);
            s.resize(n);
            TRY(eii_table_rope(n_pos, c.data(), s.data()));
            rope_cos = c.data();
            rope_sin = s.data();
        }
        h.resize(PATTN_EXP_BYTES / 4 + 2 * n);  // (zeros behind the exp table)
    } catch (const std::bad_alloc&) {
        return fail(EII_ERR_ARG, "out of host memory for %d positions", n_pos);
    }
    TRY(eii_table_exp(e.data()));
    for (int i = 0; i <= PAGED_DMAX; ++i) h[i] = static_cast<int32_t>(e[i]);
    for (size_t i = 0; i < n; ++i) {
        const int64_t one = int64_t(1) << 30;
        if (rope_cos[i] < -one || rope_cos[i] > one || rope_sin[i] < -one || rope_sin[i] > one)
            return fail(EII_ERR_ARG, "rope table entry %zu lies outside [-2^30, 2^30]", i);
        h[PATTN_EXP_BYTES / 4 + i] = static_cast<int32_t>(rope_cos[i]);
        h[PATTN_EXP_BYTES / 4 + n + i] = static_cast<int32_t>(rope_sin[i]);
    }
    TRY(check_device(device));
    DeviceGuard dg(device);
    CK(dg.st);
    eii_paged* p = new (std::nothrow) eii_paged;
    if (!p) return fail(EII_ERR_ARG, "out of host memory");
    p->device = device;
    p->n_heads = n_heads; p->n_kv = n_kv; p->hd = head_dim; p->bits = cache_bits; p->n_pos = n_pos;
    while ((1 << p->page_shift) < page_size) ++p->page_shift;
    const size_t exp_bytes = PATTN_EXP_BYTES, rope_bytes = n * 4;  // rope rows stay 16-byte aligned
    int rc = EII_OK;
    if (cudaDeviceGetAttribute(&p->num_sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaMalloc(&p->mem, exp_bytes + 2 * rope_bytes + 16) != cudaSuccess)
        rc = fail(EII_ERR_CUDA, "device memory for the cache's tables: %s", cudaGetErrorString(cudaGetLastError()));
    if (rc == EII_OK) {
        p->exp_tab = reinterpret_cast<int32_t*>(p->mem);
        p->rope_c = reinterpret_cast<int32_t*>(p->mem + exp_bytes);
        p->rope_s = reinterpret_cast<int32_t*>(p->mem + exp_bytes + rope_bytes);
        p->err = reinterpret_cast<int*>(p->mem + exp_bytes + 2 * rope_bytes);
        // (a copy from pageable memory and a memset may return before they are done, and a stream that does not wait
        // for the default stream may have the first call)
        if (cudaMemcpy(p->mem, h.data(), exp_bytes + 2 * rope_bytes, cudaMemcpyHostToDevice) != cudaSuccess ||
            cudaMemset(p->err, 0, sizeof(int)) != cudaSuccess || cudaStreamSynchronize(nullptr) != cudaSuccess)
            rc = fail(EII_ERR_CUDA, "table upload failed: %s", cudaGetErrorString(cudaGetLastError()));
    }
    if (rc == EII_OK && head_dim == 64) rc = cache_bits == 4 ? allow_attention<64, 4>() : allow_attention<64, 16>();
    else if (rc == EII_OK) rc = cache_bits == 4 ? allow_attention<128, 4>() : allow_attention<128, 16>();
    if (rc != EII_OK) {
        cudaFree(p->mem);
        delete p;
        return rc;
    }
    *out = p;
    return EII_OK;
}

int64_t eii_paged_pool_bytes(const eii_paged* p, int64_t n_pages) {
    if (!p) return -static_cast<int64_t>(fail(EII_ERR_ARG, "cache is null"));
    if (n_pages < 1 || n_pages > INT32_MAX)
        return -static_cast<int64_t>(fail(EII_ERR_ARG, "n_pages must be in [1, 2^31) (got %lld)", (long long)n_pages));
    return n_pages * p->n_kv * slab_bytes(p);
}

int eii_paged_append(eii_paged* p, const eii_pages* pages, const void* q, int64_t ldq, const void* k, int64_t ldk,
                     const void* v, int64_t ldv, int in_bits, int n_rows, const int32_t* seq, const int32_t* pos,
                     int shift_q, int shift_k, int16_t* q_out, int64_t ldqo, int32_t* kv_out, void* stream) {
    if (!p) return fail(EII_ERR_ARG, "cache is null");
    if (n_rows < 0) return fail(EII_ERR_ARG, "n_rows must be >= 0 (got %d)", n_rows);
    if (n_rows == 0) return EII_OK;
    TRY(check_pages(pages));
    if (!k || !v || !pos) return fail(EII_ERR_ARG, "k, v or pos is null");
    if (!q != !q_out) return fail(EII_ERR_ARG, "q and q_out come together");
    if (in_bits != 16 && in_bits != 32) return fail(EII_ERR_ARG, "in_bits must be 16 or 32 (got %d)", in_bits);
    if (!seq && n_rows > pages->n_seq)
        return fail(EII_ERR_ARG, "%d rows without sequence indices but %d sequences", n_rows, pages->n_seq);
    TRY(check_ld("ldk", ldk, (int64_t)p->n_kv * p->hd));
    TRY(check_ld("ldv", ldv, (int64_t)p->n_kv * p->hd));
    if (q) {
        TRY(check_ld("ldq", ldq, (int64_t)p->n_heads * p->hd));
        TRY(check_ld("ldqo", ldqo, (int64_t)p->n_heads * p->hd));
        TRY(check_shift("shift_q", shift_q));
    }
    TRY(check_shift("shift_k", shift_k));
    const uintptr_t in = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    if (in & (in_bits / 8 - 1)) return fail(EII_ERR_ARG, "q, k and v must be aligned to their elements");
    TRY(check_aligned("seq", seq, 4));
    TRY(check_aligned("pos", pos, 4));
    TRY(check_aligned("q_out", q_out, 2));
    TRY(check_aligned("kv_out", kv_out, 4));
    DeviceGuard dg(p->device);
    CK(dg.st);
    AppendParams ap{};
    ap.g = geometry(p, pages);
    ap.q = q; ap.k = k; ap.v = v; ap.ldq = ldq; ap.ldk = ldk; ap.ldv = ldv; ap.n_rows = n_rows; ap.seq = seq; ap.pos = pos;
    ap.rope_c = p->rope_c; ap.rope_s = p->rope_s; ap.n_pos = p->n_pos; ap.shift_q = shift_q; ap.shift_k = shift_k;
    ap.q_out = q_out; ap.ldqo = ldqo; ap.kv_out = kv_out;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->hd == 64) return p->bits == 4 ? launch_append<64, 4>(ap, in_bits, p->num_sms, st)
                                          : launch_append<64, 16>(ap, in_bits, p->num_sms, st);
    return p->bits == 4 ? launch_append<128, 4>(ap, in_bits, p->num_sms, st) : launch_append<128, 16>(ap, in_bits, p->num_sms, st);
}

static int attention(eii_paged* p, const PagedAttnParams& ap, cudaStream_t st) {
    if (p->hd == 64) return p->bits == 4 ? launch_attention<64, 4>(p, ap, st) : launch_attention<64, 16>(p, ap, st);
    return p->bits == 4 ? launch_attention<128, 4>(p, ap, st) : launch_attention<128, 16>(p, ap, st);
}

int eii_paged_attention(eii_paged* p, const eii_pages* pages, const int16_t* q, int64_t ldq, int n_rows,
                        const int32_t* seq, const int32_t* len, int max_len, int shift_s, int prob_bits, int shift_c,
                        int bits_c, int32_t* ctx, int64_t ldc, void* stream) {
    if (!p) return fail(EII_ERR_ARG, "cache is null");
    if (n_rows < 0) return fail(EII_ERR_ARG, "n_rows must be >= 0 (got %d)", n_rows);
    if (n_rows == 0) return EII_OK;
    TRY(check_pages(pages));
    if (!q || !len || !ctx) return fail(EII_ERR_ARG, "q, len or ctx is null");
    if (!seq && n_rows > pages->n_seq)
        return fail(EII_ERR_ARG, "%d rows without sequence indices but %d sequences", n_rows, pages->n_seq);
    if (max_len < 0 || max_len > EII_PAGED_MAX_LEN)
        return fail(EII_ERR_ARG, "max_len must be in [0, %d] (got %d)", EII_PAGED_MAX_LEN, max_len);
    TRY(check_ld("ldq", ldq, (int64_t)p->n_heads * p->hd));
    TRY(check_ld("ldc", ldc, (int64_t)p->n_heads * p->hd));
    TRY(check_shift("shift_s", shift_s));
    if (shift_c < -16 || shift_c > 62) return fail(EII_ERR_ARG, "shift_c must be in [-16, 62] (got %d)", shift_c);
    if (prob_bits < 16 || prob_bits > 19) return fail(EII_ERR_ARG, "prob_bits must be in [16, 19] (got %d)", prob_bits);
    if (bits_c < 2 || bits_c > 32) return fail(EII_ERR_ARG, "bits_c must be in [2, 32] (got %d)", bits_c);
    if ((reinterpret_cast<uintptr_t>(q) & 1) || (reinterpret_cast<uintptr_t>(ctx) & 3))
        return fail(EII_ERR_ARG, "q and ctx must be aligned to their elements");
    TRY(check_aligned("seq", seq, 4));
    TRY(check_aligned("len", len, 4));
    DeviceGuard dg(p->device);
    CK(dg.st);
    PagedAttnParams ap{};
    ap.g = geometry(p, pages);
    ap.q = q; ap.ldq = ldq; ap.n_rows = n_rows; ap.seq = seq; ap.len = len; ap.max_len = max_len;
    ap.shift_s = shift_s; ap.prob_bits = prob_bits; ap.shift_c = shift_c; ap.bits_c = bits_c; ap.ctx = ctx; ap.ldc = ldc;
    return attention(p, ap, static_cast<cudaStream_t>(stream));
}

int eii_paged_sync(eii_paged* p, void* stream) {
    if (!p) return fail(EII_ERR_ARG, "cache is null");
    DeviceGuard dg(p->device);
    CK(dg.st);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int code = 0;
    CK(cudaMemcpyAsync(&code, p->err, sizeof(int), cudaMemcpyDeviceToHost, st));
    CK(cudaStreamSynchronize(st));
    if (!code) return EII_OK;
    CK(cudaMemsetAsync(p->err, 0, sizeof(int), st));
    CK(cudaStreamSynchronize(st));
    switch (code) {
        case ERR_PAGED_SEQ: return fail(EII_ERR_ARG, "a row's sequence index is not below n_seq");
        case ERR_PAGED_POS: return fail(EII_ERR_ARG, "a row's position lies outside the rope table or the page table");
        case ERR_PAGED_PAGE: return fail(EII_ERR_ARG, "the page table names a page outside [0, n_pages)");
        case ERR_PAGED_LEN: return fail(EII_ERR_ARG, "a row's length exceeds max_len or the page table");
        case ERR_PAGED_INPUT: return fail(EII_ERR_ARG, "a q, k or v value lies outside the int16 range");
    }
    return fail(EII_ERR_DEVICE, "kernel reported error %d", code);
}

}  // extern "C"

int eii::paged_attention_planes(eii_paged* p, const eii_pages& pages, const int16_t* q, int n_rows, const int32_t* seq,
                                const int32_t* pos, int max_len, int shift_s, int shift_c, int bits_c, uint8_t* planes,
                                int n_planes, int offset, cudaStream_t st) {
    PagedAttnParams ap{};
    ap.g = geometry(p, &pages);
    ap.q = q; ap.ldq = p->n_heads * p->hd; ap.n_rows = n_rows; ap.seq = seq; ap.len = pos; ap.len_add = 1; ap.max_len = max_len;
    ap.shift_s = shift_s; ap.prob_bits = 16; ap.shift_c = shift_c; ap.bits_c = bits_c;
    ap.planes = planes; ap.n_planes = n_planes; ap.offset = offset;
    return attention(p, ap, st);
}

extern "C" {

void eii_paged_close(eii_paged* p) {
    if (!p) return;
    DeviceGuard dg(p->device);
    cudaFree(p->mem);
    delete p;
}

}  // extern "C"
