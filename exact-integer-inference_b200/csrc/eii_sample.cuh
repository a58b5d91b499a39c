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

#include <type_traits>

#include "eii_cluster.cuh"
#include "eii_int.cuh"

namespace eii {

constexpr uint32_t SAMPLE_C1 = 744163075, SAMPLE_C2 = 257059888, SAMPLE_C3 = 57045411, SAMPLE_C4 = 7277686;
constexpr int64_t SAMPLE_LOG2E_Q24 = 24204406;
constexpr int32_t SAMPLE_MASKED = INT32_MIN;
constexpr int SAMPLE_MAX_VOCAB = 262144;  // 2^18 weights of at most 2^30: sums are at most 2^48
constexpr int32_t SAMPLE_MAX_INV_TEMP = 1 << 22;
constexpr int SAMPLE_MAX_ROWS = 1 << 30;

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

// A row's weights.
struct SampleScale {
    uint32_t row_max, b2;
    // The polynomial runs on the double-precision pipe, the integer one being what bounds the kernel: u = f 2^-24
    // exactly, and y u + 2^52 rounded down is 2^52 + floor(y u) for every y below 2^30 (one rounding, at the units'
    // place).  RS(y, n) = ((2 y >> n) + 1) >> 1.
    template <bool CHECK>
    __device__ __forceinline__ uint32_t at_distance(uint32_t d) const {
        const uint64_t x = static_cast<uint64_t>(d) * b2;
        const uint32_t hi = static_cast<uint32_t>(x >> 32), lo = static_cast<uint32_t>(x);
        constexpr double M = 4503599627370496.0;  // 2^52
        const double u = __hiloint2double(static_cast<int>((__funnelshift_r(lo, hi, 20) & 0xFFFFFu) | 0x3FF00000u),
                                          static_cast<int>((lo << 12) & 0xF0000000u)) - 1.0;
        double y = (M + SAMPLE_C3) - __fma_rd(static_cast<double>(SAMPLE_C4), u, M);
        y = (M + SAMPLE_C2) - __fma_rd(y, u, M);
        y = (M + SAMPLE_C1) - __fma_rd(y, u, M);
        const uint32_t k = static_cast<uint32_t>(__double2loint(__fma_rd(y, u, M)));
        const uint32_t w = (__funnelshift_rc((1u << 31) - 2 * k, 0, hi >> 8) + 1) >> 1;
        return !CHECK || hi < (31u << 8) ? w : 0;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t logit) const {
        return logit != static_cast<uint32_t>(SAMPLE_MASKED) ? at_distance<true>(row_max - logit) : 0;
    }
    // Whether at_distance<false> gives every logit's weight: from 32 octaves on the shift leaves nothing, in the
    // 31st it leaves something for f = 0 only; so masked logits have to be 32 octaves away, and no distance may
    // hit that place (at most one can, for b2 > 2^16).  The comparisons would be a quarter of a weight's cost.
    __device__ bool plain() const {
        constexpr uint64_t edge = 31ull << 40;
        if (b2 <= 1u << 16 || static_cast<uint64_t>(row_max - static_cast<uint32_t>(SAMPLE_MASKED)) * b2 < 32ull << 40) return false;
        const uint32_t d = static_cast<uint32_t>(static_cast<double>(edge) / b2);
        bool hit = false;
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) hit |= static_cast<uint64_t>(d + i - 1) * b2 - edge < 1u << 16;
        return !hit;
    }
};

// ceil(p mass / 2^16), at least 1.
__device__ __forceinline__ uint64_t sample_goal(uint64_t mass, int p) {
    const uint64_t g = p * (mass >> 16) + ((p * (mass & 0xFFFF) + 0xFFFF) >> 16);
    return g ? g : 1;
}
// floor(u mass / 2^32).
__device__ __forceinline__ uint64_t sample_target(uint64_t mass, uint32_t u) {
    return (u * (mass >> 24) + ((u * (mass & 0xFFFFFF)) >> 24)) >> 8;
}

// ------------------------------------------------------------------------------------------ kernel
// A cluster of `cs` blocks per row, the row's weights in shared memory from the one time it is read: a thread
// owns 4 ch consecutive ones (index order is block, thread, chunk of four, word).  The grid is persistent.
//
// The kept tokens are a prefix of the order (weight descending, index ascending): all weights above theta
// and the first `quota` of those equal to it.  A cut is found by narrowing a window [lo, hi) around it:
// with passes over the row, the first at places that a sample of the row suggests, until the window is
// short enough for a list; with passes over that list; and, from SAMPLE_FEW on, by comparing each with all.
// Every decision rests on exact sums; the sample only chooses where to look.  Each thread knows the mass of
// its own weights above the window, and its entries of the list are contiguous, so the draw needs no
// further pass: a row is read for its maximum, for the weights, and once or twice for the cut.
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_MAX_CHUNKS = 12;  // clusters of at most eight: 8 x 12 x 4096 logits
constexpr int SAMPLE_GUESS_CHUNKS = 6;
constexpr int SAMPLE_LIST = 8192, SAMPLE_FEW = 64;
constexpr uint32_t SAMPLE_TOP = (1u << 30) + 1;  // above every weight

// Words that are exchanged come in two sets that take turns, so that one is not overwritten before its slowest
// reader has it: between two uses of a set lies another exchange, whose barrier the reader reaches after
// its reads.  The words of a block's threads (warp_*) and those of a cluster's blocks (block_*) take turns apart: a
// block barrier does not hold back the other blocks, so an exchange within a block must not turn the cluster's sets.
struct SampleTurns {
    int block = 0, cluster = 0;
    __host__ __device__ __forceinline__ int next_block() { return block ^= 1; }
    __host__ __device__ __forceinline__ int next_cluster() { return cluster ^= 1; }
};
struct SampleShared {
    uint32_t w[SAMPLE_LIST];  // the list; of a cluster's blocks the first half, the second for all
    uint32_t few[SAMPLE_FEW];
    int32_t warp_max[2][SAMPLE_WARPS];
    uint64_t warp_mass[2][SAMPLE_WARPS];
    uint32_t warp_n[2][SAMPLE_WARPS];
    int32_t block_max[2];
    uint64_t block_mass[2];
    uint32_t block_n[2];
    uint32_t few_n, theta, above_n;
    uint64_t above;
};
static_assert(SAMPLE_MAX_CHUNKS * 16 * SAMPLE_THREADS + sizeof(SampleShared) <= 227 * 1024, "shared memory");

// Bound by one row at a time on an SM (its weights fill the shared memory): no other block has work while this one waits
// at its barriers and searches its list.  Of 49,000 cycles of a row of 49152 (top-p) the weights take about 14,000, each
// of two passes 5,000, the sample 6,000, the list and its search 12,000; over all of them 63% of the issue slots
// and 55% of the integer pipe are busy, with a small top-k 49% and 32%.  4096 such rows take 858 us, 0.94 TB/s of the
// 6.5 that a copy reaches.  The weights in registers instead of shared memory (96 per thread, 512 threads) took
// 1,600 us: unrolled code and spills.
__global__ void __launch_bounds__(SAMPLE_THREADS, 1) k_sample(const SampleParams p, const int cs, const int ch, const int aligned) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem + ch * 16 * SAMPLE_THREADS);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cs > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int base = (rank * SAMPLE_THREADS + tid) * 4 * ch;  // this thread's first logit
    const int step = gridDim.x / cs;
    uint4* warp_buf = reinterpret_cast<uint4*>(smem) + warp * 32 * ch;
    uint4* buf = warp_buf + lane * ch;
    // A thread goes through its chunks from one that depends on its lane on, so that where ch is even eight
    // neighbours read from eight banks.
    int start = ch & 1 ? 0 : lane & 7;
    while (start >= ch) start -= ch;
    SampleTurns turns;

    // f(number of a chunk, the chunk) over this thread's chunks
    auto each = [&](auto f) {
        int k = start;
#pragma unroll 4
        for (int i = 0; i < ch; ++i) {
            f(k, buf + k);
            k = k + 1 == ch ? 0 : k + 1;
        }
    };
    // this warp's part of row r to shared memory, masked behind the row's end
    const int first = base - lane * 4 * ch;  // the warp's first logit
    const bool whole = aligned && p.vocab - first >= 128 * ch;
    auto copy = [&](int r) {
        if (r < p.n_rows) {
            const int32_t* row = p.logits + r * p.ld + first;
            if (whole) {
#pragma unroll 4
                for (int c = lane; c < 32 * ch; c += 32) cp_async16(warp_buf + c, row + 4 * c);
            } else {
                for (int c = lane; c < 32 * ch; c += 32) {
                    const int left = p.vocab - first - 4 * c;
                    if (aligned && left >= 4) cp_async16(warp_buf + c, row + 4 * c);
                    else
                        for (int j = 0; j < 4; ++j) {
                            if (j < left) cp_async4(reinterpret_cast<uint32_t*>(warp_buf + c) + j, row + 4 * c + j);
                            else reinterpret_cast<int32_t*>(warp_buf + c)[j] = SAMPLE_MASKED;
                        }
                }
            }
        }
        cp_async_commit();
    };
    // sums over the threads of the block's first `warps` warps, in every thread
    auto total = [&](uint64_t& m, uint32_t& n, int warps) {
        const int turn = turns.next_block();
        if (warp < warps) {
            m = warp_sum47(m);
            n = __reduce_add_sync(~0u, n);
            if (lane == 0) {
                sh.warp_mass[turn][warp] = m;
                sh.warp_n[turn][warp] = n;
            }
        }
        __syncthreads();
        m = warp_sum47(lane < warps ? sh.warp_mass[turn][lane] : 0);
        n = __reduce_add_sync(~0u, lane < warps ? sh.warp_n[turn][lane] : 0);
    };
    // ... and over the cluster's
    auto total_cluster = [&](uint64_t& m, uint32_t& n) {
        total(m, n, SAMPLE_WARPS);
        if (cs > 1) {
            const int turn = turns.next_cluster();
            if (tid == 0) {
                sh.block_mass[turn] = m;
                sh.block_n[turn] = n;
            }
            cluster_barrier();
            m = warp_sum47(lane < cs ? static_cast<uint64_t>(ld_remote64(remote_smem(&sh.block_mass[turn], lane))) : 0);
            n = __reduce_add_sync(~0u, lane < cs ? static_cast<uint32_t>(ld_remote32(remote_smem(&sh.block_n[turn], lane))) : 0);
        }
    };
    // sums over the threads before this one (and, with `blocks`, the blocks before this one)
    auto before = [&](uint64_t m, uint32_t n, bool blocks, uint64_t& M, uint32_t& N) {
        uint64_t sm = m;
        uint32_t sn = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint64_t x = __shfl_up_sync(~0u, sm, o);
            const uint32_t y = __shfl_up_sync(~0u, sn, o);
            if (lane >= o) {
                sm += x;
                sn += y;
            }
        }
        const int turn = turns.next_block();
        if (lane == 31) {
            sh.warp_mass[turn][warp] = sm;
            sh.warp_n[turn][warp] = sn;
        }
        __syncthreads();
        const uint64_t pm = sh.warp_mass[turn][lane];
        const uint32_t pn = sh.warp_n[turn][lane];
        M = sm - m + warp_sum47(lane < warp ? pm : 0);
        N = sn - n + __reduce_add_sync(~0u, lane < warp ? pn : 0);
        if (blocks) {
            const uint64_t bm = warp_sum47(pm);
            const uint32_t bn = __reduce_add_sync(~0u, pn);
            const int at = turns.next_cluster();
            if (tid == 0) {
                sh.block_mass[at] = bm;
                sh.block_n[at] = bn;
            }
            cluster_barrier();
            M += warp_sum47(lane < rank ? static_cast<uint64_t>(ld_remote64(remote_smem(&sh.block_mass[at], lane))) : 0);
            N += __reduce_add_sync(~0u, lane < rank ? static_cast<uint32_t>(ld_remote32(remote_smem(&sh.block_n[at], lane))) : 0);
        }
    };

    copy(blockIdx.x / cs);
    for (int r = blockIdx.x / cs; r < p.n_rows; r += step) {
        const SampleRow q = sample_row(p, r);
        const uint32_t u = p.u[r];
        cp_async_wait<0>();
        __syncwarp();
        int32_t mx = SAMPLE_MASKED;
        each([&](int, uint4* x) {
            const int4 v = *reinterpret_cast<int4*>(x);
            mx = max(mx, max(max(v.x, v.y), max(v.z, v.w)));
        });
        const int32_t own_max = mx;
        const int now = turns.next_block();
        mx = __reduce_max_sync(~0u, mx);
        if (lane == 0) sh.warp_max[now][warp] = mx;
        __syncthreads();
        mx = __reduce_max_sync(~0u, sh.warp_max[now][lane]);
        if (cs > 1) {
            const int turn = turns.next_cluster();
            if (tid == 0) sh.block_max[turn] = mx;
            cluster_barrier();
            mx = __reduce_max_sync(~0u, lane < cs ? ld_remote32(remote_smem(&sh.block_max[turn], lane)) : SAMPLE_MASKED);
        }
        if (!q.ok || mx == SAMPLE_MASKED) {  // (the whole cluster agrees)
            if (tid == 0 && rank == 0) {
                if (!q.ok) atomicCAS(p.err, 0, ERR_SAMPLE_PARAM);
                p.token[r] = -1;
                if (p.kept) p.kept[r] = 0;
                if (p.prob) p.prob[r] = 0;
            }
            copy(r + step);
            continue;
        }
        // Weights.  min-p first, whose cut is known: weights below it go.  (All three keep prefixes of one order.)
        const SampleScale scale{static_cast<uint32_t>(mx), q.b2};
        const uint32_t least = max(static_cast<uint32_t>(q.mp) << 14, 1u);
        const bool cuts_mass = q.p < 65536;
        uint64_t own_mass = 0, mass = 0;
        uint32_t own_n = 0, some = 0, n = p.vocab;

        // The list: its length, what this thread has of it and above it, and whether it reaches up to the maximum.
        uint32_t list_n = 0, mine_at = 0, mine_n = 0;
        uint64_t mine_above = 0;
        bool have_list = false, list_to_top = false, by_row = false;
        const uint32_t* lw = cs > 1 ? sh.w + SAMPLE_LIST / 2 : sh.w;
        const uint32_t room = cs > 1 ? SAMPLE_LIST / 2 : SAMPLE_LIST;
        // makes the list of the mine_n words that put(place) stores for each thread
        auto collect = [&](auto put) {
            uint64_t none;
            before(0, mine_n, false, none, mine_at);
            if (mine_n) put(mine_at);
            if (cs > 1) {
                const int turn = turns.next_cluster();
                if (tid == SAMPLE_THREADS - 1) sh.block_n[turn] = mine_at + mine_n;
                cluster_barrier();
                uint32_t to = SAMPLE_LIST / 2;
                for (int b = 0; b < cs; ++b) {
                    const uint32_t have = static_cast<uint32_t>(ld_remote32(remote_smem(&sh.block_n[turn], b)));
                    for (uint32_t i = tid; i < have; i += SAMPLE_THREADS)
                        sh.w[to + i] = static_cast<uint32_t>(ld_remote32(remote_smem(&sh.w[i], b)));
                    to += have;
                }
                list_n = to - SAMPLE_LIST / 2;
                cluster_barrier();
            } else {
                if (tid == SAMPLE_THREADS - 1) sh.few_n = mine_at + mine_n;
                __syncthreads();
                list_n = sh.few_n;
            }
        };
        // Once a warp needs its part of the row no more, the next row's may come.
        bool released = false;
        auto release = [&]() {
            if (!released) {
                __syncwarp();
                copy(r + step);
                released = true;
            }
        };

        // A small top-k needs the weights of the highest logits only.  The distance that some more than k threads'
        // maxima lie within is found like a guess below; all logits within it go on the list.  If k of them weigh more
        // than a logit at that distance would, none outside can be among the k.
        // (With k 50, all weights first and then a search: 500 rows of 20000 69 us, of 12000 61, 1000 of 4000 82, one of
        // 4000 11.6; this way 47, 42, 67 and 10.0.)
        bool quick = q.k > 0 && q.k <= SAMPLE_THREADS / 2;
        if (quick) {
            sh.w[tid] = own_max == SAMPLE_MASKED ? ~0u : static_cast<uint32_t>(mx) - static_cast<uint32_t>(own_max);
            __syncthreads();
            const uint32_t want = q.k + q.k / 8 + 1;
            uint32_t within = 0, unit = 0;  // threshold so far and what the next round adds
#pragma unroll 1
            for (int round = 0; round < 2; ++round) {
                // warp b's threshold: 2^b, then one of 32 parts of the last octave
                const uint32_t th = round == 0 ? 1u << warp : within + (warp + 1) * unit;
                uint32_t f = 0;
#pragma unroll
                for (int i = lane; i < SAMPLE_THREADS / 4; i += 32) {
                    const uint4 w = reinterpret_cast<const uint4*>(sh.w)[i];
                    f += (w.x < th) + (w.y < th) + (w.z < th) + (w.w < th);
                }
                f = __reduce_add_sync(~0u, f);
                const int turn = turns.next_block();
                if (lane == 0) sh.warp_n[turn][warp] = f;
                __syncthreads();
                const uint32_t reach = __ballot_sync(~0u, sh.warp_n[turn][lane] >= want);
                const int b = __ffs(reach) - 1;
                if (round == 0) {
                    // (Where too few threads have any logit near, `unit` stays 0: the second round finds nothing then.)
                    within = b <= 0 ? 0 : 1u << (b - 1);
                    if (b >= 0) unit = max(within >> 5, 1u);
                } else {
                    within += (b < 0 ? 32 : b + 1) * unit;
                }
            }
            if (unit == 0) within = 0;
            if (cs > 1) {  // the first block's distance is the cluster's
                const int turn = turns.next_cluster();
                if (tid == 0) sh.block_n[turn] = within;
                cluster_barrier();
                within = static_cast<uint32_t>(ld_remote32(remote_smem(&sh.block_n[turn], 0)));
            }
            each([&](int, uint4* at) {
                const uint4 v = *at;
                own_n += (scale.row_max - v.x < within) + (scale.row_max - v.y < within) + (scale.row_max - v.z < within) +
                         (scale.row_max - v.w < within);
            });
            uint32_t found = own_n;
            total_cluster(mass, found);
            quick = found >= static_cast<uint32_t>(q.k) && found <= room;
            if (quick) {
                const uint32_t outside = scale.at_distance<true>(within);
                uint32_t sure = 0;
                mine_n = own_n;
                collect([&](uint32_t at) {
                    each([&](int, uint4* from) {
                        const uint4 v = *from;
                        auto put = [&](uint32_t l) {
                            if (scale.row_max - l < within) {
                                const uint32_t w = scale(l);
                                sure += w > outside && w >= least;
                                sh.w[at++] = w >= least ? w : 0;
                            }
                        };
                        put(v.x);
                        put(v.y);
                        put(v.z);
                        put(v.w);
                    });
                });
                total_cluster(mass, sure);
                quick = sure >= static_cast<uint32_t>(q.k);
                have_list = list_to_top = quick;
                n = list_n;
            }
            if (!quick) {
                own_n = mine_n = 0;
                n = p.vocab;
            }
        }
        if (!quick) {
            auto weigh_all = [&](auto checked, auto counted) {
                each([&](int k, uint4* x) {
                    uint4 v = *x;
                    auto weigh = [&](uint32_t l) {
                        uint32_t w;
                        if (decltype(checked)::value) {
                            w = scale(l);
                            w = w >= least ? w : 0;
                        } else {
                            w = scale.at_distance<false>(scale.row_max - l);
                        }
                        if (decltype(counted)::value) own_n += w != 0;
                        return w;
                    };
                    v = make_uint4(weigh(v.x), weigh(v.y), weigh(v.z), weigh(v.w));
                    *x = v;
                    own_mass += v.x + v.y;  // (two are at most 2^31)
                    own_mass += v.z + v.w;
                    if (k == ch >> 1) some = v.x;
                });
            };
            const bool need_n = q.k != 0 || !cuts_mass;
            if (q.mp || !scale.plain()) weigh_all(std::true_type{}, std::true_type{});
            else if (need_n) weigh_all(std::false_type{}, std::true_type{});
            else weigh_all(std::false_type{}, std::false_type{});
            mass = own_mass;
            uint32_t x = own_n;
            total_cluster(mass, x);
            if (need_n) n = x;
            mine_above = own_mass;
        }
        const bool cuts_n = quick || (q.k != 0 && static_cast<uint32_t>(q.k) < n);
        if (quick || (!cuts_n && !cuts_mass)) release();

        // theta, the mass and the number of the weights above it, and how many equal to it are kept
        uint32_t theta = 0, above_n = n;
        uint64_t above = mass, quota = 0;
#pragma unroll 1
        for (int stage = 0; stage < 2; ++stage) {
            const bool by_count = stage == 0;  // top-k, then top-p
            uint64_t goal;
            if (by_count) {
                if (!cuts_n) continue;
                goal = q.k;
            } else {
                if (!cuts_mass) continue;
                goal = sample_goal(mass, q.p);
                if (above < goal) {  // (within the ties that top-k kept)
                    quota = (goal - above + theta - 1) / theta;
                    mass = above + quota * theta;
                    continue;
                }
            }
            // The largest theta whose weights >= theta number or weigh `goal` lies in [lo, hi), where c weights (at most)
            // are; hi_mass and hi_n are at or above hi.  Weights up to (above - goal) / vocab, all together, are not missed.
            uint32_t lo = theta + 1, hi = SAMPLE_TOP, hi_n = 0, c = above_n;
            uint64_t hi_mass = 0;
            if (!by_count) lo = max(lo, static_cast<uint32_t>((above - goal) / static_cast<uint32_t>(p.vocab)) + 1);
            auto middle = [&]() {
                if (hi > 4 * lo) return 1u << ((63 - __clz(lo) - __clz(hi)) / 2);  // (between: their lengths differ by two)
                return lo + (hi - lo) / 2;
            };
            // narrows the window to [mid, hi), with mass m and x weights, or to [lo, mid); true for the first
            auto narrow = [&](uint32_t mid, uint64_t m, uint32_t x) {
                if ((by_count ? hi_n + x : hi_mass + m) >= goal) {
                    lo = mid;
                    c = x;
                    return true;
                }
                hi = mid;
                hi_mass += m;
                hi_n += x;
                c -= x;
                return false;
            };
            if (!(have_list && list_to_top)) {
                // Where to look first.  For a count: the greatest of 1024 thresholds that `goal` threads' largest weights
                // reach, which as many weights then do.  For a mass: a sample of one weight per thread tells where the
                // mass that may be missed is expected to lie below.  (Not worth it where a pass is short: one row of 49152
                // on four blocks takes 20 us without and 23 with, 500 of 20000 on one 85 and 98.)
                uint32_t guess = 0;
                if (c > room && ch >= SAMPLE_GUESS_CHUNKS && (!by_count || goal <= SAMPLE_THREADS / 2)) {
                    const uint32_t top = scale(static_cast<uint32_t>(own_max));
                    sh.w[tid] = by_count ? (top >= least ? top : 0) : (some + 1024) >> 11;  // (masses in units of 2^11)
                    __syncthreads();
                    const uint64_t want = by_count ? goal : (above - goal) / static_cast<uint32_t>(4 * ch * cs);
                    uint32_t unit = 1;
#pragma unroll 1
                    for (int round = 0; round < 2; ++round) {
                        // warp b's threshold: the octave 2^b, then its 32nd parts
                        const uint32_t th = round == 0 ? 1u << warp : guess + warp * unit, th11 = (th + 1024) >> 11;
                        uint32_t f = 0;
#pragma unroll
                        for (int i = lane; i < SAMPLE_THREADS / 4; i += 32) {
                            const uint4 w = reinterpret_cast<const uint4*>(sh.w)[i];
                            if (by_count) f += (w.x >= th) + (w.y >= th) + (w.z >= th) + (w.w >= th);
                            else f += (w.x < th11 ? w.x : 0) + (w.y < th11 ? w.y : 0) + (w.z < th11 ? w.z : 0) + (w.w < th11 ? w.w : 0);
                        }
                        f = __reduce_add_sync(~0u, f);
                        const int turn = turns.next_block();
                        if (lane == 0) sh.warp_n[turn][warp] = f;
                        __syncthreads();
                        f = sh.warp_n[turn][lane];
                        // (true up to some threshold)
                        const int b = 31 - __clz(__ballot_sync(~0u, by_count ? f >= want : static_cast<uint64_t>(f) << 11 <= want));
                        guess = round == 0 ? 1u << max(b, 0) : guess + max(b, 0) * unit;
                        unit = max(guess >> 5, 1u);
                        if (by_count && b < 0) guess = 0;  // (fewer threads than that have any weight)
                    }
                    if (cs > 1) {  // the first block's guess is the cluster's
                        const int turn = turns.next_cluster();
                        if (tid == 0) sh.block_n[turn] = guess;
                        cluster_barrier();
                        guess = static_cast<uint32_t>(ld_remote32(remote_smem(&sh.block_n[turn], 0)));
                    }
                }
                // this thread's weights in [lo, hi) (once known) and at or above hi
                uint32_t in_n = 0, up_n = 0;
                uint64_t up_mass = 0;
                bool known = false;
                for (int k = 0; c > room && hi - lo > 1; ++k) {
                    // around a guessed mass first a fifth below, then a quarter above
                    uint32_t mid = k == 0 ? (by_count ? guess : guess - guess / 5) : k == 1 && !by_count ? guess + guess / 4 : 0;
                    if (mid <= lo || mid >= hi) mid = middle();
                    uint64_t m = 0;
                    uint32_t x = 0;
                    each([&](int, uint4* at) {
                        // max(v, mid) summed, and how often it is above max(v, mid - 1), which tells the others
                        const uint4 v = *at;
                        auto add = [&](uint32_t w) {
                            const uint32_t a = max(w, mid), b = max(w, mid - 1);
                            m += a;
                            x += a - b;
                        };
                        add(v.x);
                        add(v.y);
                        add(v.z);
                        add(v.w);
                    });
                    m -= static_cast<uint64_t>(mid) * x;  // (x weights lie below mid)
                    x = 4 * ch - x;
                    const uint64_t own_m = m;
                    const uint32_t own_x = x;
                    total_cluster(m, x);
                    if (narrow(mid, m - hi_mass, x - hi_n)) {
                        in_n = own_x - up_n;
                        known = true;
                    } else {
                        in_n -= own_x - up_n;
                        up_n = own_x;
                        up_mass = own_m;
                    }
                }
                by_row = hi - lo == 1;  // (the cut fell on the way: the draw counts the row again)
                if (!by_row) {
                    // the window's weights, by thread
                    if (!known) {
                        in_n = 0;
                        each([&](int, uint4* at) {
                            const uint4 v = *at;
                            in_n += (v.x - lo < hi - lo) + (v.y - lo < hi - lo) + (v.z - lo < hi - lo) + (v.w - lo < hi - lo);
                        });
                    }
                    mine_n = in_n;
                    mine_above = up_mass;
                    collect([&](uint32_t at) {
                        each([&](int, uint4* from) {
                            const uint4 v = *from;
                            if (max(max(v.x, v.y), max(v.z, v.w)) < lo) return;
                            auto put = [&](uint32_t w) {
                                const bool in = w - lo < hi - lo;
                                if (in) sh.w[at] = w;
                                at += in;
                            };
                            put(v.x);
                            put(v.y);
                            put(v.z);
                            put(v.w);
                        });
                    });
                    c = list_n;
                    have_list = true;
                    list_to_top = hi == SAMPLE_TOP;
                    if (list_to_top || !by_count || !cuts_mass) release();
                }
            }
            const int busy = min(static_cast<int>(list_n + 127) / 128, SAMPLE_WARPS);  // warps that share the list
            while (c > SAMPLE_FEW && hi - lo > 1) {
                const uint32_t mid = middle();
                uint64_t m = 0;
                uint32_t x = 0;
                if (warp < busy)
                    for (uint32_t i = tid; i < list_n; i += 32 * busy) {
                        const uint32_t w = lw[i];
                        if (w - mid < hi - mid) {
                            m += w;
                            ++x;
                        }
                    }
                total(m, x, busy);
                narrow(mid, m, x);
            }
            if (hi - lo > 1) {
                const uint32_t* few = lw;
                uint32_t few_n = list_n;
                if (list_n > SAMPLE_FEW) {
                    __syncthreads();
                    if (tid == 0) sh.few_n = 0;
                    __syncthreads();
                    if (warp < busy)
                        for (uint32_t i = tid; i < list_n; i += 32 * busy) {
                            const uint32_t w = lw[i];
                            if (w - lo < hi - lo) sh.few[atomicAdd(&sh.few_n, 1u)] = w;
                        }
                    __syncthreads();
                    few = sh.few;
                    few_n = sh.few_n;
                } else if (!by_count) {
                    __syncthreads();  // (top-k's words have been read)
                }
                // warp b: candidates b, b + 32, ... (a short list as it is may hold weights outside the window)
                for (uint32_t j = warp; j < few_n; j += SAMPLE_WARPS) {
                    const uint32_t mine = few[j];
                    if (mine - lo >= hi - lo) continue;
                    uint64_t m = 0;  // of those above mine
                    uint32_t x = 0, same = 0;
                    for (uint32_t i = lane; i < few_n; i += 32) {
                        const uint32_t w = few[i];
                        if (w > mine && w < hi) {
                            m += w;
                            ++x;
                        }
                        same += w == mine;
                    }
                    m = warp_sum47(m) + hi_mass;
                    x = __reduce_add_sync(~0u, x) + hi_n;
                    same = __reduce_add_sync(~0u, same);
                    // (warps of equal weights write equal words)
                    if (lane == 0 && (by_count ? x : m) < goal &&
                        (by_count ? x + same : m + static_cast<uint64_t>(same) * mine) >= goal) {
                        sh.theta = mine;
                        sh.above = m;
                        sh.above_n = x;
                    }
                }
                __syncthreads();
                theta = sh.theta;
                above = sh.above;
                above_n = sh.above_n;
            } else {
                theta = lo;
                above = hi_mass;
                above_n = hi_n;
            }
            quota = by_count ? goal - above_n : (goal - above + theta - 1) / theta;
            mass = above + quota * theta;
        }
        const uint64_t target = sample_target(mass, u);

        // The draw: kept mass and ties of each thread's part of the row, in index order.
        uint64_t m = mine_above;
        uint32_t t = 0;
        if (by_row) {
            m = 0;
            each([&](int, uint4* at) {
                const uint4 v = *at;
                m += (v.x > theta ? v.x : 0) + (v.y > theta ? v.y : 0);
                m += (v.z > theta ? v.z : 0) + (v.w > theta ? v.w : 0);
                t += (v.x == theta) + (v.y == theta) + (v.z == theta) + (v.w == theta);
            });
        } else if (have_list) {
            for (uint32_t i = mine_at; i < mine_at + mine_n; ++i) {
                const uint32_t w = sh.w[i];
                m += w > theta ? w : 0;
                t += w == theta;
            }
        }
        uint64_t cur;
        uint32_t ties;
        before(m, t, cs > 1, cur, ties);
        uint64_t used = ties;
        cur += theta * min(used, quota);
        const bool mine = cur <= target && target < cur + m + theta * min(static_cast<uint64_t>(t), quota - min(quota, used));
        const uint32_t winner = __ballot_sync(~0u, mine);
        if (winner) {
            // one thread of the cluster; its warp weighs its logits again, 32 at a time
            const int who = __ffs(winner) - 1, from = __shfl_sync(~0u, base, who);
            uint64_t run = __shfl_sync(~0u, cur, who), seen = __shfl_sync(~0u, used, who);
            for (int i0 = 0; i0 < 4 * ch; i0 += 32) {
                const int at = from + i0 + lane;
                uint32_t w = i0 + lane < 4 * ch && at < p.vocab ? scale(static_cast<uint32_t>(p.logits[r * p.ld + at])) : 0;
                if (w < least) w = 0;
                const bool tie = w == theta && w != 0;
                const uint32_t tied = __ballot_sync(~0u, tie);
                if (tie && seen + __popc(tied & ((1u << lane) - 1)) >= quota) w = 0;
                if (w < theta) w = 0;
                uint64_t to = w;  // kept mass up to and with this one
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const uint64_t x = __shfl_up_sync(~0u, to, o);
                    if (lane >= o) to += x;
                }
                if (w != 0 && run + to - w <= target && target < run + to) {
                    p.token[r] = at;
                    if (p.kept) p.kept[r] = static_cast<int32_t>(above_n + quota);
                    if (p.prob) p.prob[r] = static_cast<int32_t>(((static_cast<uint64_t>(w) << 30) + (mass >> 1)) / mass);
                }
                run += __shfl_sync(~0u, to, 31);
                seen += __popc(tied);
            }
        }
        release();
        __syncthreads();  // the list has been read
    }
    cp_async_wait<0>();
    if (cs > 1) cluster_barrier();  // no block leaves while its words are read
}

}  // namespace eii
