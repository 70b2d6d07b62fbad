// Eviction from the paged cache: choosing the tokens a budget keeps by their
// attention mass, and moving them to the front of their pages.
//
// Each (sequence, layer, KV head) chooses for itself -- its tokens sit in pages
// of its own -- and every head keeps the same number, so block tables and
// lengths stay common to all heads and the ordinary rollback ends the eviction.

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"

namespace sdc {
namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------
// Selection.
//
// Of the candidates [sinks, T - recent) the `need` largest are kept: the
// need-th largest key is found by a radix descent over order-preserving 32-bit
// keys (digits of 11, 11 and 10 bits, a histogram each), which ends early when
// every key of the bin it stands in is kept; one ordered sweep then writes the
// candidates above it, and the first of those equal to it.  RANKS blocks (a
// cluster) serve one (sequence, layer, head), each a contiguous share of the
// keys; the blocks' histograms and counts meet over distributed shared memory.
// A thread holds up to 32 keys in registers and a block of 1024 threads as many
// again in shared memory, so the mass pages are read once; what a share has
// beyond that is read again (from L2) for every step.  Keys are handled four at
// a time, as the pages hold them; a key that is no candidate is 0, below every
// mass's key.
//
// Measured (B200): 8 x 6000 to 8192 tokens, 256 (layer, head) rows each, to 2048:
// 67 us for 75 MB; 131072 tokens, 64 rows, to 16384: 57 us; 1021 tokens, 128 rows:
// 6.3 us.  Bound by instruction issue (56 % of the slots, 2500 instructions a warp
// for 16 keys a thread) and by the descent's barriers, not by HBM.  All keys in
// shared memory instead of registers: 73, 80 and 7.1 us.
// ---------------------------------------------------------------------------

constexpr int kSelectCluster = 8;
constexpr int kBins = 2048;

struct SelectArgs {
    Pool pool;
    const float* mass;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* lens;
    int64_t max_len;
    int64_t budget, recent, sinks;
    uint32_t parked;  // groups a block keeps in shared memory
    int32_t vec;   // four tokens of a group lie in one block, 16-byte aligned
    int32_t* kept;
    FastDiv div_block;
    FastDiv div_heads;
    FastDiv div_layers;
    int32_t* status;
};

// Larger mass, larger key; -0 as +0, NaN above everything; never 0.
__device__ __forceinline__ uint32_t mass_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return x != x ? 0xffffffffu : k;
}

template <int THREADS, int GROUPS>
struct SelectShared {
    static constexpr int kWarps = THREADS / 32;
    __align__(16) uint32_t hist[kBins];  // this block's counts, highest bin first, read by the cluster
    uint32_t warp_sum[kWarps];
    uint32_t before_warp[2][GROUPS * kWarps + 1];  // (above, equal) before a warp's groups of each step
    uint2 counts;                                         // this block's (above, equal), read by the cluster
    uint32_t slice_total[kSelectCluster];                 // written by the slices' blocks
    uint32_t digit, before, inside;                       // written by the block that finds them
};

// GROUPS of four keys a thread; at most 64 registers (1024 threads an SM: 20 %
// faster than the 128 that the loops would take; eight groups spill 48 to 64
// bytes a thread).
template <int RANKS, int THREADS, int GROUPS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) select_tokens_kernel(SelectArgs a) {
    using Shared = SelectShared<THREADS, GROUPS>;
    constexpr int kSelectThreads = THREADS, kSelectWarps = THREADS / 32;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const auto sync = [&] {
        if constexpr (RANKS == 1) {
            __syncthreads();
        } else {
            cluster.sync();
        }
    };
    const uint32_t rank = RANKS == 1 ? 0 : cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t item = blockIdx.x / RANKS;
    uint32_t rest, h, b, layer;
    a.div_heads.divmod(item, rest, h);
    a.div_layers.divmod(rest, b, layer);
    int32_t* out = a.kept + static_cast<int64_t>(item) * a.budget;
    const int64_t T = __ldg(a.lens + b);
    const bool bad_length = T < 0 || T > a.max_len || T > a.table_stride * a.pool.block_size;
    if (bad_length || T <= a.budget) {  // the whole cluster agrees
        if (bad_length && threadIdx.x == 0 && rank == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
        for (int64_t j = static_cast<int64_t>(rank) * kSelectThreads + threadIdx.x; j < a.budget;
             j += RANKS * kSelectThreads) {
            out[j] = !bad_length && j < T ? static_cast<int32_t>(j) : -1;
        }
        return;
    }
    // tokens kept whatever their mass
    for (int64_t j = static_cast<int64_t>(rank) * kSelectThreads + threadIdx.x; j < a.sinks + a.recent;
         j += RANKS * kSelectThreads) {
        if (j < a.sinks) {
            out[j] = static_cast<int32_t>(j);
        } else {
            out[a.budget - a.recent + j - a.sinks] = static_cast<int32_t>(T - a.recent + j - a.sinks);
        }
    }
    uint32_t need = static_cast<uint32_t>(a.budget - a.sinks - a.recent);  // below the candidates' number: T > budget
    if (need == 0) return;

    const int32_t* table = a.tables + b * a.table_stride;
    const float* mass = a.mass + layer * a.pool.sls + h * a.pool.shs;
    const uint32_t lo = static_cast<uint32_t>(a.sinks), hi = static_cast<uint32_t>(T - a.recent);  // candidates
    const uint32_t g_lo = lo / 4, groups = (hi + 3) / 4 - g_lo;
    const uint32_t share = (groups + RANKS - 1) / RANKS;
    const uint32_t g0 = g_lo + min(groups, share * rank), g1 = g_lo + min(groups, share * (rank + 1));
    const uint32_t count = g1 - g0;
    constexpr uint32_t kRound = GROUPS * THREADS;  // groups a block holds
    const uint32_t rounds = (count + kRound - 1) / kRound;
    bool missing = false;
    auto fetch = [&](uint32_t g) -> uint4 {  // keys of tokens 4 (g0 + g) .. + 3, from their pages
        const uint32_t t = 4 * (g0 + g);
        uint32_t j, off;
        float4 m = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.vec) {
            a.div_block.divmod(t, j, off);
            const int64_t block = __ldg(table + j);
            if (block >= 0 && block < a.pool.num_blocks) {
                m = __ldg(reinterpret_cast<const float4*>(mass + block * a.pool.sbs + off));
            } else {
                missing = true;
            }
        } else {
            float* x = reinterpret_cast<float*>(&m);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                if (t + e < lo || t + e >= hi) continue;  // (past the context the table may end)
                a.div_block.divmod(t + e, j, off);
                const int64_t block = __ldg(table + j);
                if (block >= 0 && block < a.pool.num_blocks) {
                    x[e] = __ldg(mass + block * a.pool.sbs + off);
                } else {
                    missing = true;
                }
            }
        }
        uint4 k = make_uint4(mass_key(m.x), mass_key(m.y), mass_key(m.z), mass_key(m.w));
        if (t < lo || t + 4 > hi) {
            if (t < lo || t >= hi) k.x = 0u;
            if (t + 1 < lo || t + 1 >= hi) k.y = 0u;
            if (t + 2 < lo || t + 2 >= hi) k.z = 0u;
            if (t + 3 < lo || t + 3 >= hi) k.w = 0u;
        }
        return k;
    };

    // This thread's groups: u * THREADS + threadIdx.x of each round, the first
    // round's in registers, the next rounds' in shared memory as far as it goes.
    extern __shared__ uint4 parked[];
    uint4 k[GROUPS];
    const auto fetch_at = [&](uint32_t g) { return g < count ? fetch(g) : make_uint4(0u, 0u, 0u, 0u); };
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) k[u] = fetch_at(u * THREADS + threadIdx.x);
    for (uint32_t g = kRound + threadIdx.x; g < count && g - kRound < a.parked; g += THREADS) {
        parked[g - kRound] = fetch(g);  // read by this thread only
    }
    const auto group = [&](uint32_t round, int u) {  // rounds past the first
        const uint32_t g = round * kRound + u * THREADS + threadIdx.x;
        return g < count && g - kRound < a.parked ? parked[g - kRound] : fetch_at(g);
    };

    // radix descent: `prefix` holds the digits found so far, under `mask`
    uint32_t prefix = 0, mask = 0;
    bool found_all = false;
    const auto descend = [&](auto digit) {
        constexpr int kPass = decltype(digit)::value;
        constexpr int shift = kPass == 0 ? 21 : kPass == 1 ? 10 : 0;
        constexpr uint32_t bins = kPass == 2 ? 1024 : kBins;
        for (uint32_t i = threadIdx.x * 4; i < bins; i += THREADS * 4) {
            *reinterpret_cast<uint4*>(&sh.hist[i]) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
        // (a key 0 falls in the last bin of the first digit, behind every candidate)
        const auto add = [&](uint32_t x) {
            if (kPass == 0 || (x & mask) == prefix) atomicAdd(&sh.hist[~(x >> shift) & (bins - 1)], 1u);
        };
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
            if (u * THREADS < count) add(k[u].x), add(k[u].y), add(k[u].z), add(k[u].w);  // (the same on all threads)
        }
        for (uint32_t round = 1; round < rounds; ++round) {
            for (int u = 0; u < GROUPS && round * kRound + u * THREADS < count; ++u) {
                const uint4 x = group(round, u);
                add(x.x), add(x.y), add(x.z), add(x.w);
            }
        }
        sync();
        // Block r sums slice r of the cluster's histograms (each remote word is
        // read once); the bin where the running count from the top passes
        // `need` lies in one slice, whose block tells the others.
        constexpr int kOwn = kBins / RANKS / kSelectThreads < 4 ? 4 : kBins / RANKS / kSelectThreads;  // bins a thread
        const uint32_t slice = bins / RANKS;
        uint32_t n[kOwn] = {}, mine = 0;
        if (threadIdx.x * kOwn < slice) {
#pragma unroll
            for (int q = 0; q < kOwn; q += 4) {
                uint4 c[RANKS];
#pragma unroll
                for (int o = 0; o < RANKS; ++o) {
                    const uint4* from = reinterpret_cast<const uint4*>(&sh.hist[rank * slice + threadIdx.x * kOwn + q]);
                    if constexpr (RANKS > 1) from = cluster.map_shared_rank(from, o);
                    c[o] = *from;
                }
#pragma unroll
                for (int o = 0; o < RANKS; ++o) {
                    n[q] += c[o].x, n[q + 1] += c[o].y, n[q + 2] += c[o].z, n[q + 3] += c[o].w;
                }
            }
#pragma unroll
            for (int e = 0; e < kOwn; ++e) mine += n[e];
        }
        uint32_t run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(kFullMask, run, o);
            if (lane >= o) run += y;
        }
        if (lane == 31) sh.warp_sum[warp] = run;
        __syncthreads();
        uint32_t before = lane < kSelectWarps ? sh.warp_sum[lane] : 0u;  // inclusive sum over the warps
#pragma unroll
        for (int o = 1; o < kSelectWarps; o <<= 1) {
            const uint32_t y = __shfl_up_sync(kFullMask, before, o);
            if (lane >= o) before += y;
        }
        if constexpr (RANKS > 1) {
            const uint32_t total = __shfl_sync(kFullMask, before, kSelectWarps - 1);
            if (threadIdx.x < RANKS) *cluster.map_shared_rank(&sh.slice_total[rank], threadIdx.x) = total;
        }
        before = __shfl_sync(kFullMask, before, max(warp - 1, 0));
        before = (warp == 0 ? 0u : before) + run - mine;
        if constexpr (RANKS > 1) {
            cluster.sync();
            for (uint32_t o = 0; o < rank; ++o) before += sh.slice_total[o];
        }
        if (before < need && before + mine >= need) {  // exactly one thread
            bool found = false;
#pragma unroll
            for (uint32_t e = 0; e < kOwn; ++e) {
                if (!found && before + n[e] >= need) {
                    const uint32_t digit = bins - 1 - (rank * slice + threadIdx.x * kOwn + e);
#pragma unroll
                    for (int o = 0; o < RANKS; ++o) {
                        Shared* to = &sh;
                        if constexpr (RANKS > 1) to = cluster.map_shared_rank(to, o);
                        to->digit = digit, to->before = before, to->inside = n[e];
                    }
                    found = true;
                }
                before += n[e];
            }
        }
        sync();  // the histograms are read until here
        prefix |= sh.digit << shift;
        mask |= (bins - 1) << shift;
        need -= sh.before;  // of the keys equal to the prefix under the mask, this many are kept
        if (sh.inside == need) {  // all of them: whatever is not below the prefix
            prefix -= 1;
            need = 0;
            found_all = true;
        }
        __syncthreads();
    };
    descend(std::integral_constant<int, 0>());
    if (!found_all) descend(std::integral_constant<int, 1>());
    if (!found_all) descend(std::integral_constant<int, 2>());
    // kept: keys above `prefix`, and the first `need` equal to it

    // Ordered sweep.  The tokens of step u come before those of step u + 1, a
    // warp's before the next warp's: a key's rank is what came before its warp
    // and step, plus the lanes before its own, plus its group's earlier keys.
    // `which`: keys above the prefix, or those equal to it.
    const auto hits = [&](uint4 x, int which) -> uint32_t {
        return which == 0 ? (x.x > prefix ? 1u : 0u) + (x.y > prefix ? 1u : 0u) + (x.z > prefix ? 1u : 0u) +
                                (x.w > prefix ? 1u : 0u)
                          : (x.x == prefix ? 1u : 0u) + (x.y == prefix ? 1u : 0u) + (x.z == prefix ? 1u : 0u) +
                                (x.w == prefix ? 1u : 0u);
    };
    // ranks of this thread's groups of the round among its block's; returns the block's number
    const auto rank_groups = [&](int which, uint32_t (&at)[GROUPS]) -> uint32_t {
        // four steps' counts to a word: a warp's sum is at most 128
        constexpr int kWords = (GROUPS + 3) / 4;
        uint32_t own[kWords] = {}, run[kWords];
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) own[u / 4] |= hits(k[u], which) << (8 * (u % 4));
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            run[w] = own[w];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(kFullMask, run[w], o);
                if (lane >= o) run[w] += y;
            }
        }
        uint32_t* table = sh.before_warp[which];
        if (lane == 31) {
#pragma unroll
            for (int u = 0; u < GROUPS; ++u) table[u * kSelectWarps + warp] = run[u / 4] >> (8 * (u % 4)) & 255u;
        }
        __syncthreads();
        if (warp == 0) {  // exclusive sums in place, the total behind them
            constexpr int kEntries = GROUPS * kSelectWarps, kEach = (kEntries + 31) / 32;
            uint32_t v[kEach], sum = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                v[e] = sum;
                if (lane * kEach + e < kEntries) sum += table[lane * kEach + e];
            }
            uint32_t inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(kFullMask, inc, o);
                if (lane >= o) inc += y;
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (lane * kEach + e < kEntries) table[lane * kEach + e] = v[e] + inc - sum;
            }
            if (lane == 31) table[GROUPS * kSelectWarps] = inc;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
            at[u] = table[u * kSelectWarps + warp] + ((run[u / 4] - own[u / 4]) >> (8 * (u % 4)) & 255u);
        }
        return table[GROUPS * kSelectWarps];
    };
    uint32_t above = 0, equal = 0;  // of the tokens before this round
    if constexpr (RANKS > 1) {
        uint32_t up = 0, eq = 0;
#pragma unroll
        for (int u = 0; u < GROUPS; ++u) {
            up += hits(k[u], 0);
            if (need != 0) eq += hits(k[u], 1);
        }
        for (uint32_t round = 1; round < rounds; ++round) {
            for (int u = 0; u < GROUPS; ++u) {
                const uint4 x = group(round, u);
                up += hits(x, 0);
                if (need != 0) eq += hits(x, 1);
            }
        }
        up = __reduce_add_sync(kFullMask, up);
        eq = __reduce_add_sync(kFullMask, eq);
        if (threadIdx.x == 0) sh.counts = make_uint2(0u, 0u);
        __syncthreads();
        if (lane == 0) atomicAdd(&sh.counts.x, up), atomicAdd(&sh.counts.y, eq);
        cluster.sync();
        for (uint32_t o = 0; o < rank; ++o) {
            const uint2 v = *cluster.map_shared_rank(&sh.counts, o);
            above += v.x, equal += v.y;
        }
    }
    for (uint32_t round = 0; round < rounds; ++round) {
        if (round > 0) {
#pragma unroll
            for (int u = 0; u < GROUPS; ++u) k[u] = group(round, u);
        }
        uint32_t at[GROUPS], eq_at[GROUPS];
        const uint32_t ups = rank_groups(0, at);
        uint32_t eqs = 0;
        const uint32_t t0 = 4 * (g0 + round * kRound + threadIdx.x);
        if (need == 0) {
#pragma unroll
            for (int u = 0; u < GROUPS; ++u) {
                int32_t* to = out + (lo + above + at[u]);
                const uint32_t x[4] = {k[u].x, k[u].y, k[u].z, k[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (x[e] > prefix) *to = static_cast<int32_t>(t0 + 4 * u * THREADS + e);
                    to += x[e] > prefix ? 1 : 0;
                }
            }
        } else {
            eqs = rank_groups(1, eq_at);
#pragma unroll
            for (int u = 0; u < GROUPS; ++u) {
                uint32_t up = above + at[u], eq = equal + eq_at[u];
                const uint32_t x[4] = {k[u].x, k[u].y, k[u].z, k[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool larger = x[e] > prefix, same = x[e] == prefix;
                    // kept before this one: every larger key, and the equal ones up to `need`
                    if (larger || (same && eq < need)) {
                        out[lo + up + min(eq, need)] = static_cast<int32_t>(t0 + 4 * u * THREADS + e);
                    }
                    up += larger ? 1u : 0u;
                    eq += same ? 1u : 0u;
                }
            }
        }
        above += ups, equal += eqs;
    }
    if (missing) report_fault(a.status, SDC_FAULT_BLOCK_RANGE);
    if constexpr (RANKS > 1) cluster.sync();  // `counts` is read until here
}

template <int RANKS, int THREADS, int GROUPS>
sdc_status_t launch_select(SelectArgs a, int64_t items, cudaStream_t st) {
    // shared memory for a second round of keys where a share may need one
    const int64_t share = ceil_div(ceil_div(a.max_len, 4) + 1, RANKS);
    a.parked = THREADS == 1024 && share > THREADS * GROUPS ? THREADS * GROUPS : 0;
    const size_t smem = a.parked * sizeof(uint4);
    if (smem > 0 && cudaFuncSetAttribute(select_tokens_kernel<RANKS, THREADS, GROUPS>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem)) != cudaSuccess) {
        return SDC_STATUS_CUDA_ERROR;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * RANKS));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = RANKS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, select_tokens_kernel<RANKS, THREADS, GROUPS>, a) != cudaSuccess) return SDC_STATUS_CUDA_ERROR;
    return launch_status();
}

// ---------------------------------------------------------------------------
// Compaction.
//
// Row j takes row kept[j] >= j, in place.  A block walks the destination rows
// of one (sequence, layer, head, keys | values) in order, a tile at a time: all
// of a tile's rows are loaded before any is stored (one barrier), and a later
// tile's sources lie behind every row an earlier tile writes, so loads run
// ahead: at tile t a thread reads the kept indices of tile t + 3, the block ids
// of tile t + 2 and the rows of tile t + 1.  128 threads and at most 72 registers
// (44 bytes a thread spill) let seven blocks share an SM: the blocks of a usual
// batch (sequences x layers x heads x 2) run as one wave.
//
// Measured (B200): 8 x 6000 to 8192 tokens to 4096, 8 layers x 8 heads of 128: 229 us
// for 1132 MB (4.9 TB/s, 75 % of the measured copy); six or eight blocks an SM 340
// and 245 us; loads one tile ahead of their own index chain, not three: 335 us.
// ---------------------------------------------------------------------------

constexpr int kCompactThreads = 128;
constexpr int kCompactDepth = 4;  // 16-byte chunks per thread and tile

struct CompactArgs {
    Pool pool;
    float* mass;  // or null
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* lens;
    const int32_t* kept;
    int64_t budget;
    int32_t tile_rows;
    uint64_t block_units;  // code stride of a block, in 16 bytes
    uint32_t row_units;    // of a row
    uint64_t block_scales; // scale stride of a block
    FastDiv div_chunks;  // 16-byte chunks of a code row
    FastDiv div_block;
    FastDiv div_heads;
    FastDiv div_layers;
    int32_t* status;
};

template <typename Index>
__global__ void __launch_bounds__(kCompactThreads, 7) compact_tokens_kernel(CompactArgs a) {
    __shared__ int s_faults;
    __shared__ uint32_t s_first;
    uint32_t rest, h, b, layer;
    a.div_heads.divmod(blockIdx.x, rest, h);
    a.div_layers.divmod(rest, b, layer);
    const int64_t T = __ldg(a.lens + b);
    const uint32_t N = static_cast<uint32_t>(a.budget);
    if (T <= a.budget) return;
    if (T > a.table_stride * a.pool.block_size) {
        if (threadIdx.x == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
        return;
    }
    const int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
    const int32_t* table = a.tables + b * a.table_stride;
    if (threadIdx.x == 0) s_faults = 0, s_first = N;
    __syncthreads();
    // the whole row is checked before anything moves; leading rows in place are skipped
    int faults = 0;
    uint32_t moved = N;
    for (uint32_t j = threadIdx.x; j < N; j += kCompactThreads) {
        const int32_t k = __ldg(kept + j), prev = j > 0 ? __ldg(kept + j - 1) : -1;
        if (k <= prev || k >= T) {
            faults |= SDC_FAULT_KEPT_ORDER;
        } else {
            const int32_t src = __ldg(table + a.div_block.div(static_cast<uint32_t>(k)));
            const int32_t dst = __ldg(table + a.div_block.div(j));
            if (src < 0 || src >= a.pool.num_blocks || dst < 0 || dst >= a.pool.num_blocks) {
                faults |= SDC_FAULT_BLOCK_RANGE;
            }
            if (static_cast<uint32_t>(k) != j) moved = min(moved, j);
        }
    }
    if (faults) atomicOr(&s_faults, faults);
    if (moved < N) atomicMin(&s_first, moved);
    __syncthreads();
    if (s_faults) {
        if (threadIdx.x == 0) report_fault(a.status, s_faults);
        return;
    }

    const bool is_key = blockIdx.y == 0;
    uint4* codes = reinterpret_cast<uint4*>((is_key ? a.pool.keys : a.pool.values) + layer * a.pool.cls +
                                            h * a.pool.chs);
    float* scales = (is_key ? a.pool.key_scales : a.pool.value_scales) + layer * a.pool.sls + h * a.pool.shs;
    float* mass = is_key && a.mass != nullptr ? a.mass + layer * a.pool.sls + h * a.pool.shs : nullptr;
    const uint32_t rows = static_cast<uint32_t>(a.tile_rows);
    const uint32_t first = s_first;
    if (first >= N) return;
    // this thread's rows and chunk of a tile (every row has one thread for its scale)
    uint32_t row[kCompactDepth], chunk[kCompactDepth];
#pragma unroll
    for (int u = 0; u < kCompactDepth; ++u) {
        a.div_chunks.divmod(threadIdx.x + u * kCompactThreads, row[u], chunk[u]);
        if (row[u] >= rows) row[u] = N;  // past every tile
    }
    const auto there = [&](uint32_t j0, uint32_t r) { return r < rows && j0 + r < N; };
    const auto kept_at = [&](uint32_t j0, uint32_t r) -> uint32_t {
        return there(j0, r) ? static_cast<uint32_t>(__ldg(kept + j0 + r)) : 0u;
    };
    // a token's code row in units of 16 bytes, and its scale's index
    const auto code_row = [&](uint32_t token) -> Index {
        uint32_t j, off;
        a.div_block.divmod(token, j, off);
        return static_cast<Index>(__ldg(table + j)) * static_cast<Index>(a.block_units) + off * a.row_units;
    };
    const auto scale_index = [&](uint32_t token) -> Index {
        uint32_t j, off;
        a.div_block.divmod(token, j, off);
        return static_cast<Index>(__ldg(table + j)) * static_cast<Index>(a.block_scales) + off;
    };
    // The pipeline's stages, oldest data first.  Loads and stores share the
    // pages, so they are plain accesses: the read-only path could return a
    // row as it was before an earlier store.
    uint4 data[2][kCompactDepth];
    float scale[2], weight[2] = {0.0f, 0.0f};
    Index source[kCompactDepth + 1];  // the last: of the scale's row
    uint32_t token[kCompactDepth + 1];
    const auto fetch_tokens = [&](uint32_t j0) {
#pragma unroll
        for (int u = 0; u < kCompactDepth; ++u) token[u] = kept_at(j0, row[u]);
        token[kCompactDepth] = kept_at(j0, threadIdx.x);
    };
    const auto fetch_sources = [&] {  // (a token outside a tile stands for token 0)
#pragma unroll
        for (int u = 0; u < kCompactDepth; ++u) source[u] = code_row(token[u]) + chunk[u];
        source[kCompactDepth] = scale_index(token[kCompactDepth]);
    };
    const auto fetch_rows = [&](uint32_t j0, uint4 (&v)[kCompactDepth], float& sv, float& mv) {
#pragma unroll
        for (int u = 0; u < kCompactDepth; ++u) {
            if (there(j0, row[u])) v[u] = codes[source[u]];
        }
        if (there(j0, threadIdx.x)) {
            sv = scales[source[kCompactDepth]];
            if (mass != nullptr) mv = mass[source[kCompactDepth]];
        }
    };
    const auto store_rows = [&](uint32_t j0, const uint4 (&v)[kCompactDepth], float sv, float mv) {
#pragma unroll
        for (int u = 0; u < kCompactDepth; ++u) {
            if (there(j0, row[u])) codes[code_row(j0 + row[u]) + chunk[u]] = v[u];
        }
        if (there(j0, threadIdx.x)) {
            const Index at = scale_index(j0 + threadIdx.x);
            scales[at] = sv;
            if (mass != nullptr) mass[at] = mv;
        }
    };
    fetch_tokens(first);
    fetch_sources();
    fetch_tokens(first + rows);
    fetch_rows(first, data[0], scale[0], weight[0]);
    fetch_sources();
    fetch_tokens(first + 2 * rows);
    for (uint32_t j0 = first; j0 < N; j0 += 2 * rows) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t j = j0 + e * rows;
            if (j >= N) break;
            fetch_rows(j + rows, data[1 - e], scale[1 - e], weight[1 - e]);
            fetch_sources();
            fetch_tokens(j + 3 * rows);
            __syncthreads();  // every row of this tile is loaded
            store_rows(j, data[e], scale[e], weight[e]);
        }
    }
}

struct ClearArgs {
    Pool pool;
    float* mass;
    const int64_t* slots;
    int64_t count;
    uint32_t per_slot;  // layers x heads
    FastDiv div_heads;
    FastDiv div_block;
    int32_t* status;
};

// Consecutive threads take consecutive slots: tokens of a block lie side by side
// in each layer and head.
__global__ void __launch_bounds__(256) clear_mass_kernel(ClearArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.count) return;
    const int64_t slot = __ldg(a.slots + i);
    if (slot < 0 || slot >= a.pool.num_blocks * a.pool.block_size) {
        if (blockIdx.y == 0) report_fault(a.status, SDC_FAULT_SLOT_RANGE);
        return;
    }
    uint32_t block, off;
    a.div_block.divmod(static_cast<uint32_t>(slot), block, off);
    float* page = a.mass + block * a.pool.sbs + off;
    for (uint32_t e = blockIdx.y; e < a.per_slot; e += gridDim.y) {
        uint32_t layer, h;
        a.div_heads.divmod(e, layer, h);
        page[layer * a.pool.sls + h * a.pool.shs] = 0.0f;
    }
}

sdc_status_t check_pool_indices(const sdc_page_pool_t* pool) {
    if (pool->num_blocks >= INT32_MAX / pool->block_size || pool->num_layers > INT32_MAX / pool->num_heads) {
        return SDC_STATUS_OVERFLOW;
    }
    return SDC_STATUS_OK;
}

}  // namespace
}  // namespace sdc

using namespace sdc;

extern "C" {

SDC_API sdc_status_t sdc_select_tokens(const sdc_page_pool_t* pool, const float* mass, int64_t batch,
                                       const int32_t* block_tables, int64_t table_stride, const int32_t* context_lens,
                                       int64_t max_context_len, int64_t budget, int64_t recent, int64_t sinks,
                                       int32_t* kept, int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (mass == nullptr || block_tables == nullptr || context_lens == nullptr || kept == nullptr ||
            device_status == nullptr) {
            return SDC_STATUS_NULL_ARGUMENT;
        }
        if (batch < 1 || table_stride < 1 || max_context_len < 1 || budget < 1) return SDC_STATUS_INVALID_SIZE;
        if (recent < 0 || sinks < 0 || recent > budget || sinks > budget - recent) return SDC_STATUS_INVALID_ARGUMENT;
        if (!aligned(mass) || !aligned(block_tables) || !aligned(context_lens) || !aligned(kept) ||
            !aligned(device_status)) {
            return SDC_STATUS_MISALIGNED;
        }
        rc = check_pool_indices(pool);
        if (rc != SDC_STATUS_OK) return rc;
        const int64_t heads = pool->num_layers * pool->num_heads;
        if (max_context_len >= INT32_MAX || budget >= INT32_MAX || batch > INT32_MAX / kSelectCluster / heads ||
            table_stride > (int64_t(1) << 40) / batch) {
            return SDC_STATUS_OVERFLOW;
        }
        SelectArgs a;
        a.pool = to_pool(pool);
        a.mass = mass;
        a.tables = block_tables;
        a.table_stride = table_stride;
        a.lens = context_lens;
        a.max_len = max_context_len;
        a.budget = budget;
        a.recent = recent;
        a.sinks = sinks;
        a.kept = kept;
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.div_heads = FastDiv(static_cast<uint32_t>(pool->num_heads));
        a.div_layers = FastDiv(static_cast<uint32_t>(pool->num_layers));
        a.status = device_status;
        const int64_t items = batch * heads;
        // Four tokens of a group: one 16-byte load where blocks and strides allow
        // (a group past the context's end then stays inside its block).
        a.vec = pool->block_size % 4 == 0 && aligned16(mass) && pool->scale_block_stride % 4 == 0 &&
                pool->scale_layer_stride % 4 == 0 && pool->scale_head_stride % 4 == 0;
        // The fewest blocks that hold a row of keys: a cluster's barriers cost
        // more than its threads bring, unless SMs stay idle (one / two / four /
        // eight blocks of 1024 threads, microseconds: 256 rows of 20000 keys
        // 32 / 68 / 132 / 275, 64 rows of 65536 keys 40 / 28 / 44 / 85, 64 rows
        // of 131072 keys 115 / 57 / 59 / 101, 8 rows of 131072 keys 94 / 45 / 27 /
        // 24).  Short rows: 1021 keys 6.2 with 256 threads, 10 with 32 keys a
        // thread; 256 rows of 8000 keys 12 with 512 threads, 17 with 256.
        cudaStream_t st = as_stream(stream);
        if (max_context_len <= 2048) return launch_select<1, 256, 2>(a, items, st);
        if (max_context_len <= 8192) return launch_select<1, 512, 4>(a, items, st);
        if (max_context_len <= 16384) return launch_select<1, 512, 8>(a, items, st);
        int64_t ranks = 1;
        while (ranks < kSelectCluster && (max_context_len > ranks * 65536 ||
                                          (max_context_len > ranks * 32768 && items * ranks * 2 <= device_sms()))) {
            ranks *= 2;
        }
        switch (ranks) {
            case 1: return launch_select<1, 1024, 8>(a, items, st);
            case 2: return launch_select<2, 1024, 8>(a, items, st);
            case 4: return launch_select<4, 1024, 8>(a, items, st);
            default: return launch_select<8, 1024, 8>(a, items, st);
        }
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

SDC_API sdc_status_t sdc_compact_tokens(const sdc_page_pool_t* pool, float* mass, int64_t batch,
                                        const int32_t* block_tables, int64_t table_stride,
                                        const int32_t* context_lens, const int32_t* kept, int64_t budget,
                                        int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (block_tables == nullptr || context_lens == nullptr || kept == nullptr || device_status == nullptr) {
            return SDC_STATUS_NULL_ARGUMENT;
        }
        if (batch < 1 || table_stride < 1 || budget < 1) return SDC_STATUS_INVALID_SIZE;
        if (!aligned(mass) || !aligned(block_tables) || !aligned(context_lens) || !aligned(kept) ||
            !aligned(device_status)) {
            return SDC_STATUS_MISALIGNED;
        }
        rc = check_pool_indices(pool);
        if (rc != SDC_STATUS_OK) return rc;
        const int64_t heads = pool->num_layers * pool->num_heads;
        if (budget >= INT32_MAX / 2 || batch > INT32_MAX / heads || table_stride > (int64_t(1) << 40) / batch) {
            return SDC_STATUS_OVERFLOW;
        }
        CompactArgs a;
        a.pool = to_pool(pool);
        a.mass = mass;
        a.tables = block_tables;
        a.table_stride = table_stride;
        a.lens = context_lens;
        a.kept = kept;
        a.budget = budget;
        const int64_t chunks = pool->head_dim / 16;
        a.tile_rows = static_cast<int32_t>(
            std::min<int64_t>(kCompactThreads, kCompactThreads * kCompactDepth / chunks));
        a.block_units = static_cast<uint64_t>(pool->code_block_stride / 16);
        a.row_units = static_cast<uint32_t>(chunks);
        a.block_scales = static_cast<uint64_t>(pool->scale_block_stride);
        a.div_chunks = FastDiv(static_cast<uint32_t>(chunks));
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.div_heads = FastDiv(static_cast<uint32_t>(pool->num_heads));
        a.div_layers = FastDiv(static_cast<uint32_t>(pool->num_layers));
        a.status = device_status;
        const dim3 grid(static_cast<unsigned>(batch * heads), 2);
        // rows of a pool of up to 64 GiB of key codes and 16 GiB of scales are
        // addressed in 32 bits: 228 us against 236 in 64 (the large case above)
        const bool narrow = pool->code_block_stride / 16 <= UINT32_MAX / pool->num_blocks &&
                            pool->scale_block_stride <= UINT32_MAX / pool->num_blocks;
        auto kernel = narrow ? compact_tokens_kernel<uint32_t> : compact_tokens_kernel<uint64_t>;
        kernel<<<grid, kCompactThreads, 0, as_stream(stream)>>>(a);
        return launch_status();
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

SDC_API sdc_status_t sdc_clear_mass(const sdc_page_pool_t* pool, float* mass, const int64_t* clear_slots,
                                    int64_t num_clear, int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (mass == nullptr || device_status == nullptr) return SDC_STATUS_NULL_ARGUMENT;
        if (num_clear < 0) return SDC_STATUS_INVALID_SIZE;
        if (num_clear == 0) return SDC_STATUS_OK;
        if (clear_slots == nullptr) return SDC_STATUS_NULL_ARGUMENT;
        if (!aligned(mass) || !aligned(clear_slots) || !aligned(device_status)) return SDC_STATUS_MISALIGNED;
        rc = check_pool_indices(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (num_clear > int64_t(INT32_MAX) * 256) return SDC_STATUS_OVERFLOW;
        ClearArgs a;
        a.pool = to_pool(pool);
        a.mass = mass;
        a.slots = clear_slots;
        a.count = num_clear;
        a.per_slot = static_cast<uint32_t>(pool->num_layers * pool->num_heads);
        a.div_heads = FastDiv(static_cast<uint32_t>(pool->num_heads));
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.status = device_status;
        const dim3 grid(static_cast<unsigned>(ceil_div(num_clear, 256)), std::min(a.per_slot, 65535u));
        clear_mass_kernel<<<grid, 256, 0, as_stream(stream)>>>(a);
        return launch_status();
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

}  // extern "C"
