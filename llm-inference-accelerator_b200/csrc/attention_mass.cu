// Attention mass: the softmax weight every cached token gets from a window's
// queries, added to the token's running sum in its page.
//
// For sequence b, KV head h and query row r = (g, i) (query head h G + g,
// window row i, position p = T - window + i):
//   s_rt = (q_r . k_t) / sqrt(D) for t <= p,   k_t = code_t * scale_t,
//   mass[t] += sum_r exp(s_rt) / sum_u exp(s_ru).
// Every key row is needed twice, once for the rows' sums and once for the
// weights, but HBM should deliver it once.  A thread-block cluster owns one
// (sequence, KV head); its blocks split the context into contiguous shares.
//   pass 1: a warp takes 16-token tiles, forms all rows' scores with f16
//     tensor-core MMAs and keeps the running maximum and sum of each row; the
//     scores of the first tiles of a block's share stay in shared memory, in
//     the MMA's own register layout;
//   exchange: the blocks' maxima and sums meet over distributed shared memory;
//   pass 2: the weights of each tile, from the kept scores or from scores
//     formed again (from L2: the tiles that did not fit were read by this
//     cluster a moment ago), summed over the rows and added to the mass.
// One launch, no workspace; a token's mass is updated by one thread, so the
// result does not depend on scheduling.
//
// Precision.  INT8 codes are exact in f16.  A query row is scaled by a power
// of two to a maximum in [2^14, 2^15) and held in f16: exact for bf16 and f16
// inputs (bf16 elements smaller than 2^-32 of the row's largest lose bits below
// 2^-39 of it), and as two f16 parts (22 bits) for f32 inputs, whose scores
// take two MMAs.  Products are exact and accumulate in float32.
//
// Operand layout.  mma.m16n8k16 with the keys as A (16 tokens) and the query
// rows as B (8 per MMA).  Only the pairing of A's and B's k matters, so thread
// c of a quad takes dims 16 c .. 16 c + 15 of each 64: one 16-byte load per
// key row straight from the page feeds four MMAs, with no shared-memory
// staging; byte permutes turn codes into f16 (1024 + 128 + code, less 1152).

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "host_common.h"

namespace sdc {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarpsMass = 8;
constexpr int kThreadsMass = kWarpsMass * 32;
constexpr int kTileTokens = 16;
constexpr int kMaxRows = 64;
constexpr int kMaxCluster = 16;

struct MassArgs {
    Pool pool;
    int64_t layer;
    float* mass;
    const void* query;
    int32_t query_dtype;
    int32_t rows;    // query rows per KV head: group * window
    int32_t window;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* lens;
    int64_t max_len;
    int32_t kept_tiles;  // tiles a warp keeps in shared memory
    float score_scale;   // log2(e) / sqrt(D)
    FastDiv div_block;
    int32_t* status;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float r;  // 2 ulp; weights below 2^-126 flush to zero
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four codes as two f16 pairs, exact: the biased byte u = code + 128 becomes
// the low mantissa byte of 1024 + u.
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), bias);
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
}

// Element i of the query (its type is the same for the whole grid).
__device__ __forceinline__ float query_value(const MassArgs& a, int64_t i) {
    if (a.query_dtype == SDC_DTYPE_F32) return static_cast<const float*>(a.query)[i];
    if (a.query_dtype == SDC_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.query)[i]);
    return __half2float(static_cast<const __half*>(a.query)[i]);
}

// The codes and scales of one tile in flight: rows lane / 4 and lane / 4 + 8,
// each thread's quarter of a row.
template <int D>
struct Tile {
    static constexpr int kWords = D / 16;  // 32-bit words per thread and row
    uint32_t code[2][kWords];
    float scale[2];
    bool valid[2];  // inside the context and the pool
};

template <int D, int NT, bool SPLIT>
struct MassKernel {
    static constexpr int KS = D / 16;  // k steps of 16
    static constexpr int PARTS = SPLIT ? 2 : 1;
    // B fragments: registers while they leave room for the tiles in flight
    static constexpr bool kQueryInRegisters = KS * NT * PARTS * 2 <= 64;

    struct Shared {
        float2 block_ml[NT * 8];                // this block's (max, sum) per row, read by the cluster
        float2 warp_ml[kWarpsMass][NT * 8];
        float row_max[NT * 8], row_inv[NT * 8];
        float row_scale[NT * 8];
        uint2 query[PARTS][NT][KS][32];         // B fragments
        int bad;
    };

    static __device__ __forceinline__ void load(const MassArgs& a, const int32_t* table, int64_t code_base,
                                                int64_t scale_base, int64_t tile, int64_t T, int lane, Tile<D>& out) {
        constexpr int W = Tile<D>::kWords;
        const int c = lane & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t t = tile * kTileTokens + (lane >> 2) + 8 * r;
            out.valid[r] = false;
            out.scale[r] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) out.code[r][w] = 0u;
            if (t >= T) continue;
            uint32_t j, off;
            a.div_block.divmod(static_cast<uint32_t>(t), j, off);
            const int64_t block = __ldg(table + j);
            if (block < 0 || block >= a.pool.num_blocks) continue;
            out.valid[r] = true;
            out.scale[r] = __ldg(a.pool.key_scales + block * a.pool.sbs + scale_base + off);
            const int8_t* row = a.pool.keys + block * a.pool.cbs + code_base + static_cast<int64_t>(off) * D;
            if constexpr (D >= 64) {
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + 64 * g + 16 * c));
                    out.code[r][4 * g] = v.x, out.code[r][4 * g + 1] = v.y;
                    out.code[r][4 * g + 2] = v.z, out.code[r][4 * g + 3] = v.w;
                }
            } else if constexpr (D == 32) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + 8 * c));
                out.code[r][0] = v.x, out.code[r][1] = v.y;
            } else {
                out.code[r][0] = __ldg(reinterpret_cast<const uint32_t*>(row + 4 * c));
            }
        }
    }

    // Scores in the log2 domain of a tile: s[n][0..1] for token lane / 4 and
    // rows 8 n + 2 c + {0, 1}, s[n][2..3] for token lane / 4 + 8.
    static __device__ __forceinline__ void scores(const MassArgs& a, const Shared& sh,
                                                  const uint2 (&q)[kQueryInRegisters ? PARTS * NT * KS : 1],
                                                  const Tile<D>& tile, int64_t first, int64_t T, int lane,
                                                  float (&s)[NT][4]) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t a0, a1, a2, a3;
            codes_to_f16(tile.code[0][k], a0, a2);
            codes_to_f16(tile.code[1][k], a1, a3);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint2 b;
                    if constexpr (kQueryInRegisters) {
                        b = q[(p * NT + n) * KS + k];
                    } else {
                        b = sh.query[p][n][k][lane];
                    }
                    mma_f16(s[n], a0, a1, a2, a3, b.x, b.y);
                }
            }
        }
        const int c = lane & 3;
        // only the window's own positions are hidden from some rows
        const bool masked = first + kTileTokens > T - a.window;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 8 * n + 2 * c + (e & 1), r = e >> 1;
                float x = s[n][e] * sh.row_scale[row] * tile.scale[r];
                if (masked) {
                    const int64_t t = first + (lane >> 2) + 8 * r;
                    if (t > T - a.window + row % a.window) x = -INFINITY;
                }
                s[n][e] = tile.valid[r] ? x : -INFINITY;
            }
        }
    }
};

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreadsMass) observe_attention_kernel(MassArgs a) {
    using K = MassKernel<D, NT, SPLIT>;
    constexpr int KS = K::KS;
    extern __shared__ __align__(16) unsigned char raw[];
    typename K::Shared& sh = *reinterpret_cast<typename K::Shared*>(raw);
    float4* kept = reinterpret_cast<float4*>(raw + (sizeof(typename K::Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x / ranks;
    const int64_t b = item / a.pool.num_heads, h = item - b * a.pool.num_heads;
    const int R = a.rows;

    const int64_t T = __ldg(a.lens + b);
    if (T < a.window || T > a.max_len || T > a.table_stride * a.pool.block_size) {  // the whole cluster agrees
        if (threadIdx.x == 0 && rank == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
        return;
    }
    const int32_t* table = a.tables + b * a.table_stride;
    const int64_t code_base = a.layer * a.pool.cls + h * a.pool.chs;
    const int64_t scale_base = a.layer * a.pool.sls + h * a.pool.shs;

    // this block's tiles, dealt to its warps in turn
    const int64_t tiles = (T + kTileTokens - 1) / kTileTokens;
    const int64_t share = (tiles + ranks - 1) / ranks;
    const int64_t tile0 = min(tiles, share * rank), tile1 = min(tiles, share * (rank + 1));

    // two tiles in flight per warp: the first loads overlap the query's conversion
    Tile<D> flight[2];
    K::load(a, table, code_base, scale_base, tile0 + warp, tile0 + warp < tile1 ? T : 0, lane, flight[0]);
    K::load(a, table, code_base, scale_base, tile0 + warp + kWarpsMass, tile0 + warp + kWarpsMass < tile1 ? T : 0,
            lane, flight[1]);

    // query rows (contiguous per KV head) to f16 fragments
    const int64_t q0 = item * R * D;
    if (threadIdx.x == 0) sh.bad = 0;
    for (int r = warp; r < NT * 8; r += kWarpsMass) {
        float m = 0.0f;
        if (r < R) {
            for (int d = lane; d < D; d += 32) m = max_nan(m, fabsf(query_value(a, q0 + r * D + d)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFullMask, m, o));
        const bool finite = m < INFINITY;
        int e = 0;
        if (finite && m > 0.0f) frexpf(m, &e);  // m in [2^(e - 1), 2^e)
        const int up = 15 - e;
        if (lane == 0) {
            // a row that is not finite scores NaN and is left out below
            sh.row_scale[r] = finite ? ldexpf(a.score_scale, -up) : NAN;
        }
        for (int i = lane; i < KS * 8; i += 32) {  // (k step, half, quad thread): two dims each
            const int k = i >> 3, half = (i >> 2) & 1, c = i & 3;
            // k step 4 g + w of a 64-dim group g, word w: dims 64 g + 16 c + 4 w + 2 half
            const int dim = D >= 64 ? 64 * (k >> 2) + 16 * c + 4 * (k & 3) + 2 * half : (D / 4) * c + 4 * k + 2 * half;
            float x = 0.0f, y = 0.0f;
            if (r < R && finite) {
                x = ldexpf(query_value(a, q0 + r * D + dim), up);
                y = ldexpf(query_value(a, q0 + r * D + dim + 1), up);
            }
            const __half2 hi = __floats2half2_rn(x, y);
            uint32_t* dst = reinterpret_cast<uint32_t*>(&sh.query[0][r >> 3][k][(r & 7) * 4 + c]);
            dst[half] = *reinterpret_cast<const uint32_t*>(&hi);
            if (SPLIT) {
                const float2 back = __half22float2(hi);
                const __half2 lo = __floats2half2_rn(x - back.x, y - back.y);
                dst = reinterpret_cast<uint32_t*>(&sh.query[K::PARTS - 1][r >> 3][k][(r & 7) * 4 + c]);
                dst[half] = *reinterpret_cast<const uint32_t*>(&lo);
            }
        }
    }
    __syncthreads();
    uint2 qf[K::kQueryInRegisters ? K::PARTS * NT * KS : 1];
    if constexpr (K::kQueryInRegisters) {
#pragma unroll
        for (int p = 0; p < K::PARTS; ++p) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int k = 0; k < KS; ++k) qf[(p * NT + n) * KS + k] = sh.query[p][n][k][lane];
            }
        }
    }

    // pass 1: running (max, sum) of rows 8 n + 2 c + {0, 1} over this thread's tokens
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }
    bool missing = false;
    int count = 0;
    auto pass1 = [&](Tile<D>& tile, int64_t at) {
        float s[NT][4];
        K::scores(a, sh, qf, tile, at * kTileTokens, T, lane, s);
        const int64_t t = at * kTileTokens + (lane >> 2);
        missing |= (t < T && !tile.valid[0]) || (t + 8 < T && !tile.valid[1]);
        K::load(a, table, code_base, scale_base, at + 2 * kWarpsMass, at + 2 * kWarpsMass < tile1 ? T : 0, lane, tile);
        if (count < a.kept_tiles) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                kept[((warp * a.kept_tiles + count) * NT + n) * 32 + lane] =
                    make_float4(s[n][0], s[n][1], s[n][2], s[n][3]);
            }
        }
        ++count;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float top = fmaxf(s[n][j], s[n][j + 2]);
                if (top > m[n][j]) {  // rare once the maximum has settled
                    l[n][j] *= exp2_approx(m[n][j] - top);
                    m[n][j] = top;
                }
                // a row with nothing visible yet keeps its maximum at -inf: no term
                const float base = m[n][j] == -INFINITY ? 0.0f : m[n][j];
                l[n][j] += exp2_approx(s[n][j] - base) + exp2_approx(s[n][j + 2] - base);
            }
        }
    };
    int64_t at = tile0 + warp;
    for (; at + kWarpsMass < tile1; at += 2 * kWarpsMass) {
        pass1(flight[0], at);
        pass1(flight[1], at + kWarpsMass);
    }
    if (at < tile1) pass1(flight[0], at);
    if (missing) report_fault(a.status, SDC_FAULT_BLOCK_RANGE);

    // the quad rows' eight threads, the block's warps, the cluster's blocks
    auto merge = [](float& m0, float& l0, float m1, float l1) {
        const float top = fmaxf(m0, m1);
        const float base = top == -INFINITY ? 0.0f : top;
        l0 = l0 * exp2_approx(m0 - base) + l1 * exp2_approx(m1 - base);
        m0 = top;
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                merge(m[n][j], l[n][j], __shfl_xor_sync(kFullMask, m[n][j], o),
                      __shfl_xor_sync(kFullMask, l[n][j], o));
            }
            if (lane < 4) sh.warp_ml[warp][8 * n + 2 * lane + j] = make_float2(m[n][j], l[n][j]);
        }
    }
    __syncthreads();
    if (threadIdx.x < NT * 8) {
        float mr = -INFINITY, lr = 0.0f;
        for (int w = 0; w < kWarpsMass; ++w) {
            const float2 v = sh.warp_ml[w][threadIdx.x];
            merge(mr, lr, v.x, v.y);
        }
        sh.block_ml[threadIdx.x] = make_float2(mr, lr);
    }
    cluster.sync();
    if (threadIdx.x < NT * 8) {
        const int r = threadIdx.x;
        float mr = -INFINITY, lr = 0.0f;
        for (int c = 0; c < ranks; ++c) {
            const float2 v = *cluster.map_shared_rank(&sh.block_ml[r], c);
            merge(mr, lr, v.x, v.y);
        }
        const bool fine = lr > 0.0f && lr < INFINITY && mr < INFINITY;
        if (r < R && !fine && rank == 0) report_fault(a.status, SDC_FAULT_NONFINITE_VALUE);
        sh.row_max[r] = fine ? mr : 0.0f;
        sh.row_inv[r] = r < R && fine ? 1.0f / lr : 0.0f;
    }
    // block_ml is read remotely until every block is past this point
    cluster.sync();

    // pass 2
    float top[NT][2], inv[NT][2];
    const int c = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[n][j] = sh.row_max[8 * n + 2 * c + j];
            inv[n][j] = sh.row_inv[8 * n + 2 * c + j];
        }
    }
    float* mass = a.mass + scale_base;
    auto pass2 = [&](const float (&s)[NT][4], int64_t tile) {
        float w0 = 0.0f, w1 = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // a row left out may hold NaN scores: its factor is zero, its terms are dropped
                const float e0 = exp2_approx(s[n][j] - top[n][j]), e1 = exp2_approx(s[n][j + 2] - top[n][j]);
                w0 += inv[n][j] > 0.0f ? e0 * inv[n][j] : 0.0f;
                w1 += inv[n][j] > 0.0f ? e1 * inv[n][j] : 0.0f;
            }
        }
        w0 += __shfl_xor_sync(kFullMask, w0, 1);
        w1 += __shfl_xor_sync(kFullMask, w1, 1);
        w0 += __shfl_xor_sync(kFullMask, w0, 2);
        w1 += __shfl_xor_sync(kFullMask, w1, 2);
        const int64_t t = tile * kTileTokens + (lane >> 2) + 8 * c;  // threads 0 and 1 of a quad
        if (c < 2 && t < T) {
            uint32_t j, off;
            a.div_block.divmod(static_cast<uint32_t>(t), j, off);
            const int64_t block = __ldg(table + j);
            // one thread per token: the add at L2 is a plain sum, without the load's latency
            if (block >= 0 && block < a.pool.num_blocks) atomicAdd(mass + block * a.pool.sbs + off, c == 0 ? w0 : w1);
        }
    };
    at = tile0 + warp;
    for (int i = 0; i < a.kept_tiles && at < tile1; ++i, at += kWarpsMass) {
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 v = kept[((warp * a.kept_tiles + i) * NT + n) * 32 + lane];
            s[n][0] = v.x, s[n][1] = v.y, s[n][2] = v.z, s[n][3] = v.w;
        }
        pass2(s, at);
    }
    if (at < tile1) {  // the tiles that were not kept
        K::load(a, table, code_base, scale_base, at, T, lane, flight[0]);
        K::load(a, table, code_base, scale_base, at + kWarpsMass, at + kWarpsMass < tile1 ? T : 0, lane, flight[1]);
        auto again = [&](Tile<D>& tile, int64_t which) {
            float s[NT][4];
            K::scores(a, sh, qf, tile, which * kTileTokens, T, lane, s);
            K::load(a, table, code_base, scale_base, which + 2 * kWarpsMass,
                    which + 2 * kWarpsMass < tile1 ? T : 0, lane, tile);
            pass2(s, which);
        };
        for (; at + kWarpsMass < tile1; at += 2 * kWarpsMass) {
            again(flight[0], at);
            again(flight[1], at + kWarpsMass);
        }
        if (at < tile1) again(flight[0], at);
    }
}

template <int D, int NT, bool SPLIT>
sdc_status_t launch_rows(MassArgs a, int64_t items, cudaStream_t st) {
    using K = MassKernel<D, NT, SPLIT>;
    auto kernel = observe_attention_kernel<D, NT, SPLIT>;
    const int64_t tiles = ceil_div(a.max_len, kTileTokens);
    // Blocks per (sequence, KV head): enough that the grid fills the SMs
    // twice and that a block's scores fit its half of an SM's shared memory,
    // as long as each warp of a block still has a tile.
    constexpr size_t kFixed = (sizeof(typename K::Shared) + 15) / 16 * 16;
    constexpr size_t kTileBytes = size_t(NT) * 32 * 16;
    constexpr size_t kBudget = 100 * 1024;
    const int64_t room = kBudget > kFixed ? int64_t((kBudget - kFixed) / (kTileBytes * kWarpsMass)) : 0;
    int ranks = 1;
    while (ranks < kMaxCluster && tiles > int64_t(ranks) * kWarpsMass &&
           (items * ranks < int64_t(device_sms()) * 2 || ceil_div(tiles, ranks * kWarpsMass) > room)) {
        ranks *= 2;
    }
    a.kept_tiles = static_cast<int32_t>(std::min<int64_t>(room, ceil_div(ceil_div(tiles, ranks), kWarpsMass)));
    const size_t smem = kFixed + kTileBytes * kWarpsMass * static_cast<size_t>(a.kept_tiles);
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)) != cudaSuccess) {
        return SDC_STATUS_CUDA_ERROR;
    }
    if (ranks > 8 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        return SDC_STATUS_CUDA_ERROR;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
    cfg.blockDim = dim3(kThreadsMass);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return SDC_STATUS_CUDA_ERROR;
    return launch_status();
}

// Rows are padded to 8, 16, 24, 32 or 64 (the MMA's n in steps of 8).
template <int D, bool SPLIT>
sdc_status_t launch_dim(const MassArgs& a, int64_t items, cudaStream_t st) {
    if (a.rows <= 8) return launch_rows<D, 1, SPLIT>(a, items, st);
    if (a.rows <= 16) return launch_rows<D, 2, SPLIT>(a, items, st);
    if (a.rows <= 24) return launch_rows<D, 3, SPLIT>(a, items, st);
    if (a.rows <= 32) return launch_rows<D, 4, SPLIT>(a, items, st);
    return launch_rows<D, 8, SPLIT>(a, items, st);
}

template <bool SPLIT>
sdc_status_t launch_query(const MassArgs& a, int64_t items, cudaStream_t st) {
    switch (a.pool.head_dim) {
        case 16: return launch_dim<16, SPLIT>(a, items, st);
        case 32: return launch_dim<32, SPLIT>(a, items, st);
        case 64: return launch_dim<64, SPLIT>(a, items, st);
        case 128: return launch_dim<128, SPLIT>(a, items, st);
        case 256: return launch_dim<256, SPLIT>(a, items, st);
        default: return SDC_STATUS_UNSUPPORTED;
    }
}

}  // namespace
}  // namespace sdc

using namespace sdc;

extern "C" {

SDC_API sdc_status_t sdc_observe_attention(const sdc_page_pool_t* pool, int64_t layer, float* mass, const void* query,
                                           int query_dtype, int64_t batch, int64_t num_query_heads, int64_t window,
                                           const int32_t* block_tables, int64_t table_stride,
                                           const int32_t* context_lens, int64_t max_context_len,
                                           int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (mass == nullptr || query == nullptr || block_tables == nullptr || context_lens == nullptr ||
            device_status == nullptr) {
            return SDC_STATUS_NULL_ARGUMENT;
        }
        if (layer < 0 || layer >= pool->num_layers) return SDC_STATUS_INVALID_SIZE;
        if (batch < 1 || num_query_heads < 1 || window < 1 || max_context_len < 1 || table_stride < 1) {
            return SDC_STATUS_INVALID_SIZE;
        }
        if (num_query_heads % pool->num_heads) return SDC_STATUS_INVALID_ARGUMENT;
        if (window > max_context_len) return SDC_STATUS_INVALID_SIZE;
        const int64_t group = num_query_heads / pool->num_heads;
        if (group > kMaxRows || window > kMaxRows / group) return SDC_STATUS_UNSUPPORTED;
        if (query_dtype != SDC_DTYPE_BF16 && query_dtype != SDC_DTYPE_F16 && query_dtype != SDC_DTYPE_F32) {
            return SDC_STATUS_UNSUPPORTED;
        }
        if (reinterpret_cast<uintptr_t>(query) % dtype_size(query_dtype) || (reinterpret_cast<uintptr_t>(mass) & 3u)) {
            return SDC_STATUS_MISALIGNED;
        }
        if (max_context_len >= INT32_MAX || batch > INT32_MAX / kMaxCluster / pool->num_heads ||
            pool->block_size >= INT32_MAX || table_stride > (int64_t(1) << 40) / batch) {
            return SDC_STATUS_OVERFLOW;
        }
        MassArgs a;
        a.pool = to_pool(pool);
        a.layer = layer;
        a.mass = mass;
        a.query = query;
        a.query_dtype = query_dtype;
        a.rows = static_cast<int32_t>(group * window);
        a.window = static_cast<int32_t>(window);
        a.tables = block_tables;
        a.table_stride = table_stride;
        a.lens = context_lens;
        a.max_len = max_context_len;
        a.score_scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(pool->head_dim)));
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.status = device_status;
        const int64_t items = batch * pool->num_heads;
        cudaStream_t st = as_stream(stream);
        return query_dtype == SDC_DTYPE_F32 ? launch_query<true>(a, items, st) : launch_query<false>(a, items, st);
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

}  // extern "C"
