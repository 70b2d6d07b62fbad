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

constexpr int kWarpsMass = 4;
constexpr int kThreadsMass = kWarpsMass * 32;
constexpr int kTileTokens = 32;
constexpr int kHalf = 16;  // tokens of one MMA
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
    int32_t whole_halves;  // block_size is a multiple of 16: half a tile lies in one block
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

// Query elements 8 i .. 8 i + 7 (the type is the same for the whole grid).
__device__ __forceinline__ void load_query8(const MassArgs& a, int64_t i, float (&x)[8]) {
    if (a.query_dtype == SDC_DTYPE_F32) {
        const float4* p = static_cast<const float4*>(a.query) + 2 * i;
        const float4 u = __ldg(p), v = __ldg(p + 1);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        return;
    }
    const uint4 v = __ldg(static_cast<const uint4*>(a.query) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (a.query_dtype == SDC_DTYPE_BF16) {
            x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        }
    }
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// The codes and scales of one tile in flight: tokens lane / 4 + 8 r, r < 4, each
// thread's quarter of a row.
template <int D>
struct Tile {
    static constexpr int kWords = D / 16;  // 32-bit words per thread and row
    uint32_t code[4][kWords];
    float scale[4];
    uint32_t valid;  // bit r: inside the context and the pool
};

// Not hoisted out of the loop over tiles, where it would spill.
__device__ __forceinline__ uint4 load_shared(const uint4* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
    return v;
}

template <int D, int NT, bool SPLIT>
struct MassKernel {
    static constexpr int KS = D / 16;  // k steps of 16
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int KP = (KS + 1) / 2;  // pairs of k steps: one 16-byte fragment load
    // B fragments: registers while they leave room for the tiles in flight
    static constexpr bool kQueryInRegisters = KP * NT * PARTS * 4 <= 32;
    // tiles in flight per warp: few rows leave registers for a second one
    static constexpr int kDepth = (NT == 1 && D <= 128 && !SPLIT) || (NT <= 2 && D <= 64) ? 2 : 1;
    // blocks per SM, which bounds a thread's registers (128, 168, 255)
    static constexpr int kBlocks = NT == 8 ? 2 : NT == 4 || D == 256 ? 3 : 4;

    struct Shared {
        float2 block_ml[NT * 8];  // this block's (max, sum) per row, read by the cluster
        float2 warp_ml[kWarpsMass][NT * 8];
        float row_max[NT * 8], row_inv[NT * 8];
        float row_scale[NT * 8];
        uint4 query[PARTS][NT][KP][32];  // B fragments of two k steps
        int dropped;                     // a row's weights are not finite
    };

    const MassArgs& a;
    Shared& sh;
    const int32_t* table;
    const int8_t* keys;   // of this layer and head
    const float* scales;
    int64_t T, tile0, tile1;
    int warp, lane;
    int32_t ids;  // lane j: block of half j % 2 of this warp's tile 16 n + j / 2
    uint4 q[kQueryInRegisters ? PARTS * NT * KP : 1];

    __device__ __forceinline__ MassKernel(const MassArgs& args, Shared& shared) : a(args), sh(shared) {}

    // Blocks of this warp's tiles i .. i + 15, two halves each (whole_halves).
    __device__ __forceinline__ void fetch_ids(int i) {
        const int64_t tile = tile0 + warp + static_cast<int64_t>(i + lane / 2) * kWarpsMass;
        const uint32_t t = static_cast<uint32_t>(tile) * kTileTokens + (lane & 1) * kHalf;
        ids = tile < tile1 && t < T ? __ldg(table + a.div_block.div(t)) : -1;
    }

    __device__ __forceinline__ void load_row(const int8_t* row, uint32_t (&code)[Tile<D>::kWords]) const {
        const int c = lane & 3;
        if constexpr (D >= 64) {
#pragma unroll
            for (int g = 0; g < D / 64; ++g) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + 64 * g + 16 * c));
                code[4 * g] = v.x, code[4 * g + 1] = v.y, code[4 * g + 2] = v.z, code[4 * g + 3] = v.w;
            }
        } else if constexpr (D == 32) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + 8 * c));
            code[0] = v.x, code[1] = v.y;
        } else {
            code[0] = __ldg(reinterpret_cast<const uint32_t*>(row + 4 * c));
        }
    }

    // Issues the loads of this warp's i-th tile; past the share, an empty tile.
    __device__ __forceinline__ void load(int i, Tile<D>& out) {
        const int64_t tile = tile0 + warp + static_cast<int64_t>(i) * kWarpsMass;
        if (a.whole_halves && i % 16 == 0) fetch_ids(i);
        const int32_t half_ids[2] = {__shfl_sync(kFullMask, ids, 2 * i & 31), __shfl_sync(kFullMask, ids, (2 * i & 31) + 1)};
        out.valid = 0;
        if (tile >= tile1) return;
        const uint32_t t0 = static_cast<uint32_t>(tile) * kTileTokens;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t half_off = 0;
            if (a.whole_halves) {
                uint32_t j;
                a.div_block.divmod(t0 + half * kHalf, j, half_off);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 2 * half + e;
                const uint32_t t = t0 + (lane >> 2) + 8 * r;
                int64_t block = half_ids[half];
                uint32_t off = half_off + (lane >> 2) + 8 * e;
                if (!a.whole_halves) {
                    uint32_t j;
                    a.div_block.divmod(t, j, off);
                    block = t < T ? __ldg(table + j) : -1;
                }
                out.scale[r] = 0.0f;
#pragma unroll
                for (int w = 0; w < Tile<D>::kWords; ++w) out.code[r][w] = 0u;
                if (t < T && block >= 0 && block < a.pool.num_blocks) {
                    out.valid |= 1u << r;
                    out.scale[r] = __ldg(scales + block * a.pool.sbs + off);
                    load_row(keys + block * a.pool.cbs + static_cast<int64_t>(off) * D, out.code[r]);
                }
            }
        }
    }

    // Scores of a tile in the log2 domain: s[n][r] of token lane / 4 + 8 r for
    // rows 8 n + 2 c + {0, 1}; -inf for hidden and missing tokens.  Both
    // halves of the tile share each B fragment.
    __device__ __forceinline__ void scores(const Tile<D>& tile, int64_t first, const float2 (&scale)[NT],
                                           float2 (&s)[NT][4]) const {
        float d[2][NT][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) d[half][n][0] = d[half][n][1] = d[half][n][2] = d[half][n][3] = 0.0f;
        }
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
            uint32_t f[2][2][4];  // A fragments: [k step][half]
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (2 * kp + e >= KS) break;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    codes_to_f16(tile.code[2 * half][2 * kp + e], f[e][half][0], f[e][half][2]);
                    codes_to_f16(tile.code[2 * half + 1][2 * kp + e], f[e][half][1], f[e][half][3]);
                }
            }
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 b;
                    if constexpr (kQueryInRegisters) {
                        b = q[(p * NT + n) * KP + kp];
                    } else {
                        b = load_shared(&sh.query[p][n][kp][lane]);
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        mma_f16(d[half][n], f[0][half][0], f[0][half][1], f[0][half][2], f[0][half][3], b.x, b.y);
                        if (2 * kp + 1 < KS) {
                            mma_f16(d[half][n], f[1][half][0], f[1][half][1], f[1][half][2], f[1][half][3], b.z, b.w);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float2 ks = make_float2(tile.scale[r], tile.scale[r]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 x = make_float2(d[r >> 1][n][2 * (r & 1)], d[r >> 1][n][2 * (r & 1) + 1]);
                s[n][r] = __fmul2_rn(__fmul2_rn(x, ks), scale[n]);
            }
        }
        // only the window's own positions are hidden from some rows
        const bool whole = first + kTileTokens <= T - a.window + 1;
        if (!whole || !__all_sync(kFullMask, tile.valid == 15u)) {
            const int c = lane & 3;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int64_t last0 = T - a.window + (8 * n + 2 * c) % a.window;
                const int64_t last1 = T - a.window + (8 * n + 2 * c + 1) % a.window;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t t = first + (lane >> 2) + 8 * r;
                    const bool valid = (tile.valid >> r) & 1u;
                    if (!valid || t > last0) s[n][r].x = -INFINITY;
                    if (!valid || t > last1) s[n][r].y = -INFINITY;
                }
            }
        }
    }

    // The query rows (contiguous per KV head) as f16 B fragments: eight
    // elements per thread and step, a row's maximum over the lanes that share it.
    __device__ __forceinline__ void convert_query(int64_t q0) {
        constexpr int kLanes = D / 8;  // per row: 2 .. 32
        const int R = a.rows;
        for (int i = threadIdx.x; i < NT * 8 * kLanes; i += kThreadsMass) {  // whole warps: NT * 8 * kLanes % 32 == 0
            const int r = i / kLanes, part = i % kLanes;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.0f;
            if (r < R) load_query8(a, (q0 + static_cast<int64_t>(r) * D) / 8 + part, x);
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(x[j]));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(__activemask(), m, o));
            const bool finite = m < INFINITY;
            int e = 15;
            if (finite && m > 0.0f) frexpf(m, &e);  // m in [2^(e - 1), 2^e)
            // to a maximum in [2^14, 2^15); a row below 2^-105 stays below it (its scores vanish anyway)
            const int up = min(15 - e, 120);
            // a row that is not finite scores NaN and is dropped below
            if (part == 0) sh.row_scale[r] = finite ? a.score_scale * power_of_two(-up) : NAN;
            const float f = finite ? power_of_two(up) : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {  // four dims: one k step of one quad thread
                const int dim = 8 * part + j;
                const int k = D >= 64 ? (dim >> 6) * 4 + ((dim >> 2) & 3) : D == 32 ? (dim >> 2) & 1 : 0;
                const int c = D >= 64 ? (dim >> 4) & 3 : D == 32 ? dim >> 3 : dim >> 2;
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float u = finite ? x[j + 2 * half] * f : 0.0f, v = finite ? x[j + 2 * half + 1] * f : 0.0f;
                    const __half2 h = __floats2half2_rn(u, v);
                    const float2 back = __half22float2(h);
                    const __half2 l = __floats2half2_rn(u - back.x, v - back.y);
                    hi[half] = *reinterpret_cast<const uint32_t*>(&h);
                    lo[half] = *reinterpret_cast<const uint32_t*>(&l);
                }
                uint2* dst = reinterpret_cast<uint2*>(&sh.query[0][r >> 3][k >> 1][(r & 7) * 4 + c]);
                dst[k & 1] = make_uint2(hi[0], hi[1]);
                if (SPLIT) {
                    dst = reinterpret_cast<uint2*>(&sh.query[PARTS - 1][r >> 3][k >> 1][(r & 7) * 4 + c]);
                    dst[k & 1] = make_uint2(lo[0], lo[1]);
                }
            }
        }
    }
};

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreadsMass, (MassKernel<D, NT, SPLIT>::kBlocks)) observe_attention_kernel(MassArgs a) {
    using K = MassKernel<D, NT, SPLIT>;
    extern __shared__ __align__(16) unsigned char raw[];
    typename K::Shared& sh = *reinterpret_cast<typename K::Shared*>(raw);
    float4* kept = reinterpret_cast<float4*>(raw + (sizeof(typename K::Shared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    K k(a, sh);
    const int warp = k.warp = threadIdx.x >> 5, lane = k.lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x / ranks;
    const int64_t b = item / a.pool.num_heads, h = item - b * a.pool.num_heads;
    const int R = a.rows;

    const int64_t T = k.T = __ldg(a.lens + b);
    if (T < a.window || T > a.max_len || T > a.table_stride * a.pool.block_size) {  // the whole cluster agrees
        if (threadIdx.x == 0 && rank == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
        return;
    }
    k.table = a.tables + b * a.table_stride;
    k.keys = a.pool.keys + a.layer * a.pool.cls + h * a.pool.chs;
    const int64_t scale_base = a.layer * a.pool.sls + h * a.pool.shs;
    k.scales = a.pool.key_scales + scale_base;

    // this block's tiles, dealt to its warps in turn
    const int64_t tiles = (T + kTileTokens - 1) / kTileTokens;
    const int64_t share = (tiles + ranks - 1) / ranks;
    k.tile0 = min(tiles, share * rank);
    k.tile1 = min(tiles, share * (rank + 1));
    const int count = static_cast<int>(max(int64_t(0), k.tile1 - k.tile0 - warp + kWarpsMass - 1) / kWarpsMass);
    const auto first_token = [&](int i) { return (k.tile0 + warp + static_cast<int64_t>(i) * kWarpsMass) * kTileTokens; };

    // the first loads overlap the query's conversion
    Tile<D> flight[K::kDepth];
    k.ids = -1;
#pragma unroll
    for (int e = 0; e < K::kDepth; ++e) k.load(e, flight[e]);
    k.convert_query(item * R * D);
    if (threadIdx.x == 0) sh.dropped = 0;
    __syncthreads();
    const int c = lane & 3;
    if constexpr (K::kQueryInRegisters) {
#pragma unroll
        for (int p = 0; p < K::PARTS; ++p) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < K::KP; ++j) k.q[(p * NT + n) * K::KP + j] = sh.query[p][n][j][lane];
            }
        }
    }
    float2 scale[NT];  // rows 8 n + 2 c + {0, 1}
#pragma unroll
    for (int n = 0; n < NT; ++n) scale[n] = *reinterpret_cast<const float2*>(&sh.row_scale[8 * n + 2 * c]);

    // pass 1: running maximum and sum of each row over this thread's tokens;
    // neg = -max once there is one (a fused scale * product - max would save an
    // instruction, but its exact product differs from the rounded maximum by
    // half an ulp, which is large where scores are)
    float2 neg[NT], l[NT];
    constexpr float kNone = INFINITY;  // neg of a row that has seen no token
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        neg[n] = make_float2(kNone, kNone);
        l[n] = make_float2(0.0f, 0.0f);
    }
    bool missing = false;
    auto pass1 = [&](Tile<D>& tile, int i) {
        float2 s[NT][4];
        const int64_t first = first_token(i);
        k.scores(tile, first, scale, s);
        const int64_t left = T - first - (lane >> 2);  // tokens lane / 4 + 8 r inside the context: r < left / 8
        missing |= tile.valid != (left > 24 ? 15u : left > 16 ? 7u : left > 8 ? 3u : left > 0 ? 1u : 0u);
        k.load(i + K::kDepth, tile);
        if (i < a.kept_tiles) {
            float4* to = kept + (warp * a.kept_tiles + i) * NT * 64 + lane;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                to[n * 64] = make_float4(s[n][0].x, s[n][0].y, s[n][1].x, s[n][1].y);
                to[n * 64 + 32] = make_float4(s[n][2].x, s[n][2].y, s[n][3].x, s[n][3].y);
            }
        }
        float2 top[NT];
        bool higher = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n].x = fmaxf(fmaxf(s[n][0].x, s[n][1].x), fmaxf(s[n][2].x, s[n][3].x));
            top[n].y = fmaxf(fmaxf(s[n][0].y, s[n][1].y), fmaxf(s[n][2].y, s[n][3].y));
            higher |= top[n].x > -neg[n].x || top[n].y > -neg[n].y;
        }
        if (higher) {  // rare once the maxima have settled
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (top[n].x > -neg[n].x) {
                    l[n].x *= exp2_approx(-neg[n].x - top[n].x);  // of nothing: exp2(-inf)
                    neg[n].x = -top[n].x;
                }
                if (top[n].y > -neg[n].y) {
                    l[n].y *= exp2_approx(-neg[n].y - top[n].y);
                    neg[n].y = -top[n].y;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // a row with nothing visible yet: exp2(-inf + 0), no term
            const float2 base = make_float2(neg[n].x == kNone ? 0.0f : neg[n].x, neg[n].y == kNone ? 0.0f : neg[n].y);
            float2 e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float2 u = __fadd2_rn(s[n][r], base);
                e[r] = make_float2(exp2_approx(u.x), exp2_approx(u.y));
            }
            l[n] = __fadd2_rn(l[n], __fadd2_rn(__fadd2_rn(e[0], e[1]), __fadd2_rn(e[2], e[3])));
        }
    };
    int i = 0;
    for (; i < count; i += K::kDepth) {
#pragma unroll
        for (int e = 0; e < K::kDepth; ++e) {
            if (i + e < count) pass1(flight[e], i + e);
        }
    }
    if (missing) report_fault(a.status, SDC_FAULT_BLOCK_RANGE);

    // the eight threads that share rows, the block's warps, the cluster's blocks
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
            float mr = j == 0 ? -neg[n].x : -neg[n].y, lr = j == 0 ? l[n].x : l[n].y;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                merge(mr, lr, __shfl_xor_sync(kFullMask, mr, o), __shfl_xor_sync(kFullMask, lr, o));
            }
            if (lane < 4) sh.warp_ml[warp][8 * n + 2 * lane + j] = make_float2(mr, lr);
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
        for (int o = 0; o < ranks; ++o) {
            const float2 v = *cluster.map_shared_rank(&sh.block_ml[r], o);
            merge(mr, lr, v.x, v.y);
        }
        const bool fine = lr > 0.0f && lr < INFINITY && fabsf(mr) < INFINITY;
        if (!fine) sh.dropped = 1;
        if (r < R && !fine && rank == 0) report_fault(a.status, SDC_FAULT_NONFINITE_VALUE);
        sh.row_max[r] = fine ? -mr : 0.0f;
        sh.row_inv[r] = r < R && fine ? 1.0f / lr : 0.0f;
    }
    // block_ml is read remotely until every block is past this point
    cluster.sync();

    // pass 2
    float2 inv[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        neg[n] = *reinterpret_cast<const float2*>(&sh.row_max[8 * n + 2 * c]);
        inv[n] = *reinterpret_cast<const float2*>(&sh.row_inv[8 * n + 2 * c]);
    }
    const bool dropped = sh.dropped != 0;
    float* mass = a.mass + scale_base;
    auto pass2 = [&](const float2 (&s)[NT][4], int64_t first) {
        float2 w[4] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float2 u = __fadd2_rn(s[n][r], neg[n]);
                float2 e = make_float2(exp2_approx(u.x), exp2_approx(u.y));
                if (dropped) {  // its terms may be NaN
                    if (!(inv[n].x > 0.0f)) e.x = 0.0f;
                    if (!(inv[n].y > 0.0f)) e.y = 0.0f;
                }
                w[r] = __ffma2_rn(e, inv[n], w[r]);
            }
        }
        // the quad's partial sums: thread c ends with token lane / 4 + 8 c
        const float x0 = w[0].x + w[0].y, x1 = w[1].x + w[1].y, x2 = w[2].x + w[2].y, x3 = w[3].x + w[3].y;
        const bool odd = c & 1, upper = c & 2;
        const float y0 = (odd ? x1 : x0) + __shfl_xor_sync(kFullMask, odd ? x0 : x1, 1);  // token 0 or 1
        const float y1 = (odd ? x3 : x2) + __shfl_xor_sync(kFullMask, odd ? x2 : x3, 1);  // token 2 or 3
        const float sum = (upper ? y1 : y0) + __shfl_xor_sync(kFullMask, upper ? y0 : y1, 2);
        const uint32_t t = static_cast<uint32_t>(first) + (lane >> 2) + 8 * c;
        if (t < T) {
            uint32_t j, off;
            a.div_block.divmod(t, j, off);
            const int64_t block = __ldg(k.table + j);
            // one thread per token: the add at L2 is a plain sum, without the load's latency
            if (block >= 0 && block < a.pool.num_blocks) atomicAdd(mass + block * a.pool.sbs + off, sum);
        }
    };
    const int held = min(count, a.kept_tiles);
    for (i = 0; i < held; ++i) {
        float2 s[NT][4];
        const float4* from = kept + (warp * a.kept_tiles + i) * NT * 64 + lane;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 u = from[n * 64], v = from[n * 64 + 32];
            s[n][0] = make_float2(u.x, u.y), s[n][1] = make_float2(u.z, u.w);
            s[n][2] = make_float2(v.x, v.y), s[n][3] = make_float2(v.z, v.w);
        }
        pass2(s, first_token(i));
    }
    if (i < count) {  // the tiles that were not kept
        if (a.whole_halves) k.fetch_ids(i / 16 * 16);
#pragma unroll
        for (int e = 0; e < K::kDepth; ++e) k.load(i + e, flight[e]);
        for (; i < count; i += K::kDepth) {
#pragma unroll
            for (int e = 0; e < K::kDepth; ++e) {
                if (i + e < count) {
                    float2 s[NT][4];
                    k.scores(flight[e], first_token(i + e), scale, s);
                    k.load(i + e + K::kDepth, flight[e]);
                    pass2(s, first_token(i + e));
                }
            }
        }
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
    constexpr size_t kTileBytes = size_t(NT) * 8 * kTileTokens * sizeof(float);
    constexpr size_t kBudget = 220 * 1024 / K::kBlocks - 1024;
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
        if (!aligned16(query) || (reinterpret_cast<uintptr_t>(mass) & 3u)) {
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
        a.whole_halves = pool->block_size % kHalf == 0;
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
