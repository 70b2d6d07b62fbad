// Attention mass: the softmax weight every cached token gets from a window's
// queries, added to the token's running sum in its page.
//
// For sequence b, KV head h and query row r = (g, i) (query head h G + g,
// window row i, position p = T - window + i):
//   s_rt = (q_r . k_t) / sqrt(D) for t <= p,   k_t = code_t * scale_t,
//   mass[t] += sum_r exp(s_rt) / sum_u exp(s_ru).
// A weight needs its row's sum over the whole context, so there are two
// launches.  The first reads every key once: a block takes a chunk of one
// (sequence, KV head), its warps take 32-token tiles, form all rows' scores with
// f16 tensor-core MMAs, keep the running maximum and sum of each row and store the
// scores (float32, in the MMA's own register layout).  The second merges the
// chunks' maxima and sums, turns the scores into weights, sums them over the
// rows and adds them to the mass.  A stored score costs 4 bytes a row against
// the head_dim + 4 bytes of the key and is read back from L2 where it fits;
// forming them again would read the keys a second time.  A short context's
// scores stay in the shared memory of the one block that takes it, in one
// launch.  A token's mass is updated by one thread, so the result does not
// depend on scheduling.
//
// Measured (B200, device time): 32 sequences of 1024 to 8192 tokens, 8 KV heads of
// 128, 20 rows: 76 us, 53 of them the first launch (155 MB of keys read, 113 MB of
// scores written: 5 TB/s) and 22 to 27 the second (113 MB read); 64 x 1100
// tokens, head_dim 64, 4 rows: 17 us in one launch, 22 in two; one context of
// 131071 tokens, 24 rows: 62 us; of 8192 tokens, 16 rows: 9.9 us.  Large calls
// are bound by latency (16 warps of 128 registers an SM issue in half of the
// slots): leaving out the conversions, the MMAs or the softmax changes the time
// by 0 to 5 %, the score stores by 9 %, the key loads by 15 %, the scores of
// padded rows (17 % of their traffic) by nothing.  Small ones are bound by the
// tiles that a warp takes one after the other (0.7 to 1.2 us each) and the
// launches.  A form with the scores of a cluster's blocks in shared memory took
// 86, 22 and 140 us: sixteen blocks of a cluster wait for one another, and a few
// contexts cannot fill the GPU.
//
// Precision.  INT8 codes are exact in f16.  A query row is scaled by a power
// of two to a maximum in [2^14, 2^15) and held in f16: exact for bf16 and f16
// inputs (bf16 elements smaller than 2^-32 of the row's largest lose bits below
// 2^-39 of it), and as two f16 parts (22 bits) for f32 inputs, whose scores
// take two MMAs.  Products are exact and accumulate in float32.
//
// Operand layout.  A warp copies its next tile's rows into shared memory while it
// works on this one (cp.async, two stages).  mma.m16n8k16 takes the keys as A (16
// tokens) and the query rows as B (8 per MMA).  Only the pairing of A's and B's k
// matters, so thread c of a quad takes dims 16 c .. 16 c + 15 of each 64: one
// 16-byte shared load per key row feeds four MMAs.  Byte permutes turn codes
// into f16 (1024 + 128 + code, less 1152).

#include <algorithm>
#include <cmath>

#include "host_common.h"

namespace sdc {
namespace {

constexpr int kWarpsMass = 4;
constexpr int kThreadsMass = kWarpsMass * 32;
constexpr int kTileTokens = 32;
constexpr int kHalf = 16;  // tokens of one MMA
constexpr int64_t kWarpTiles = 8;  // tiles a warp takes of a chunk, at most
constexpr int64_t kMergeChunks = 128;
constexpr int64_t kSMs = 148;  // a constant: the workspace's size and the call plan alike, whatever the current device
constexpr int kThreadsWeigh = 128;
constexpr int kMaxRows = 64;

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
    float score_scale;   // log2(e) / sqrt(D)
    int32_t whole_halves;  // block_size is a multiple of 16: half a tile lies in one block
    int32_t max_tiles;    // of a sequence: the stride of an item's scores
    int32_t chunk_tiles;  // tiles one block takes
    int32_t chunks;       // at most, per item
    uint32_t item0;       // first item of this launch
    float4* scores;       // [item][max_tiles][rows / 8][2][lane]
    float2* ml;           // [item][chunks][rows]: (max, sum)
    FastDiv div_chunks;
    FastDiv div_block;
    FastDiv div_heads;
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

// One tile of keys in shared memory, and which of its tokens are there.
template <int D>
struct Stage {
    int8_t code[kTileTokens * D];  // row r's 16-byte chunk i at chunk i ^ swizzle(r)
    float scale[kTileTokens];
    // Rows of 128 bytes and more: the eight lanes of a load phase read four
    // chunks of two rows, which this keeps in different banks.
    static __device__ __forceinline__ int swizzle(int row) {
        return D >= 128 ? ((row & 1) << 2) | ((row >> 1) & 3) : 0;
    }
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// Asynchronous copies; with fill they write zeros and read nothing.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool fill) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(dst)), "l"(src), "r"(fill ? 0 : 16)
                 : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src, bool fill) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_address(dst)), "l"(src), "r"(fill ? 0 : 4)
                 : "memory");
}

// Not hoisted out of the loop over tiles, where it would spill.
__device__ __forceinline__ uint4 load_shared(const uint4* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(shared_address(p)));
    return v;
}

template <int D, int NT, bool SPLIT>
struct MassKernel {
    static constexpr int kDim = D, kTiles = NT;
    static constexpr int KS = D / 16;  // k steps of 16
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int KP = (KS + 1) / 2;  // pairs of k steps: one 16-byte fragment load
    // B fragments: registers while they leave room for the tiles in flight
    static constexpr bool kQueryInRegisters = KP * NT * PARTS * 4 <= 32;
    static constexpr int kStages = 2;  // tiles of a warp in shared memory (three: 5 to 15 % slower)
    // blocks per SM, which bounds a thread's registers to 128, 168 or 255: no
    // spills but a few words with three eights of rows (float32 at head_dim 64: 24
    // bytes stored, 56 loaded; five blocks of 96 registers: 17 % slower)
    static constexpr int kBlocks = NT == 8 ? 2 : NT == 4 || D == 256 ? 3 : 4;

    struct Shared {
        float2 warp_ml[kWarpsMass][NT * 8];
        float row_scale[NT * 8];
        uint4 query[PARTS][NT][KP][32];  // B fragments of two k steps
        __align__(16) Stage<D> stage[kWarpsMass][kStages];
    };

    const MassArgs& a;
    Shared& sh;
    const int32_t* table;
    const int8_t* keys;   // of this layer and head
    const float* scales;
    int32_t T, tile0, tile1;
    int warp, lane;
    int32_t ids;  // lane j: block of half j % 2 of this warp's tile 16 n + j / 2
    uint4 q[kQueryInRegisters ? PARTS * NT * KP : 1];

    __device__ __forceinline__ MassKernel(const MassArgs& args, Shared& shared) : a(args), sh(shared) {}

    __device__ __forceinline__ int first_token(int i) const { return (tile0 + warp + i * kWarpsMass) * kTileTokens; }

    // Blocks of this warp's tiles i .. i + 15, two halves each (whole_halves).
    __device__ __forceinline__ void fetch_ids(int i) {
        const int t = first_token(i + lane / 2) + (lane & 1) * kHalf;
        ids = t < T && t < tile1 * kTileTokens ? __ldg(table + a.div_block.div(static_cast<uint32_t>(t))) : -1;
    }

    __device__ __forceinline__ bool in_pool(int64_t block) const { return block >= 0 && block < a.pool.num_blocks; }

    // Starts the copies of this warp's i-th tile, one commit group whether or
    // not there is such a tile; returns the mask of its tokens that are in the
    // context and the pool.  Consecutive lanes copy the chunks of a row.
    __device__ __forceinline__ uint32_t load(int i, Stage<D>& to) {
        constexpr int kChunks = D / 16, kRows = 32 / kChunks;  // of a row; rows of one copy instruction
        const int t0 = first_token(i);
        uint32_t mask = 0;
        if (t0 < tile1 * kTileTokens) {
            const int row0 = lane / kChunks, chunk = lane % kChunks;
            if (a.whole_halves && i % 16 == 0) fetch_ids(i);
            bool whole = a.whole_halves && t0 + kTileTokens <= T;
            int64_t block[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                block[half] = __shfl_sync(kFullMask, ids, (2 * i & 31) + half);
                whole = whole && in_pool(block[half]);
            }
            if (whole) {
                mask = kFullMask;
                const int8_t* src[2];
                const float* scale[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t j, off;
                    a.div_block.divmod(static_cast<uint32_t>(t0 + half * kHalf), j, off);
                    src[half] = keys + block[half] * a.pool.cbs + static_cast<int64_t>(off) * D + row0 * D + chunk * 16;
                    scale[half] = scales + block[half] * a.pool.sbs + off;
                }
                copy4(&to.scale[lane], (lane < kHalf ? scale[0] : scale[1]) + (lane & 15), false);
#pragma unroll
                for (int u = 0; u < kChunks; ++u) {
                    const int row = u * kRows + row0;
                    const int8_t* from;
                    if constexpr (kChunks == 1) {
                        from = (lane < kHalf ? src[0] : src[1] - kHalf * D);
                    } else {
                        from = src[u / (kChunks / 2)] + (u % (kChunks / 2)) * kRows * D;
                    }
                    copy16(&to.code[row * D + (chunk ^ Stage<D>::swizzle(row)) * 16], from, false);
                }
            } else {
                const int t = t0 + lane;
                uint32_t j, off;
                a.div_block.divmod(static_cast<uint32_t>(t), j, off);
                const int64_t mine = t < T ? __ldg(table + j) : -1;  // lane l: the block of token l
                const bool ok = t < T && in_pool(mine);
                mask = __ballot_sync(kFullMask, ok);
                const int64_t code_at = ok ? mine * a.pool.cbs + static_cast<int64_t>(off) * D : 0;
                copy4(&to.scale[lane], scales + (ok ? mine * a.pool.sbs + off : 0), !ok);
#pragma unroll
                for (int u = 0; u < kChunks; ++u) {
                    const int row = u * kRows + row0;
                    const int64_t from = __shfl_sync(kFullMask, code_at, row);
                    copy16(&to.code[row * D + (chunk ^ Stage<D>::swizzle(row)) * 16], keys + from + chunk * 16,
                           !((mask >> row) & 1u));
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return mask;
    }

    // The oldest of the stages in flight has landed, for all lanes.
    static __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
    }

    // Scores of a tile in the log2 domain: s[n][r] of token lane / 4 + 8 r for
    // rows 8 n + 2 c + {0, 1}; -inf for hidden and missing tokens.  Both
    // halves of the tile share each B fragment.
    __device__ __forceinline__ void scores(const Stage<D>& from, uint32_t mask, int first, const float2 (&scale)[NT],
                                           float2 (&s)[NT][4]) const {
        constexpr int kWords = D >= 64 ? 4 : D / 16;  // 32-bit words of one load: a k step each
        const int c = lane & 3, g = lane >> 2;
        float d[2][NT][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) d[half][n][0] = d[half][n][1] = d[half][n][2] = d[half][n][3] = 0.0f;
        }
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += kWords) {
            uint32_t code[4][kWords];  // tokens g + 8 r
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = g + 8 * r;
                const int8_t* p = from.code + row * D;
                if constexpr (D >= 64) {
                    const uint4 v = load_shared(
                        reinterpret_cast<const uint4*>(p + ((k0 + c) ^ Stage<D>::swizzle(row)) * 16));
                    code[r][0] = v.x, code[r][1] = v.y, code[r][2] = v.z, code[r][3] = v.w;
                } else if constexpr (D == 32) {
                    const uint2 v = *reinterpret_cast<const uint2*>(p + 8 * c);
                    code[r][0] = v.x, code[r][1] = v.y;
                } else {
                    code[r][0] = *reinterpret_cast<const uint32_t*>(p + 4 * c);
                }
            }
#pragma unroll
            for (int w0 = 0; w0 < kWords; w0 += 2) {  // two k steps: one B fragment load
                uint32_t f[2][2][4];  // A fragments: [k step][half]
#pragma unroll
                for (int e = 0; e < 2 && w0 + e < kWords; ++e) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        codes_to_f16(code[2 * half][w0 + e], f[e][half][0], f[e][half][2]);
                        codes_to_f16(code[2 * half + 1][w0 + e], f[e][half][1], f[e][half][3]);
                    }
                }
                const int kp = (k0 + w0) / 2;
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
                            if (w0 + 1 < kWords) {
                                mma_f16(d[half][n], f[1][half][0], f[1][half][1], f[1][half][2], f[1][half][3], b.z,
                                        b.w);
                            }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float ks = from.scale[g + 8 * r];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 x = make_float2(d[r >> 1][n][2 * (r & 1)], d[r >> 1][n][2 * (r & 1) + 1]);
                s[n][r] = __fmul2_rn(__fmul2_rn(x, make_float2(ks, ks)), scale[n]);
            }
        }
        // only the window's own positions are hidden from some rows
        if (mask != kFullMask || first + kTileTokens > T - a.window + 1) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int last0 = T - a.window + (8 * n + 2 * c) % a.window;
                const int last1 = T - a.window + (8 * n + 2 * c + 1) % a.window;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = first + g + 8 * r;
                    const bool valid = (mask >> (g + 8 * r)) & 1u;
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
        constexpr int kItems = NT * 8 * kLanes;
        const int R = a.rows;
        // whole warps take part in the shuffles: head_dim 16 with an odd number of
        // eights fills half of the last one
        for (int i = threadIdx.x; i < (kItems + 31) / 32 * 32; i += kThreadsMass) {
            const int r = i / kLanes, part = i % kLanes;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.0f;
            if (r < R) load_query8(a, (q0 + static_cast<int64_t>(r) * D) / 8 + part, x);
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(x[j]));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFullMask, m, o));
            if (i >= kItems) continue;
            const bool finite = m < INFINITY;
            // m in [2^(e - 1), 2^e), to a maximum in [2^14, 2^15); a row below
            // 2^-105 stays below it (its scores vanish anyway)
            const int e = finite ? static_cast<int>(__float_as_uint(m) >> 23) - 126 : 15;
            const int up = min(15 - e, 120);
            // a row that is not finite scores NaN and is dropped below
            if (part == 0) sh.row_scale[r] = finite ? a.score_scale * power_of_two(-up) : NAN;
            const float f = power_of_two(up);
            if (!finite) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j += 4) {  // four dims: one k step of one quad thread
                const int dim = 8 * part + j;
                const int k = D >= 64 ? (dim >> 6) * 4 + ((dim >> 2) & 3) : D == 32 ? (dim >> 2) & 1 : 0;
                const int c = D >= 64 ? (dim >> 4) & 3 : D == 32 ? dim >> 3 : dim >> 2;
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float u = x[j + 2 * half] * f, v = x[j + 2 * half + 1] * f;
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

__device__ __forceinline__ void merge(float& m0, float& l0, float m1, float l1) {
    const float top = fmaxf(m0, m1);
    const float base = top == -INFINITY ? 0.0f : top;
    l0 = l0 * exp2_approx(m0 - base) + l1 * exp2_approx(m1 - base);
    m0 = top;
}

// Running maximum and sum of rows 8 n + 2 c + {0, 1} over a thread's tokens;
// neg = -max once there is one (a fused scale * product - max would save an
// instruction, but its exact product differs from the rounded maximum by half an
// ulp, which is large where scores are).
template <int NT>
struct RowSums {
    static constexpr float kNone = INFINITY;  // neg of a row that has seen no token
    float2 neg[NT], l[NT];

    __device__ __forceinline__ RowSums() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            neg[n] = make_float2(kNone, kNone);
            l[n] = make_float2(0.0f, 0.0f);
        }
    }
    __device__ __forceinline__ void add(const float2 (&s)[NT][4]) {
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
    }
    // (max, sum) of every row over the warp
    __device__ __forceinline__ void write(float2* rows, int lane) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float mine = j == 0 ? -neg[n].x : -neg[n].y;
                float top = mine, lr = j == 0 ? l[n].x : l[n].y;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
                lr *= exp2_approx(mine - (top == -INFINITY ? 0.0f : top));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) lr += __shfl_xor_sync(kFullMask, lr, o);
                if (lane < 4) rows[8 * n + 2 * lane + j] = make_float2(top, lr);
            }
        }
    }
};

// What turns scores into weights: -max and 1 / sum of every row, in shared memory.
template <int NT>
struct RowFactors {
    float neg[NT * 8], inv[NT * 8];
    int dropped;  // a row's weights are not finite

    // Row r of the whole context (one thread each, after `dropped` is cleared).
    __device__ __forceinline__ void set(const MassArgs& a, int r, float top, float sum, bool report) {
        const bool fine = sum > 0.0f && sum < INFINITY && fabsf(top) < INFINITY;
        if (!fine) dropped = 1;
        if (r < a.rows && !fine && report) report_fault(a.status, SDC_FAULT_NONFINITE_VALUE);
        neg[r] = fine ? -top : 0.0f;
        inv[r] = r < a.rows && fine ? 1.0f / sum : 0.0f;
    }
};

template <int NT>
struct Weigher {
    float2 neg[NT], inv[NT];
    bool drop;
    const int32_t* table;
    float* mass;

    __device__ __forceinline__ Weigher(const MassArgs& a, const RowFactors<NT>& f, uint32_t b, uint32_t h, int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            neg[n] = make_float2(f.neg[8 * n + 2 * c], f.neg[8 * n + 2 * c + 1]);
            inv[n] = make_float2(f.inv[8 * n + 2 * c], f.inv[8 * n + 2 * c + 1]);
        }
        drop = f.dropped != 0;
        table = a.tables + b * a.table_stride;
        mass = a.mass + a.layer * a.pool.sls + h * a.pool.shs;
    }
    // Adds the weights of the tile of tokens `first` ..; q: its scores as stored.
    __device__ __forceinline__ void add(const MassArgs& a, const float4 (&q)[2 * NT], int first, int T, int lane) const {
        const int c = lane & 3;
        float2 w[4] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 u = q[2 * n], v = q[2 * n + 1];
            const float2 s[4] = {make_float2(u.x, u.y), make_float2(u.z, u.w), make_float2(v.x, v.y),
                                 make_float2(v.z, v.w)};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float2 x = __fadd2_rn(s[r], neg[n]);
                float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                if (drop) {  // its terms may be NaN
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
        const int t = first + (lane >> 2) + 8 * c;
        if (t < T) {
            uint32_t j, off;
            a.div_block.divmod(static_cast<uint32_t>(t), j, off);
            const int64_t block = __ldg(table + j);
            // one thread per token: the add at L2 is a plain sum, without the load's latency
            if (block >= 0 && block < a.pool.num_blocks) atomicAdd(mass + block * a.pool.sbs + off, sum);
        }
    }
};

// Where a block stands: its item (sequence, KV head) and its tiles.
struct Chunk {
    uint32_t local;  // item of this launch
    uint32_t item, b, h;
    int index, T, tiles, tile0, tile1;
    bool fine;  // the context is inside the bounds
    __device__ __forceinline__ explicit Chunk(const MassArgs& a) {
        uint32_t i;
        a.div_chunks.divmod(blockIdx.x, local, i);
        index = static_cast<int>(i);
        item = a.item0 + local;
        a.div_heads.divmod(item, b, h);
        T = __ldg(a.lens + b);
        fine = T >= a.window && T <= a.max_len && T <= a.table_stride * a.pool.block_size;
        tiles = (T + kTileTokens - 1) / kTileTokens;
        tile0 = min(tiles, index * a.chunk_tiles);
        tile1 = min(tiles, (index + 1) * a.chunk_tiles);
    }
};

// The block's tiles: forms their scores, hands them to store(tile, scores) and
// leaves every warp's (max, sum) of each row in sh.warp_ml, behind a barrier.
template <class K, class Store>
__device__ __forceinline__ void form_scores(const MassArgs& a, const Chunk& at, typename K::Shared& sh, Store store) {
    constexpr int NT = K::kTiles;
    K k(a, sh);
    const int warp = k.warp = threadIdx.x >> 5, lane = k.lane = threadIdx.x & 31;
    k.T = at.T, k.tile0 = at.tile0, k.tile1 = at.tile1;
    k.table = a.tables + at.b * a.table_stride;
    k.keys = a.pool.keys + a.layer * a.pool.cls + at.h * a.pool.chs;
    k.scales = a.pool.key_scales + a.layer * a.pool.sls + at.h * a.pool.shs;
    const int count = max(0, k.tile1 - k.tile0 - warp + kWarpsMass - 1) / kWarpsMass;

    // the first copies overlap the query's conversion
    k.ids = -1;
    uint32_t mask[K::kStages];
#pragma unroll
    for (int e = 0; e < K::kStages; ++e) mask[e] = k.load(e, sh.stage[warp][e]);
    k.convert_query(static_cast<int64_t>(at.item) * a.rows * K::kDim);
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

    RowSums<NT> sums;
    bool missing = false;
    auto take = [&](auto& stage, uint32_t& present, int i) {
        float2 s[NT][4];
        K::wait();
        k.scores(stage, present, k.first_token(i), scale, s);
        const int left = at.T - k.first_token(i);
        missing |= present != (left >= kTileTokens ? kFullMask : (1u << left) - 1u);
        __syncwarp();  // the stage has been read
        present = k.load(i + K::kStages, stage);
        store(k.tile0 + warp + i * kWarpsMass, s);
        sums.add(s);
    };
    for (int i = 0; i < count; i += K::kStages) {
#pragma unroll
        for (int e = 0; e < K::kStages; ++e) {
            if (i + e < count) take(sh.stage[warp][e], mask[e], i + e);
        }
    }
    if (missing && lane == 0) report_fault(a.status, SDC_FAULT_BLOCK_RANGE);
    sums.write(sh.warp_ml[warp], lane);
    __syncthreads();
}

// Eight scores of a thread as two quads: s[n] for n < NT, a plane of a quad per lane.
template <int NT>
__device__ __forceinline__ void store_scores(float4* to, const float2 (&s)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        to[n * 64] = make_float4(s[n][0].x, s[n][0].y, s[n][1].x, s[n][1].y);
        to[n * 64 + 32] = make_float4(s[n][2].x, s[n][2].y, s[n][3].x, s[n][3].y);
    }
}

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreadsMass, (MassKernel<D, NT, SPLIT>::kBlocks)) observe_scores_kernel(MassArgs a) {
    using K = MassKernel<D, NT, SPLIT>;
    extern __shared__ __align__(16) unsigned char raw[];
    typename K::Shared& sh = *reinterpret_cast<typename K::Shared*>(raw);
    // the second launch may be scheduled; it waits for this grid's stores
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Chunk at(a);
    if (!at.fine && threadIdx.x == 0 && at.index == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
    if (!at.fine || at.tile0 >= at.tile1) return;
    float4* scores = a.scores + static_cast<int64_t>(at.local) * a.max_tiles * (NT * 64) + (threadIdx.x & 31);
    form_scores<K>(a, at, sh, [&](int tile, const float2 (&s)[NT][4]) {
        store_scores<NT>(scores + static_cast<int64_t>(tile) * (NT * 64), s);
    });
    if (threadIdx.x < NT * 8) {
        float mr = -INFINITY, lr = 0.0f;
        for (int w = 0; w < kWarpsMass; ++w) {
            const float2 v = sh.warp_ml[w][threadIdx.x];
            merge(mr, lr, v.x, v.y);
        }
        a.ml[(static_cast<int64_t>(at.local) * a.chunks + at.index) * (NT * 8) + threadIdx.x] = make_float2(mr, lr);
    }
}

// Scores of a tile in shared memory: as above without the padded rows of the last
// eight, so that the usual few rows leave room for more blocks (64 x 1000 to
// 1200 tokens, 4 rows: 17.4 us, 21.9 in two launches).
template <int NT>
struct ShortTile {
    int pairs;  // of rows in the last eight
    int lane, c;

    __host__ __device__ static constexpr int pairs_of(int rows) { return (rows - 8 * (NT - 1) + 1) / 2; }
    __host__ __device__ static constexpr int quads(int pairs) { return 64 * (NT - 1) + 16 * pairs; }

    __device__ __forceinline__ ShortTile(int rows, int lane_) : pairs(pairs_of(rows)), lane(lane_), c(lane_ & 3) {}
    __device__ __forceinline__ int last() const { return 64 * (NT - 1) + (lane >> 2) * pairs + c; }
    __device__ __forceinline__ void store(float4* to, const float2 (&s)[NT][4]) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 u = make_float4(s[n][0].x, s[n][0].y, s[n][1].x, s[n][1].y);
            const float4 v = make_float4(s[n][2].x, s[n][2].y, s[n][3].x, s[n][3].y);
            if (n < NT - 1) {
                to[n * 64 + lane] = u, to[n * 64 + 32 + lane] = v;
            } else if (c < pairs) {
                to[last()] = u, to[last() + 8 * pairs] = v;
            }
        }
    }
    __device__ __forceinline__ void load(float4 (&q)[2 * NT], const float4* from) const {
#pragma unroll
        for (int n = 0; n < 2 * (NT - 1); ++n) q[n] = from[n * 32 + lane];
        q[2 * NT - 2] = q[2 * NT - 1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c < pairs) q[2 * NT - 2] = from[last()], q[2 * NT - 1] = from[last() + 8 * pairs];
    }
};

// Both halves in one block for contexts whose scores its shared memory holds: no
// second launch and no workspace.
template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreadsMass, (MassKernel<D, NT, SPLIT>::kBlocks)) observe_short_kernel(MassArgs a) {
    using K = MassKernel<D, NT, SPLIT>;
    extern __shared__ __align__(16) unsigned char raw[];
    typename K::Shared& sh = *reinterpret_cast<typename K::Shared*>(raw);
    float4* scores = reinterpret_cast<float4*>(raw + sizeof(typename K::Shared));
    __shared__ RowFactors<NT> factors;
    const Chunk at(a);  // the whole context
    if (!at.fine) {
        if (threadIdx.x == 0) report_fault(a.status, SDC_FAULT_CONTEXT_RANGE);
        return;
    }
    if (threadIdx.x == 0) factors.dropped = 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const ShortTile<NT> layout(a.rows, lane);
    const int quads = layout.quads(layout.pairs);
    form_scores<K>(a, at, sh,
                   [&](int tile, const float2 (&s)[NT][4]) { layout.store(scores + tile * quads, s); });
    if (threadIdx.x < NT * 8) {
        float mr = -INFINITY, lr = 0.0f;
        for (int w = 0; w < kWarpsMass; ++w) {
            const float2 v = sh.warp_ml[w][threadIdx.x];
            merge(mr, lr, v.x, v.y);
        }
        factors.set(a, threadIdx.x, mr, lr, true);
    }
    __syncthreads();
    const Weigher<NT> weigh(a, factors, at.b, at.h, lane & 3);
    for (int tile = warp; tile < at.tiles; tile += kWarpsMass) {  // a warp's own tiles
        float4 q[2 * NT];
        layout.load(q, scores + tile * quads);
        weigh.add(a, q, tile * kTileTokens, at.T, lane);
    }
}

// Weights from the stored scores, in the same tile layout.
template <int NT>
__global__ void __launch_bounds__(kThreadsWeigh) observe_weights_kernel(MassArgs a) {
    constexpr int kRows = NT * 8, kParts = kThreadsWeigh / kRows;
    __shared__ float2 part_ml[kParts][kRows];
    __shared__ RowFactors<NT> factors;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Chunk at(a);
    if (!at.fine || at.tile0 >= at.tile1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a tile's scores are loaded while the one before is weighed, the first
    // while the rows' sums meet
    const float4* scores = a.scores + static_cast<int64_t>(at.local) * a.max_tiles * (NT * 64) + lane;
    float4 next[2 * NT];
    const auto fetch = [&](int tile) {
        if (tile >= at.tile1) return;
        const float4* from = scores + static_cast<int64_t>(tile) * (NT * 64);
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) next[n] = from[n * 32];
    };
    fetch(at.tile0 + warp);
    if (threadIdx.x == 0) factors.dropped = 0;
    {
        const int r = threadIdx.x % kRows, part = threadIdx.x / kRows;
        const int filled = (at.tiles + a.chunk_tiles - 1) / a.chunk_tiles;
        const float2* ml = a.ml + static_cast<int64_t>(at.local) * a.chunks * kRows + r;
        float mr = -INFINITY, lr = 0.0f;
        for (int i = part; i < filled && part < kParts; i += kParts) {
            const float2 v = ml[i * kRows];
            merge(mr, lr, v.x, v.y);
        }
        if (part < kParts) part_ml[part][r] = make_float2(mr, lr);
    }
    __syncthreads();
    if (threadIdx.x < kRows) {
        float mr = -INFINITY, lr = 0.0f;
        for (int i = 0; i < kParts; ++i) merge(mr, lr, part_ml[i][threadIdx.x].x, part_ml[i][threadIdx.x].y);
        factors.set(a, threadIdx.x, mr, lr, at.index == 0);
    }
    __syncthreads();
    const Weigher<NT> weigh(a, factors, at.b, at.h, lane & 3);
    for (int tile = at.tile0 + warp; tile < at.tile1; tile += kThreadsWeigh / 32) {
        float4 now[2 * NT];
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) now[n] = next[n];
        fetch(tile + kThreadsWeigh / 32);
        weigh.add(a, now, tile * kTileTokens, at.T, lane);
    }
}

constexpr int padded_tiles_of(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : rows <= 32 ? 4 : 8; }

// Work split of a call.
struct MassPlan {
    int64_t items, rows8, max_tiles, chunk_tiles, chunks;
    size_t ml_bytes, score_bytes;  // of one item
    bool single;                   // one launch
    size_t short_bytes;            // its scores
};

constexpr int64_t kSingleSmem = 226 * 1024;  // and RowFactors

// The head dims and rows of the models served here; the others take the two
// launches, which hold for every shape.
template <int D, int NT>
constexpr bool kHasSingle = (D == 64 || D == 128) && NT <= 3;

// Blocks of observe_short_kernel that an SM holds with this much for their
// scores, and of observe_scores_kernel; {0, 0} where there is no such kernel.
// The larger form of the query stands for both.
struct Residents {
    int64_t single, split;
};

template <int D, int NT>
Residents residents_of(size_t short_bytes) {
    static_assert(kHasSingle<D, NT>);
    constexpr int64_t kSmemSM = 228 * 1024, kSmemReserved = 1024;
    using K = MassKernel<D, NT, true>;
    const int64_t smem = static_cast<int64_t>(sizeof(typename K::Shared) + sizeof(RowFactors<NT>) + short_bytes);
    if (smem > kSingleSmem) return {0, K::kBlocks};
    return {std::min<int64_t>(K::kBlocks, kSmemSM / (smem + kSmemReserved)), K::kBlocks};
}

template <int D>
Residents residents_of(int64_t rows8, size_t short_bytes) {
    return rows8 == 1   ? residents_of<D, 1>(short_bytes)
           : rows8 == 2 ? residents_of<D, 2>(short_bytes)
           : rows8 == 3 ? residents_of<D, 3>(short_bytes)
                        : Residents{0, 0};
}

// One launch saves 1 to 2 us on the device and 5 us of a call (1 x 131 tokens,
// 32 query heads of 64: 11 us against 17).  Its block takes a whole context, so a
// warp takes at most four tiles, or twice what a warp of two launches
// takes: 8 contexts of 64 tokens, 8 KV heads, 3.8 us against 5.7, of 512 6.3
// against 6.2, of 1024 9.3 against 7.2; 64 of 1100 16.6 against 21.6.  And its
// blocks have to find room: where the scores in their shared memory leave fewer of
// them on an SM, a grid of more than one wave lost up to 10 % (64 x 768 tokens,
// 8 float32 rows of 128: 25.3 us against 22.7).
bool single_launch(int64_t head_dim, int64_t rows8, int64_t items, int64_t max_tiles, int64_t warp_tiles,
                   size_t short_bytes) {
    const Residents r = head_dim == 64    ? residents_of<64>(rows8, short_bytes)
                        : head_dim == 128 ? residents_of<128>(rows8, short_bytes)
                                          : Residents{0, 0};
    if (r.single == 0) return false;
    const int64_t serial = ceil_div(max_tiles, kWarpsMass);
    if (r.single == r.split) return serial <= std::max<int64_t>(4, 2 * warp_tiles);
    return items <= kSMs * r.single && serial <= std::max<int64_t>(4, warp_tiles);
}

MassPlan plan_mass(int64_t batch, int64_t heads, int64_t head_dim, int64_t rows, int64_t max_len) {
    MassPlan p;
    p.items = batch * heads;
    p.rows8 = padded_tiles_of(rows);
    p.max_tiles = ceil_div(max_len, kTileTokens);
    // even chunks: as many as fill the GPU's warps, down to a tile a warp (16 rows of
    // 128 over 8 KV heads, one context of 2048 tokens: 6.6 us, 14.5 with eight tiles a
    // warp; of 8192 tokens: 9.9 and 14.9), up to eight tiles a warp, and few enough
    // to merge (2 pairs of 32768 tokens: 128 chunks 10.6 us, 256 12.5)
    const int64_t fill = ceil_div(p.items * p.max_tiles, kSMs * 4 * kWarpsMass);
    const int64_t warp_tiles =
        std::min<int64_t>(kWarpTiles, std::max(fill, ceil_div(p.max_tiles, kMergeChunks * kWarpsMass)));
    p.chunks = ceil_div(p.max_tiles, kWarpsMass * warp_tiles);
    p.chunk_tiles = ceil_div(ceil_div(p.max_tiles, p.chunks), kWarpsMass) * kWarpsMass;
    p.chunks = ceil_div(p.max_tiles, p.chunk_tiles);
    p.score_bytes = static_cast<size_t>(p.max_tiles * p.rows8) * 8 * kTileTokens * sizeof(float);
    const int quads = p.rows8 == 1   ? ShortTile<1>::quads(ShortTile<1>::pairs_of(static_cast<int>(rows)))
                      : p.rows8 == 2 ? ShortTile<2>::quads(ShortTile<2>::pairs_of(static_cast<int>(rows)))
                                     : ShortTile<3>::quads(ShortTile<3>::pairs_of(static_cast<int>(rows)));
    p.short_bytes = static_cast<size_t>(p.max_tiles) * quads * sizeof(float4);
    p.single = single_launch(head_dim, p.rows8, p.items, p.max_tiles, warp_tiles, p.short_bytes);
    if (p.single) p.chunks = 1, p.chunk_tiles = p.max_tiles;
    p.ml_bytes = static_cast<size_t>(p.chunks * p.rows8 * 8) * sizeof(float2);
    return p;
}

template <int D, int NT, bool SPLIT>
sdc_status_t launch_rows(MassArgs a, const MassPlan& p, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    using K = MassKernel<D, NT, SPLIT>;
    if constexpr (kHasSingle<D, NT>) {
        if (p.single) {
            auto kernel = observe_short_kernel<D, NT, SPLIT>;
            const size_t smem = sizeof(typename K::Shared) + p.short_bytes;
            // beyond 48 KiB, the kernel's static part (factors, at most 208 bytes) included;
            // always the same limit: another thread's call may come between this and the launch
            constexpr size_t kStatic = 256;
            static_assert(sizeof(RowFactors<NT>) + 16 <= kStatic);
            if (smem + kStatic > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                                   static_cast<int>(kSingleSmem)) != cudaSuccess) {
                return SDC_STATUS_CUDA_ERROR;
            }
            a.item0 = 0;
            kernel<<<static_cast<unsigned>(p.items), kThreadsMass, smem, st>>>(a);
            return launch_status();
        }
    }
    auto kernel = observe_scores_kernel<D, NT, SPLIT>;
    constexpr size_t smem = sizeof(typename K::Shared);
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)) != cudaSuccess) {
        return SDC_STATUS_CUDA_ERROR;
    }
    // as many items a round as the workspace holds
    const int64_t fit = static_cast<int64_t>(workspace_bytes / (p.ml_bytes + p.score_bytes));
    const int64_t round = std::min(p.items, fit);
    for (int64_t item = 0; item < p.items; item += round) {
        const int64_t n = std::min(round, p.items - item);
        a.item0 = static_cast<uint32_t>(item);
        a.scores = static_cast<float4*>(workspace);
        a.ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.score_bytes * static_cast<size_t>(round));
        const unsigned blocks = static_cast<unsigned>(n * p.chunks);
        kernel<<<blocks, kThreadsMass, smem, st>>>(a);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(kThreadsWeigh);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, observe_weights_kernel<NT>, a) != cudaSuccess) return SDC_STATUS_CUDA_ERROR;
    }
    return launch_status();
}

// Rows are padded to 8, 16, 24, 32 or 64 (the MMA's n in steps of 8).
template <int D, bool SPLIT>
sdc_status_t launch_dim(const MassArgs& a, const MassPlan& p, void* ws, size_t bytes, cudaStream_t st) {
    if (p.rows8 == 1) return launch_rows<D, 1, SPLIT>(a, p, ws, bytes, st);
    if (p.rows8 == 2) return launch_rows<D, 2, SPLIT>(a, p, ws, bytes, st);
    if (p.rows8 == 3) return launch_rows<D, 3, SPLIT>(a, p, ws, bytes, st);
    if (p.rows8 == 4) return launch_rows<D, 4, SPLIT>(a, p, ws, bytes, st);
    return launch_rows<D, 8, SPLIT>(a, p, ws, bytes, st);
}

template <bool SPLIT>
sdc_status_t launch_query(const MassArgs& a, const MassPlan& p, void* ws, size_t bytes, cudaStream_t st) {
    switch (a.pool.head_dim) {
        case 16: return launch_dim<16, SPLIT>(a, p, ws, bytes, st);
        case 32: return launch_dim<32, SPLIT>(a, p, ws, bytes, st);
        case 64: return launch_dim<64, SPLIT>(a, p, ws, bytes, st);
        case 128: return launch_dim<128, SPLIT>(a, p, ws, bytes, st);
        case 256: return launch_dim<256, SPLIT>(a, p, ws, bytes, st);
        default: return SDC_STATUS_UNSUPPORTED;
    }
}

sdc_status_t check_mass_shape(int64_t batch, int64_t query_heads, int64_t kv_heads, int64_t head_dim, int64_t window,
                              int64_t max_len, MassPlan* p) {
    if (batch < 1 || query_heads < 1 || kv_heads < 1 || head_dim < 1 || window < 1 || max_len < 1) return SDC_STATUS_INVALID_SIZE;
    if (query_heads % kv_heads) return SDC_STATUS_INVALID_ARGUMENT;
    if (window > max_len) return SDC_STATUS_INVALID_SIZE;
    const int64_t group = query_heads / kv_heads;
    if (group > kMaxRows || window > kMaxRows / group) return SDC_STATUS_UNSUPPORTED;
    if (max_len >= INT32_MAX / 2 || batch > INT32_MAX / kv_heads) return SDC_STATUS_OVERFLOW;
    *p = plan_mass(batch, kv_heads, head_dim, group * window, max_len);
    if (p->items > INT32_MAX / p->chunks) return SDC_STATUS_OVERFLOW;
    return SDC_STATUS_OK;
}

}  // namespace
}  // namespace sdc

using namespace sdc;

extern "C" {

SDC_API sdc_status_t sdc_observe_workspace_size(int64_t batch, int64_t num_query_heads, int64_t num_kv_heads,
                                                int64_t head_dim, int64_t window, int64_t max_context_len,
                                                size_t* least, size_t* most) {
    if (least == nullptr || most == nullptr) return SDC_STATUS_NULL_ARGUMENT;
    MassPlan p;
    const sdc_status_t rc = check_mass_shape(batch, num_query_heads, num_kv_heads, head_dim, window, max_context_len, &p);
    if (rc != SDC_STATUS_OK) return rc;
    *least = p.single ? 0 : p.ml_bytes + p.score_bytes;
    *most = *least * static_cast<size_t>(p.items);
    return SDC_STATUS_OK;
}

SDC_API sdc_status_t sdc_observe_attention(const sdc_page_pool_t* pool, int64_t layer, float* mass, const void* query,
                                           int query_dtype, int64_t batch, int64_t num_query_heads, int64_t window,
                                           const int32_t* block_tables, int64_t table_stride,
                                           const int32_t* context_lens, int64_t max_context_len, void* workspace,
                                           size_t workspace_bytes, int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (mass == nullptr || query == nullptr || block_tables == nullptr || context_lens == nullptr ||
            device_status == nullptr) {
            return SDC_STATUS_NULL_ARGUMENT;
        }
        if (layer < 0 || layer >= pool->num_layers) return SDC_STATUS_INVALID_SIZE;
        if (table_stride < 1) return SDC_STATUS_INVALID_SIZE;
        MassPlan p;
        rc = check_mass_shape(batch, num_query_heads, pool->num_heads, pool->head_dim, window, max_context_len, &p);
        if (rc != SDC_STATUS_OK) return rc;
        if (query_dtype != SDC_DTYPE_BF16 && query_dtype != SDC_DTYPE_F16 && query_dtype != SDC_DTYPE_F32) {
            return SDC_STATUS_UNSUPPORTED;
        }
        if (!p.single && workspace == nullptr) return SDC_STATUS_NULL_ARGUMENT;
        if (!aligned16(query) || !aligned16(workspace) || !aligned(mass) || !aligned(block_tables) ||
            !aligned(context_lens) || !aligned(device_status)) {
            return SDC_STATUS_MISALIGNED;
        }
        if (!p.single && workspace_bytes < p.ml_bytes + p.score_bytes) return SDC_STATUS_INVALID_SIZE;
        if (pool->block_size >= INT32_MAX || table_stride > (int64_t(1) << 40) / batch) return SDC_STATUS_OVERFLOW;
        MassArgs a;
        a.pool = to_pool(pool);
        a.layer = layer;
        a.mass = mass;
        a.query = query;
        a.query_dtype = query_dtype;
        a.rows = static_cast<int32_t>(num_query_heads / pool->num_heads * window);
        a.window = static_cast<int32_t>(window);
        a.tables = block_tables;
        a.table_stride = table_stride;
        a.lens = context_lens;
        a.max_len = max_context_len;
        a.score_scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(pool->head_dim)));
        a.whole_halves = pool->block_size % kHalf == 0;
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.div_heads = FastDiv(static_cast<uint32_t>(pool->num_heads));
        a.status = device_status;
        a.max_tiles = static_cast<int32_t>(p.max_tiles);
        a.chunk_tiles = static_cast<int32_t>(p.chunk_tiles);
        a.chunks = static_cast<int32_t>(p.chunks);
        a.div_chunks = FastDiv(static_cast<uint32_t>(p.chunks));
        cudaStream_t st = as_stream(stream);
        return query_dtype == SDC_DTYPE_F32 ? launch_query<true>(a, p, workspace, workspace_bytes, st)
                                            : launch_query<false>(a, p, workspace, workspace_bytes, st);
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

}  // extern "C"
