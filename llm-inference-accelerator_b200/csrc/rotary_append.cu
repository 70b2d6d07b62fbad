// Per-head normalisation, position rotation and quantize-append of one
// layer's projections in one launch.
//
// For every token, with x a query or key head of D elements:
//   y = x * w / sqrt(mean(x^2) + eps)                  (where weights are given)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)       pairs of the first rotary_dim
// with (c, s) the cosine and sine of position * frequency from a float32
// table.  Queries are stored in the attention's [batch, head, token, dim]
// layout in their own type, rounded once; keys, and values as they come, are
// quantized from float32 into their page slot with the append rule
// (kv_pages.cu): the rotated key never exists in 16 bits.
//
// Work mapping.  A block serves one token; a group of LPV lanes serves one head
// vector at a time and walks the token's query heads, then its key and value
// heads, the next head's loads issued before this one's arithmetic.  Lane j of a
// group holds elements [8j, 8j + 8) and [D/2 + 8j, D/2 + 8j + 8), so both halves of
// a full-width rotation pair (i, i + D/2), and every adjacent pair (2i, 2i + 1),
// sit in one lane and the rotation exchanges nothing; its eight (cos, sin)
// pairs stay in registers for all heads of the token.  Narrower rotations
// exchange the pair through shared memory.
//
// Measured (B200): 16 x 512 tokens, 32 query and 8 KV heads of 128, f16, norms,
// adjacent pairs: 55 us for 185 MB (3.4 TB/s).  Bound by instruction issue (74 %
// of the slots): 16 elements a lane cost about 170 instructions as a query,
// twice that with the exact quantizer; seven blocks of 72 registers an SM are
// 6 to 15 % faster than five, six or eight for the 16-bit types, which spill up
// to 16 bytes a thread at that bound (float32 84 to 92, its raw elements taking
// twice the registers).  One launch replaces the norm, the rotation, the
// transpose and the append.

#include <cmath>
#include <type_traits>

#include "host_common.h"

namespace sdc {
namespace {

constexpr int kBlock = 128;

enum Pairing { kHalves = 0, kAdjacent = 1, kPartial = 2 };

struct RotateArgs {
    Pool pool;
    int64_t layer;
    const void* src[3];  // query, key, value
    int64_t s_batch[3], s_token[3], s_head[3];
    const int64_t* positions;
    int64_t position_stride;
    const float2* table;
    int64_t table_positions;
    int32_t rotary_dim;
    int32_t interleaved;
    const void* weight[2];  // query, key
    int32_t weight_dtype;
    float eps;
    float inv_dim;
    const int64_t* slots;
    void* out;
    FastDiv div_tokens;  // tokens per sequence
    FastDiv div_block;
    uint32_t query_heads, kv_heads, head_dim;
    int32_t* status;
};

// Eight consecutive elements as they are stored, and as floats.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&x)[16], int at) const {
        x[at] = a.x, x[at + 1] = a.y, x[at + 2] = a.z, x[at + 3] = a.w;
        x[at + 4] = b.x, x[at + 5] = b.y, x[at + 6] = b.z, x[at + 7] = b.w;
    }
};
template <typename T>
struct Raw8 {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void get(float (&x)[16], int at) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                x[at + 2 * j] = f.x, x[at + 2 * j + 1] = f.y;
            } else {  // the bits of a bf16 are the high half of a float's
                x[at + 2 * j] = __uint_as_float(w[j] << 16);
                x[at + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
};

__device__ __forceinline__ void store8(float* p, const float (&x)[16], int at) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[at], x[at + 1], x[at + 2], x[at + 3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[at + 4], x[at + 5], x[at + 6], x[at + 7]);
}
__device__ __forceinline__ uint32_t pair_bits(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_bits(__half, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[16], int at) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pair_bits(T(), x[at], x[at + 1]), pair_bits(T(), x[at + 2], x[at + 3]),
                   pair_bits(T(), x[at + 4], x[at + 5]), pair_bits(T(), x[at + 6], x[at + 7]));
}

// Sixteen weights of a lane (elements c0 .. c0 + 7 and c1 .. c1 + 7).
__device__ __forceinline__ void load_weights(const void* w, int dtype, uint32_t c0, uint32_t c1, float (&x)[16]) {
    if (dtype == SDC_DTYPE_F32) {
        Raw8<float> a, b;
        a.load(static_cast<const float*>(w) + c0), b.load(static_cast<const float*>(w) + c1);
        a.get(x, 0), b.get(x, 8);
    } else if (dtype == SDC_DTYPE_BF16) {
        Raw8<__nv_bfloat16> a, b;
        a.load(static_cast<const __nv_bfloat16*>(w) + c0), b.load(static_cast<const __nv_bfloat16*>(w) + c1);
        a.get(x, 0), b.get(x, 8);
    } else {
        Raw8<__half> a, b;
        a.load(static_cast<const __half*>(w) + c0), b.load(static_cast<const __half*>(w) + c1);
        a.get(x, 0), b.get(x, 8);
    }
}

// One head vector of a pass: where it is and what becomes of it.
template <typename T>
struct Head {
    const T* src;
    uint32_t index;  // among the query heads, or the pool's heads
    bool active;     // this lane holds elements of a head
    bool key;        // of the key and value passes
};

template <typename T, int LPV, int MODE>
__global__ void __launch_bounds__(kBlock, 7) norm_rotate_append_kernel(RotateArgs a) {
    constexpr uint32_t kGroups = kBlock / LPV;
    __shared__ __align__(16) float exchange[MODE == kPartial ? kGroups * LPV * 16 : 1];
    const uint32_t D = a.head_dim;
    const uint32_t sub = threadIdx.x % LPV, group = threadIdx.x / LPV;
    const uint32_t c0 = sub * 8, c1 = D / 2 + sub * 8;
    const bool live = c0 < D / 2;
    const uint32_t row = blockIdx.x;  // b * tokens + t
    uint32_t b, t;
    a.div_tokens.divmod(row, b, t);
    const uint32_t Hq = a.query_heads, Hk = a.kv_heads;
    const uint32_t query_passes = (Hq + kGroups - 1) / kGroups;
    const uint32_t passes = query_passes + (2 * Hk + kGroups - 1) / kGroups;

    const T* const base[3] = {static_cast<const T*>(a.src[0]) + b * a.s_batch[0] + t * a.s_token[0],
                              static_cast<const T*>(a.src[1]) + b * a.s_batch[1] + t * a.s_token[1],
                              static_cast<const T*>(a.src[2]) + b * a.s_batch[2] + t * a.s_token[2]};
    const auto locate = [&](uint32_t pass) {
        Head<T> h;
        if (pass < query_passes) {
            h.index = pass * kGroups + group;
            h.active = h.index < Hq && live;
            h.key = false;
            h.src = base[0] + h.index * a.s_head[0];
        } else {
            h.index = (pass - query_passes) * kGroups + group;
            h.active = h.index < 2 * Hk && live && pass < passes;
            h.key = h.index < Hk;
            if (!h.key) h.index -= Hk;
            h.src = h.key ? base[1] + h.index * a.s_head[1] : base[2] + h.index * a.s_head[2];
        }
        return h;
    };
    Raw8<T> lo, hi;
    Head<T> head = locate(blockIdx.y);
    if (head.active) lo.load(head.src + c0), hi.load(head.src + c1);

    const int64_t position = __ldg(a.positions + b * a.position_stride + t);
    const bool placed = position >= 0 && position < a.table_positions;
    if (!placed && blockIdx.y == 0 && threadIdx.x == 0) report_fault(a.status, SDC_FAULT_POSITION_RANGE);
    const int64_t slot = __ldg(a.slots + row);
    const bool slotted = slot >= 0 && slot < a.pool.num_blocks * a.pool.block_size;
    if (!slotted && blockIdx.y == 0 && threadIdx.x == 0) report_fault(a.status, SDC_FAULT_SLOT_RANGE);

    // this lane's eight cosines and sines; zero in lanes past the head, whose
    // elements take part in the group's maximum
    float2 cs[4] = {}, sn[4] = {};
    const float2* angles = a.table + (placed ? position : 0) * (a.rotary_dim / 2);
    if (MODE != kPartial && live) {
        // halves: pairs c0 + k; adjacent: pairs c0 / 2 + k and c1 / 2 + k
        const float4* p0 = reinterpret_cast<const float4*>(angles + (MODE == kHalves ? c0 : c0 / 2));
        const float4* p1 = reinterpret_cast<const float4*>(angles + (MODE == kHalves ? c0 + 4 : c1 / 2));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 u = __ldg(p0 + k), v = __ldg(p1 + k);
            cs[k] = make_float2(u.x, u.z), sn[k] = make_float2(u.y, u.w);
            cs[2 + k] = make_float2(v.x, v.z), sn[2 + k] = make_float2(v.y, v.w);
        }
    }
    uint32_t blk = 0, off = 0;
    if (slotted) a.div_block.divmod(static_cast<uint32_t>(slot), blk, off);

    // the same trip count on every lane: the group reductions shuffle whole warps
    for (uint32_t pass = blockIdx.y; pass < passes; pass += gridDim.y) {
        const bool is_query = pass < query_passes;
        float x[16];
        if (head.active) {
            lo.get(x, 0), hi.get(x, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.0f;
        }
        const Head<T> h = head;
        head = locate(pass + gridDim.y);
        if (head.active) lo.load(head.src + c0), hi.load(head.src + c1);

        const void* weight = a.weight[is_query ? 0 : 1];
        if (weight != nullptr) {
            float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float2 v = make_float2(x[i], x[i + 1]);
                sum2 = __ffma2_rn(v, v, sum2);
            }
            float sum = sum2.x + sum2.y;
#pragma unroll
            for (int o = LPV / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
            float inv = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
            if (__any_sync(kFullMask, !(sum < INFINITY))) {
                // elements above 2^60 whose squares pass float32: once more,
                // scaled by 2^-70 (eps is far below the sum's last bit then)
                float small = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) small = fmaf(x[i] * 0x1p-70f, x[i] * 0x1p-70f, small);
#pragma unroll
                for (int o = LPV / 2; o > 0; o >>= 1) small += __shfl_xor_sync(kFullMask, small, o);
                if (!(sum < INFINITY)) inv = rsqrtf(small * a.inv_dim) * 0x1p-70f;
            }
            if (h.active && (is_query || h.key)) {
                float w[16];
                load_weights(weight, a.weight_dtype, c0, c1, w);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float2 v = __fmul2_rn(__fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(inv, inv)),
                                                make_float2(w[i], w[i + 1]));
                    x[i] = v.x, x[i + 1] = v.y;
                }
            }
        }
        if (MODE == kHalves) {
            if (is_query || h.key) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = make_float2(x[2 * i], x[2 * i + 1]), q = make_float2(x[8 + 2 * i], x[9 + 2 * i]);
                    const float2 u = __ffma2_rn(p, cs[i], __fmul2_rn(make_float2(-q.x, -q.y), sn[i]));
                    const float2 v = __ffma2_rn(q, cs[i], __fmul2_rn(p, sn[i]));
                    x[2 * i] = u.x, x[2 * i + 1] = u.y;
                    x[8 + 2 * i] = v.x, x[9 + 2 * i] = v.y;
                }
            }
        } else if (MODE == kAdjacent) {
            if (is_query || h.key) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float c = i & 1 ? cs[i / 2].y : cs[i / 2].x, s = i & 1 ? sn[i / 2].y : sn[i / 2].x;
                    const float p = x[2 * i], q = x[2 * i + 1];
                    x[2 * i] = p * c - q * s;
                    x[2 * i + 1] = q * c + p * s;
                }
            }
        } else {
            float* mine = exchange + group * (LPV * 16);
            if (live) store8(mine + c0, x, 0), store8(mine + c1, x, 8);
            __syncwarp();
            if (h.active && (is_query || h.key)) {
                const uint32_t R = static_cast<uint32_t>(a.rotary_dim), H = R / 2;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t e = i < 8 ? c0 + i : c1 + i - 8;
                    if (e >= R) continue;
                    const bool first = a.interleaved ? (e & 1) == 0 : e < H;
                    const uint32_t partner = a.interleaved ? e ^ 1u : first ? e + H : e - H;
                    const float2 turn = __ldg(angles + (a.interleaved ? e / 2 : first ? e : e - H));
                    const float other = mine[partner];
                    x[i] = first ? x[i] * turn.x - other * turn.y : x[i] * turn.x + other * turn.y;
                }
            }
            __syncwarp();
        }

        if (is_query) {
            if (!h.active) continue;
            if (!placed) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0.0f;
            }
            T* out = static_cast<T*>(a.out) +
                     ((static_cast<int64_t>(b) * Hq + h.index) * a.div_tokens.divisor + t) * D;
            store8(out + c0, x, 0), store8(out + c1, x, 8);
            continue;
        }
        // the quantizer's maximum; all lanes take part in the shuffles
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max_nan(m, fabsf(x[i]));
#pragma unroll
        for (int o = LPV / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFullMask, m, o));
        if (!h.active || !slotted || !placed) continue;
        if (!(m < INFINITY)) {
            if (sub == 0) report_fault(a.status, SDC_FAULT_NONFINITE_VALUE);
            continue;
        }
        float s = 0.0f;
        uint4 codes = make_uint4(0u, 0u, 0u, 0u);
        if (m != 0.0f) {
            s = __fdiv_rn(m, 127.0f);
            if (!(s > 0.0f)) {
                if (sub == 0) report_fault(a.status, SDC_FAULT_INVALID_SCALE);
                continue;
            }
            if (s >= kFloatPathMinScale) {
                codes = quant16_f32(x, s, 1.0f / s);
            } else {
                int q[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) q[i] = quant_code_f64(static_cast<double>(x[i]), static_cast<double>(s));
                codes = make_uint4(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]),
                                   pack4(q[8], q[9], q[10], q[11]), pack4(q[12], q[13], q[14], q[15]));
            }
        }
        int8_t* dst = (h.key ? a.pool.keys : a.pool.values) + blk * a.pool.cbs + a.layer * a.pool.cls +
                      h.index * a.pool.chs + static_cast<int64_t>(off) * D;
        *reinterpret_cast<uint2*>(dst + c0) = make_uint2(codes.x, codes.y);
        *reinterpret_cast<uint2*>(dst + c1) = make_uint2(codes.z, codes.w);
        if (sub == 0) {
            (h.key ? a.pool.key_scales : a.pool.value_scales)[blk * a.pool.sbs + a.layer * a.pool.sls +
                                                              h.index * a.pool.shs + off] = s;
        }
    }
}

template <typename T, int LPV>
sdc_status_t launch_mode(int mode, dim3 grid, const RotateArgs& a, cudaStream_t st) {
    switch (mode) {
        case kHalves: norm_rotate_append_kernel<T, LPV, kHalves><<<grid, kBlock, 0, st>>>(a); break;
        case kAdjacent: norm_rotate_append_kernel<T, LPV, kAdjacent><<<grid, kBlock, 0, st>>>(a); break;
        default: norm_rotate_append_kernel<T, LPV, kPartial><<<grid, kBlock, 0, st>>>(a); break;
    }
    return launch_status();
}

template <typename T>
sdc_status_t launch_typed(int lpv, int mode, dim3 grid, const RotateArgs& a, cudaStream_t st) {
    switch (lpv) {
        case 1: return launch_mode<T, 1>(mode, grid, a, st);
        case 2: return launch_mode<T, 2>(mode, grid, a, st);
        case 4: return launch_mode<T, 4>(mode, grid, a, st);
        case 8: return launch_mode<T, 8>(mode, grid, a, st);
        case 16: return launch_mode<T, 16>(mode, grid, a, st);
        default: return launch_mode<T, 32>(mode, grid, a, st);
    }
}

sdc_status_t check_source(const void* p, const int64_t* strides, int es) {
    if (p == nullptr) return SDC_STATUS_NULL_ARGUMENT;
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < 0) return SDC_STATUS_INVALID_SIZE;
        if (strides[i] > (int64_t(1) << 40)) return SDC_STATUS_OVERFLOW;
        if ((strides[i] * es) % 16) return SDC_STATUS_MISALIGNED;
    }
    return aligned16(p) ? SDC_STATUS_OK : SDC_STATUS_MISALIGNED;
}

}  // namespace
}  // namespace sdc

using namespace sdc;

extern "C" {

SDC_API sdc_status_t sdc_norm_rotate_append(const sdc_page_pool_t* pool, int64_t layer,
                                            const sdc_rotate_batch_t* batch, const int64_t* slot_mapping,
                                            void* out_query, int32_t* device_status, uintptr_t stream) {
    try {
        sdc_status_t rc = validate_pool(pool);
        if (rc != SDC_STATUS_OK) return rc;
        if (batch == nullptr || slot_mapping == nullptr || out_query == nullptr || device_status == nullptr) {
            return SDC_STATUS_NULL_ARGUMENT;
        }
        const sdc_rotate_batch_t& q = *batch;
        if (q.positions == nullptr || q.table == nullptr) return SDC_STATUS_NULL_ARGUMENT;
        if (layer < 0 || layer >= pool->num_layers) return SDC_STATUS_INVALID_SIZE;
        if (q.batch < 0 || q.tokens < 0 || q.query_heads < 1 || q.table_positions < 1) return SDC_STATUS_INVALID_SIZE;
        if (q.dtype != SDC_DTYPE_F32 && q.dtype != SDC_DTYPE_BF16 && q.dtype != SDC_DTYPE_F16) {
            return SDC_STATUS_UNSUPPORTED;
        }
        const int es = dtype_size(q.dtype);
        const int64_t qs[3] = {q.query_batch_stride, q.query_token_stride, q.query_head_stride};
        const int64_t ks[3] = {q.key_batch_stride, q.key_token_stride, q.key_head_stride};
        const int64_t vs[3] = {q.value_batch_stride, q.value_token_stride, q.value_head_stride};
        rc = check_source(q.query, qs, es);
        if (rc == SDC_STATUS_OK) rc = check_source(q.key, ks, es);
        if (rc == SDC_STATUS_OK) rc = check_source(q.value, vs, es);
        if (rc != SDC_STATUS_OK) return rc;
        if (!aligned16(q.table) || !aligned16(out_query) || !aligned(q.positions) || !aligned(slot_mapping) ||
            !aligned(device_status)) {
            return SDC_STATUS_MISALIGNED;
        }
        const int64_t D = pool->head_dim;
        if (q.rotary_dim < 2 || q.rotary_dim > D || q.rotary_dim % 2) return SDC_STATUS_INVALID_ARGUMENT;
        if (q.position_stride < q.tokens && q.batch > 1) return SDC_STATUS_INVALID_SIZE;
        if (q.position_stride < 0 || q.position_stride > (int64_t(1) << 40)) return SDC_STATUS_INVALID_SIZE;
        if (q.query_weight != nullptr || q.key_weight != nullptr) {
            if (q.weight_dtype != SDC_DTYPE_F32 && q.weight_dtype != SDC_DTYPE_BF16 &&
                q.weight_dtype != SDC_DTYPE_F16) {
                return SDC_STATUS_UNSUPPORTED;
            }
            if (!aligned16(q.query_weight) || !aligned16(q.key_weight)) return SDC_STATUS_MISALIGNED;
            if (!(q.eps > 0.0f) || !std::isfinite(q.eps)) return SDC_STATUS_INVALID_ARGUMENT;
        }
        if (q.batch == 0 || q.tokens == 0) return SDC_STATUS_OK;
        if (q.batch > INT32_MAX / q.tokens || q.query_heads + 2 * pool->num_heads > INT32_MAX / 2 ||
            pool->num_blocks >= INT32_MAX / pool->block_size || q.table_positions > (int64_t(1) << 40) / D) {
            return SDC_STATUS_OVERFLOW;
        }
        RotateArgs a;
        a.pool = to_pool(pool);
        a.layer = layer;
        const void* src[3] = {q.query, q.key, q.value};
        const int64_t* strides[3] = {qs, ks, vs};
        for (int i = 0; i < 3; ++i) {
            a.src[i] = src[i];
            a.s_batch[i] = strides[i][0], a.s_token[i] = strides[i][1], a.s_head[i] = strides[i][2];
        }
        a.positions = q.positions;
        a.position_stride = q.position_stride;
        a.table = reinterpret_cast<const float2*>(q.table);
        a.table_positions = q.table_positions;
        a.rotary_dim = static_cast<int32_t>(q.rotary_dim);
        a.interleaved = q.interleaved != 0;
        a.weight[0] = q.query_weight, a.weight[1] = q.key_weight;
        a.weight_dtype = q.weight_dtype;
        a.eps = q.eps;
        a.inv_dim = 1.0f / static_cast<float>(D);
        a.slots = slot_mapping;
        a.out = out_query;
        a.div_tokens = FastDiv(static_cast<uint32_t>(q.tokens));
        a.div_block = FastDiv(static_cast<uint32_t>(pool->block_size));
        a.query_heads = static_cast<uint32_t>(q.query_heads);
        a.kv_heads = static_cast<uint32_t>(pool->num_heads);
        a.head_dim = static_cast<uint32_t>(D);
        a.status = device_status;
        const int lpv = lanes_per_vector(D);
        const int64_t rows = q.batch * q.tokens;
        const int64_t passes = ceil_div(q.query_heads, kBlock / lpv) + ceil_div(2 * pool->num_heads, kBlock / lpv);
        // few tokens: the passes over a token's heads run as blocks of their own
        int64_t splits = 1;
        while (splits < passes && rows * splits < int64_t(device_sms()) * 8) ++splits;
        if (splits > 65535) splits = 65535;
        const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(splits));
        const int mode = q.rotary_dim < D ? kPartial : q.interleaved ? kAdjacent : kHalves;
        cudaStream_t st = as_stream(stream);
        switch (q.dtype) {
            case SDC_DTYPE_F32: return launch_typed<float>(lpv, mode, grid, a, st);
            case SDC_DTYPE_BF16: return launch_typed<__nv_bfloat16>(lpv, mode, grid, a, st);
            default: return launch_typed<__half>(lpv, mode, grid, a, st);
        }
    } catch (...) {
        return SDC_STATUS_INTERNAL_ERROR;
    }
}

}  // extern "C"
