// Shared device helpers for libspecdecode_cuda (sm_100a).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "specdecode_cuda.h"

namespace sdc {

constexpr unsigned kFullMask = 0xffffffffu;

// Pool descriptor passed to kernels by value.
struct Pool {
    int8_t* keys;
    int8_t* values;
    float* key_scales;
    float* value_scales;
    int64_t num_blocks, block_size, num_layers, num_heads, head_dim;
    int64_t cbs, cls, chs;  // code block / layer / head strides (elements)
    int64_t sbs, sls, shs;  // scale block / layer / head strides (elements)
};

struct TableEdits {
    int32_t* block_tables;
    int64_t table_stride;
    int64_t table_rows;
    int32_t* context_lens;
    const int32_t* entries;
    int64_t num_entries;
    const int32_t* lengths;
    int64_t num_lengths;
};

__device__ __forceinline__ void report_fault(int32_t* status, int32_t bits) {
    if (status != nullptr) atomicOr(status, bits);
}

// Unsigned 32-bit division by a run-time constant (Granlund-Montgomery):
// q = (t + ((n - t) >> 1)) >> (shift - 1) with t = umulhi(n, mul).  Exact
// for every 32-bit n and divisor >= 1.
struct FastDiv {
    uint32_t divisor;
    uint32_t mul;
    uint32_t shift;

    FastDiv() = default;
    __host__ explicit FastDiv(uint32_t d) : divisor(d) {
        uint32_t l = 0;
        while ((uint64_t(1) << l) < d) ++l;
        shift = l;
        mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        if (shift == 0) return n;  // divisor 1
        const uint32_t t = __umulhi(n, mul);
        return (t + ((n - t) >> 1)) >> (shift - 1);
    }
    __device__ __forceinline__ void divmod(uint32_t n, uint32_t& q, uint32_t& r) const {
        q = div(n);
        r = n - q * divisor;
    }
};

// Loads 16 consecutive source elements (16-byte aligned) as Acc values.
__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
    const float4* q = reinterpret_cast<const float4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 v = __ldg(q + i);
        x[4 * i + 0] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
}

__device__ __forceinline__ void load16(const __nv_bfloat16* p, float (&x)[16]) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint4 v = __ldg(q + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // bf16 -> f32 is exact: the bf16 bits are the high half of the f32 bits.
            x[8 * i + 2 * j + 0] = __uint_as_float(w[j] << 16);
            x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void load16(const __half* p, float (&x)[16]) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint4 v = __ldg(q + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __half2 h = *reinterpret_cast<const __half2*>(&w[j]);
            float2 f = __half22float2(h);
            x[8 * i + 2 * j + 0] = f.x;
            x[8 * i + 2 * j + 1] = f.y;
        }
    }
}

__device__ __forceinline__ void load16(const double* p, double (&x)[16]) {
    const double2* q = reinterpret_cast<const double2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        double2 v = __ldg(q + i);
        x[2 * i + 0] = v.x; x[2 * i + 1] = v.y;
    }
}

// ---------------------------------------------------------------------------
// The reference's quantization rule (native/src/native.cpp:289-315):
//   scale = (double)(float)(max|x| / 127.0)
//   q     = clamp(round_half_away_from_zero(x / scale), -127, 127)
// with the division and rounding done in double.
// ---------------------------------------------------------------------------

// Scale from the vector maximum: a double division rounded once to float.
__device__ __forceinline__ float scale_from_max(double maximum) {
    return __double2float_rn(maximum / 127.0);
}

// Double path: the reference arithmetic verbatim.  CUDA's round() rounds
// halfway cases away from zero, like std::round.
__device__ __forceinline__ int quant_code_f64(double x, double scale) {
    double r = round(x / scale);
    r = fmin(fmax(r, -127.0), 127.0);
    return static_cast<int>(r);
}

// Float path for inputs that are float32 values (f32 / bf16 / f16 sources).
// Returns round_half_away(x / s) of the *exact* quotient using only float
// arithmetic.  A candidate n0 = rint(|x| * rcp) is within one of the answer
// (rcp = 1/s rounded once, so |x|*rcp is within 2^-22 relative of |x|/s).  It
// is corrected by the signs of |x| - (n0 + 1/2) s and |x| - (n0 - 1/2) s,
// each computed with one fused multiply-add: a correctly rounded result has
// the sign of the exact residual, and the residual cannot round to zero
// because it is zero or a multiple of at least 2^-149 (true whenever
// s >= 2^-100; smaller scales take the double path).  For a quotient of two
// float32 values the double-rounded quotient the reference rounds lands on
// the same integer as the exact one, because such a quotient is never within
// 2^-26 of a half-integer without being one.
__device__ __forceinline__ float quant_mag_f32(float a, float s, float rcp) {
    float n = rintf(a * rcp);
    n += (__fmaf_rn(-(n + 0.5f), s, a) >= 0.0f) ? 1.0f : 0.0f;
    n -= (__fmaf_rn(-(n - 0.5f), s, a) < 0.0f) ? 1.0f : 0.0f;
    return fminf(n, 127.0f);
}

__device__ __forceinline__ int quant_code_f32(float x, float s, float rcp) {
    const int q = static_cast<int>(quant_mag_f32(fabsf(x), s, rcp));
    return x < 0.0f ? -q : q;
}

constexpr float kFloatPathMinScale = 0x1p-100f;

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (static_cast<uint32_t>(a) & 0xffu) | ((static_cast<uint32_t>(b) & 0xffu) << 8) |
           ((static_cast<uint32_t>(c) & 0xffu) << 16) | ((static_cast<uint32_t>(d) & 0xffu) << 24);
}

// Sixteen codes of a float-valued vector with scale s >= 2^-100 (rcp = 1/s
// rounded), packed four to a word: round_half_away(x / s) clamped to 127 in
// magnitude, the same integers as quant_code_f32 but with no conversion
// instruction.  The candidate rint(|x| * rcp) comes from adding and removing
// 1.5 * 2^23 (round to nearest even of a value below 2^22, exactly what rintf
// returns); it is within one of the answer and is corrected by the exact
// signs of |x| - (n +- 1/2) s, each from one fused multiply-add.  The signed
// code plus 1.5 * 2^23 holds the code's two's-complement byte in its low
// mantissa bits, which byte permutes pack.  Pairs of elements go through the
// packed f32x2 arithmetic.
__device__ __forceinline__ uint4 quant16_f32(const float (&x)[16], float s, float rcp) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
    const float2 rcp2 = make_float2(rcp, rcp), negs2 = make_float2(-s, -s);
    const float2 m2 = make_float2(kMagic, kMagic), negm2 = make_float2(-kMagic, -kMagic);
    const float2 half2 = make_float2(0.5f, 0.5f), neghalf2 = make_float2(-0.5f, -0.5f);
    uint32_t bits[16];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float2 a = make_float2(fabsf(x[i]), fabsf(x[i + 1]));
        float2 n = __fadd2_rn(__fadd2_rn(__fmul2_rn(a, rcp2), m2), negm2);
        const float2 above = __ffma2_rn(__fadd2_rn(n, half2), negs2, a);     // a - (n + 1/2) s
        const float2 below = __ffma2_rn(__fadd2_rn(n, neghalf2), negs2, a);  // a - (n - 1/2) s
        n.x += (above.x >= 0.0f ? 1.0f : 0.0f) - (below.x < 0.0f ? 1.0f : 0.0f);
        n.y += (above.y >= 0.0f ? 1.0f : 0.0f) - (below.y < 0.0f ? 1.0f : 0.0f);
        // |x| <= m and s = fl(m / 127) give |x| / s < 127.5, so n <= 127 needs no clamp
        const float2 q = make_float2(copysignf(n.x, x[i]), copysignf(n.y, x[i + 1]));
        const float2 t = __fadd2_rn(q, m2);
        bits[i] = __float_as_uint(t.x);
        bits[i + 1] = __float_as_uint(t.y);
    }
    auto pack = [](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
        return __byte_perm(__byte_perm(w0, w1, 0x0040), __byte_perm(w2, w3, 0x0040), 0x5410);
    };
    return make_uint4(pack(bits[0], bits[1], bits[2], bits[3]), pack(bits[4], bits[5], bits[6], bits[7]),
                      pack(bits[8], bits[9], bits[10], bits[11]), pack(bits[12], bits[13], bits[14], bits[15]));
}

// max that propagates NaN, so one reduction finds both the vector maximum and
// any non-finite element (the result is then NaN or +inf).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void apply_table_edits(const TableEdits& e, int64_t index, int64_t stride,
                                                  int32_t* status) {
    for (int64_t i = index; i < e.num_entries; i += stride) {
        const int32_t row = e.entries[3 * i + 0];
        const int32_t col = e.entries[3 * i + 1];
        const int32_t val = e.entries[3 * i + 2];
        if (row < 0 || row >= e.table_rows || col < 0 || col >= e.table_stride) {
            report_fault(status, SDC_FAULT_TABLE_RANGE);
            continue;
        }
        e.block_tables[static_cast<int64_t>(row) * e.table_stride + col] = val;
    }
    for (int64_t i = index; i < e.num_lengths; i += stride) {
        const int32_t row = e.lengths[2 * i + 0];
        const int32_t len = e.lengths[2 * i + 1];
        if (row < 0 || row >= e.table_rows || len < 0) {
            report_fault(status, SDC_FAULT_TABLE_RANGE);
            continue;
        }
        e.context_lens[row] = len;
    }
}

}  // namespace sdc
