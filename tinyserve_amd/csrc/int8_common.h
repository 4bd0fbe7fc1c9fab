// int8 quantisation of activations, a float32 scale for each token:
//     s = max(max|x_k| / 127, 2^-126),  c_k = round(x_k / s), ties to even,
// both quotients rounded to float32 first. Ties in the second rounding are common (16-bit values over
// 16-bit maxima), so the quotient has to be the correctly rounded one. A token that holds an infinity or a
// NaN has a NaN as its scale and zeros as its codes: whatever is made of it is NaN.
#pragma once

#include "fp8_common.h"
#include "mm_tile.h"

namespace tsa {
namespace {

// 8 values as they lie in memory.
template <int XT>
struct I8Raw {
    u32x4 w[XT == TSA_F32 ? 2 : 1];
};

// Chunk c (8 values) of a row of K values; past the row zeros. VEC: 16-byte aligned rows of whole chunks.
template <int XT, bool VEC>
__device__ __forceinline__ I8Raw<XT> i8_load(const uint8_t* row, int64_t K, int c) {
    I8Raw<XT> v = {};
    const int64_t k = (int64_t)8 * c;
    if constexpr (VEC) {
        if (k < K) {
            const u32x4* p = reinterpret_cast<const u32x4*>(row);
            if constexpr (XT == TSA_F32) v.w[0] = p[2 * c], v.w[1] = p[2 * c + 1];
            else v.w[0] = p[c];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) {
                if constexpr (XT == TSA_F32) v.w[e >> 2][e & 3] = reinterpret_cast<const uint32_t*>(row)[k + e];
                else v.w[0][e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[k + e] << (16 * (e & 1));
            }
    }
    return v;
}

// The largest magnitude, as bits of the type (their integer order is the order of the values, an infinity above all
// numbers, a NaN above it).
template <int XT>
__device__ __forceinline__ uint32_t i8_max(const I8Raw<XT>& v, uint32_t m) {
    if constexpr (XT == TSA_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, v.w[e >> 2][e & 3] & 0x7FFFFFFFu);
    } else {
#pragma unroll
        for (int d = 0; d < 4; ++d) m = max(m, max(v.w[0][d] & 0x7FFFu, v.w[0][d] >> 16 & 0x7FFFu));
    }
    return m;
}

// Such bits as a float32's.
template <int XT>
__device__ __forceinline__ uint32_t i8_max_f32(uint32_t m) {
    return XT == TSA_F32 ? m : XT == TSA_BF16 ? m << 16 : __float_as_uint(f16_bits_to_f32(m));
}

__device__ __forceinline__ float i8_scale(uint32_t max_bits) {
    if (max_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const float s = __uint_as_float(max_bits) / 127.0f;
    return s < 0x1p-126f ? 0x1p-126f : s;
}

// The codes of 8 values of a token with scale s. The quotient by Markstein's correction, as the FP8 codes have
// it (f8_codes8), which divides where bits of the remainder could underflow; fp32 inputs divide. |q| <=
// 127 (1 + 2^-23), so adding 1.5 2^23 rounds it to an integer, ties to even, in the sum's low bits.
template <int XT>
__device__ __forceinline__ uint2 i8_codes8(const I8Raw<XT>& raw, float s) {
    if (!(s == s)) return make_uint2(0u, 0u);
    float v[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (XT == TSA_F32) v[e] = __uint_as_float(raw.w[e >> 2][e & 3]);
        else v[e] = XT == TSA_BF16 ? __uint_as_float(e & 1 ? raw.w[0][e >> 1] & 0xFFFF0000u : raw.w[0][e >> 1] << 16)
                                   : f16_bits_to_f32(raw.w[0][e >> 1] >> (16 * (e & 1)));
    }
    if (XT == TSA_F32 || !(s > F8_MIN_CORRECTED)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = v[e] / s;
    } else {
        const float r = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = v[e] * r;
            q[e] = fmaf(fmaf(-a, s, v[e]), r, a);
        }
    }
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(q[e] + 12582912.0f);
    auto pack = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {  // the low bytes
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0c0c0400u), __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u), 0x05040100u);
    };
    return make_uint2(pack(b[0], b[1], b[2], b[3]), pack(b[4], b[5], b[6], b[7]));
}

// One row quantised by the W waves that call these together (tid: the thread's number among their 64 W). A thread
// holds its first D chunks from i8_row_load on; a longer row's others are read twice. `top`: W words of LDS
// that no one else uses (the barrier is the workgroup's: every wave of it calls).
template <int XT, bool VEC, int W, int D>
__device__ __forceinline__ void i8_row_load(const uint8_t* row, int64_t K, int tid, I8Raw<XT> (&v)[D]) {
#pragma unroll
    for (int d = 0; d < D; ++d) v[d] = i8_load<XT, VEC>(row, K, tid + 64 * W * d);
}

template <int XT, bool VEC>
__device__ __forceinline__ void i8_put(const I8Raw<XT>& v, float s, uint8_t* codes, int64_t K, int c) {
    const uint2 o = i8_codes8<XT>(v, s);
    uint8_t* dst = codes + (int64_t)8 * c;
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(dst) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if ((int64_t)8 * c + e < K) dst[e] = (uint8_t)((e < 4 ? o.x : o.y) >> (8 * (e & 3)));
    }
}

template <int XT, bool VEC, int W, int D>
__device__ __forceinline__ float i8_row_codes(const uint8_t* row, int64_t K, int tid, const I8Raw<XT> (&v)[D], uint8_t* codes, uint32_t* top) {
    const int chunks = (int)((K + 7) / 8);
    uint32_t m = 0;
#pragma unroll
    for (int d = 0; d < D; ++d) m = i8_max<XT>(v[d], m);
    for (int c = tid + 64 * W * D; c < chunks; c += 64 * W) m = i8_max<XT>(i8_load<XT, VEC>(row, K, c), m);
    m = wave_max_u32(m);
    if constexpr (W > 1) {
        if ((tid & 63) == 0) top[tid >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) m = max(m, top[w]);
    }
    const float s = i8_scale(i8_max_f32<XT>(m));
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (tid + 64 * W * d < chunks) i8_put<XT, VEC>(v[d], s, codes, K, tid + 64 * W * d);
    for (int c = tid + 64 * W * D; c < chunks; c += 64 * W) i8_put<XT, VEC>(i8_load<XT, VEC>(row, K, c), s, codes, K, c);
    return s;
}

constexpr int64_t I8_MAX_K = 131056;  // K 2^14 < 2^31: the sums fit 32 bits whatever the codes

}  // namespace
}  // namespace tsa
