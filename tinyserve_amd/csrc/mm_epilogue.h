// From a tile's sums to rows of y: scales (int8), bias, one rounding.
//
// Results of 16 bits go through LDS, 16 tokens at a time, so that a wave writes whole lines (lane by lane they are 8
// bytes of 16 rows: 14 us for a 4096 x 4096 result, this way 9, its bytes at the copy rate 6.5). A row of 16 MR values
// is 2 MR pieces of 16 bytes; piece c of row r sits at c ^ (r 2 MR / 16), which spreads the rows over the banks.
#pragma once

#include "fused_common.h"
#include "mm_tile.h"

namespace tsa {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(int v) { return (float)v; }

struct MmOut {
    void* y;
    int y_dtype;
    int64_t ldy;
    const void* bias;
    int bias_dtype;
    int y_vec;  // y's rows start on multiples of 16 bytes and have whole pieces of them
};

inline MmOut mm_out(void* y, int y_dtype, int64_t N, const void* bias, int bias_dtype) {
    MmOut o{};
    o.y = y;
    o.y_dtype = y_dtype;
    o.ldy = N;
    o.bias = bias;
    o.bias_dtype = bias_dtype;
    o.y_vec = N % (y_dtype == TSA_F32 ? 4 : 8) == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
    return o;
}

template <int DT>
__device__ __forceinline__ uint2 mm_pack4(const v4f& v) {
    if constexpr (DT == TSA_BF16) return make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    return make_uint2((uint32_t)f32_to_f16_bits(v[0]) | (uint32_t)f32_to_f16_bits(v[1]) << 16,
                      (uint32_t)f32_to_f16_bits(v[2]) | (uint32_t)f32_to_f16_bits(v[3]) << 16);
}

// 16 tokens' rows of 16 M values, lane 16 q + i holding values 16 m + 4 q .. of token i in v[m]: to(r, c) is where piece c
// of token r goes, or null.
template <int M, class To>
__device__ __forceinline__ void mm_rows16(const uint2 (&v)[M], uint8_t* out, To to) {
    constexpr int P = 2 * M;  // pieces of a row
    const int lane = threadIdx.x & 63, q = lane >> 4, i = lane & 15;
#pragma unroll
    for (int m = 0; m < M; ++m)
        *reinterpret_cast<uint2*>(out + 16 * (i * P + ((2 * m + (q >> 1)) ^ (i * P / 16))) + 8 * (q & 1)) = v[m];
    asm volatile("" ::: "memory");  // LDS runs one wave's instructions in order
#pragma unroll
    for (int h = 0; h < (P + 3) / 4; ++h) {
        const int p = lane + 64 * h, r = p / P, c = p % P;
        if (P < 4 && r >= 16) continue;
        const u32x4 d = *reinterpret_cast<const u32x4*>(out + 16 * (r * P + (c ^ (r * P / 16))));
        void* dst = to(r, c);
        if (dst) *static_cast<u32x4*>(dst) = d;
    }
    asm volatile("" ::: "memory");
}

// Four floats from a table's entry n on, those below N (0 past it).
__device__ __forceinline__ v4f mm_load4(const float* p, int n, int N) {
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n + 3 < N && (reinterpret_cast<uintptr_t>(p + n) & 15) == 0) return *reinterpret_cast<const v4f*>(p + n);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (n + r < N) v[r] = p[n + r];
    return v;
}

// The same from a bias of any type.
__device__ __forceinline__ v4f mm_bias4(const void* p, int dtype, int n, int N) {
    if (dtype == TSA_F32) return mm_load4(static_cast<const float*>(p), n, N);
    const uint16_t* h = static_cast<const uint16_t*>(p) + n;
    uint2 w = make_uint2(0u, 0u);
    if (n + 3 < N && (reinterpret_cast<uintptr_t>(h) & 7) == 0) {
        w = *reinterpret_cast<const uint2*>(h);
    } else {
        if (n < N) w.x = h[0];
        if (n + 1 < N) w.x |= (uint32_t)h[1] << 16;
        if (n + 2 < N) w.y = h[2];
        if (n + 3 < N) w.y |= (uint32_t)h[3] << 16;
    }
    if (dtype == TSA_BF16)
        return v4f{bf16_bits_to_f32(w.x & 0xFFFFu), bf16_bits_to_f32(w.x >> 16), bf16_bits_to_f32(w.y & 0xFFFFu), bf16_bits_to_f32(w.y >> 16)};
    return v4f{f16_bits_to_f32(w.x & 0xFFFFu), f16_bits_to_f32(w.x >> 16), f16_bits_to_f32(w.y & 0xFFFFu), f16_bits_to_f32(w.y >> 16)};
}

// The tile's rows n0 .. (below N) of its first tn tokens; row(r): y's row of token r. int8 sums are scaled by
// xs(r) and ws[n].
template <class C, class A, class Row, class Scale>
__device__ __forceinline__ void mm_store(const A (&acc)[C::MR][C::MT], const MmOut& o, uint8_t* out, int n0, int N, int tn, Row row,
                                         Scale xs, const float* ws) {
    constexpr bool INT = std::is_same<A, v4i>::value;
    constexpr int MR = C::MR, MT = C::MT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, t0 = wave / C::WR * MT * 16, nw = n0 + wr * MR * 16;
    float sx[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        sx[t] = 1.0f;
        if constexpr (INT) sx[t] = t0 + 16 * t + i < tn ? xs(t0 + 16 * t + i) : 0.0f;
    }
    v4f sw[MR], b[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        const int n = nw + 16 * m + 4 * q;
        if constexpr (INT) sw[m] = mm_load4(ws, n, N);
        b[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (o.bias) b[m] = mm_bias4(o.bias, o.bias_dtype, n, N);
    }
    auto value = [&](int m, int t) {
        v4f v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (INT ? to_f32(acc[m][t][r]) * (sx[t] * sw[m][r]) : to_f32(acc[m][t][r])) + b[m][r];
        return v;
    };
    const bool full = o.y_vec && n0 + C::RN <= N && tn == C::TM;
    if (o.y_dtype == TSA_F32) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int tk = t0 + 16 * t + i;
            float* y = static_cast<float*>(o.y) + (full || tk < tn ? row(tk) : 0) * o.ldy;
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const int n = nw + 16 * m + 4 * q;
                const v4f v = value(m, t);
                if (full) {
                    *reinterpret_cast<v4f*>(y + n) = v;
                } else if (tk < tn) {
                    if (o.y_vec && n < N) *reinterpret_cast<v4f*>(y + n) = v;  // N % 4 == 0
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n + r < N) y[n + r] = v[r];
                }
            }
        }
        return;
    }
    auto rows16 = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (!o.y_vec) {
                const int tk = t0 + 16 * t + i;
                if (tk >= tn) continue;
                uint16_t* y = static_cast<uint16_t*>(o.y) + row(tk) * o.ldy;
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    const int n = nw + 16 * m + 4 * q;
                    const uint2 v = mm_pack4<DT>(value(m, t));
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < N) y[n + r] = (uint16_t)((r < 2 ? v.x : v.y) >> (16 * (r & 1)));
                }
                continue;
            }
            if (t0 + 16 * t >= tn) continue;  // uniform
            uint2 v[MR];
#pragma unroll
            for (int m = 0; m < MR; ++m) v[m] = mm_pack4<DT>(value(m, t));
            auto to = [&](int r, int c) -> void* {
                const int tk = t0 + 16 * t + r, n = nw + 8 * c;
                if (!full && (tk >= tn || n >= N)) return nullptr;  // N % 8 == 0
                return static_cast<uint16_t*>(o.y) + row(tk) * o.ldy + n;
            };
            mm_rows16<MR>(v, out, to);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (o.y_dtype == TSA_BF16) rows16(std::integral_constant<int, TSA_BF16>{});
    else rows16(std::integral_constant<int, TSA_F16>{});
}

}  // namespace
}  // namespace tsa
