// From a tile's sums to rows of y: scales (int8), bias, one rounding.
#pragma once

#include "fused_common.h"
#include "mm_tile.h"

namespace tsa {
namespace {

struct MmOut {
    void* y;
    int y_dtype;
    int64_t ldy;
    const void* bias;
    int bias_dtype;
    int y_vec;  // y's rows start on multiples of 16 bytes
};

inline MmOut mm_out(void* y, int y_dtype, int64_t N, const void* bias, int bias_dtype) {
    MmOut o{};
    o.y = y;
    o.y_dtype = y_dtype;
    o.ldy = N;
    o.bias = bias;
    o.bias_dtype = bias_dtype;
    o.y_vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
    return o;
}

// Values n .. n + 3 of a row of y, those below N.
__device__ __forceinline__ void mm_store4(const MmOut& o, int64_t row, int n, int N, const v4f& v) {
    const int64_t at = row * o.ldy + n;
    if (o.y_vec && o.y_dtype == TSA_BF16) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(o.y) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else if (o.y_vec && o.y_dtype == TSA_F32) {
        *reinterpret_cast<v4f*>(static_cast<float*>(o.y) + at) = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < N) store_out(o.y, o.y_dtype, at + r, v[r]);
    }
}

// The tile's rows n0 .. (below N) of its first tn tokens; row(r): y's row of token r. int8 sums are scaled by
// xs(r) and ws[n].
template <class C, class A, class Row, class Scale>
__device__ __forceinline__ void mm_store(const A (&acc)[C::MR][C::MT], const MmOut& o, int n0, int N, int tn, Row row, Scale xs,
                                         const float* ws) {
    constexpr bool INT = std::is_same<A, v4i>::value;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    float sx[C::MT];
    int64_t at[C::MT];
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
        const int tk = 16 * (C::MT * wt + t) + i;
        at[t] = tk < tn ? row(tk) : -1;
        sx[t] = 1.0f;
        if constexpr (INT) sx[t] = tk < tn ? xs(tk) : 0.0f;
    }
#pragma unroll
    for (int m = 0; m < C::MR; ++m) {
        const int n = n0 + (wr * C::MR + m) * 16 + 4 * q;
        float b[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sw[4] = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < N) {
                if (o.bias) b[r] = load_act(o.bias, o.bias_dtype, n + r);
                if constexpr (INT) sw[r] = ws[n + r];
            }
#pragma unroll
        for (int t = 0; t < C::MT; ++t) {
            if (at[t] < 0 || n >= N) continue;
            v4f v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (INT ? (float)acc[m][t][r] * (sx[t] * sw[r]) : (float)acc[m][t][r]) + b[r];
            mm_store4(o, at[t], n, N, v);
        }
    }
}

}  // namespace
}  // namespace tsa
