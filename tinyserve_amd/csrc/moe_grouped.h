// What the grouped MoE layers share: the activation, the work of a workgroup, the weighted sums.
#pragma once

#include "fp8_common.h"
#include "moe_group.h"

namespace tsa {
namespace {

__device__ __forceinline__ float moe_act(const tsa_expert_layout& L, float gate, float up) {
    if (L.act == TSA_ACT_SWIGLU_OAI) {
        // the limits by comparisons: a minimum or maximum would give its other operand for a NaN
        const float lim = L.swiglu_limit, g = gate > lim ? lim : gate, u = up > lim ? lim : up < -lim ? -lim : up;
        const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * (L.swiglu_alpha * g));
        return (u + 1.0f) * g * __builtin_amdgcn_rcpf(1.0f + e);
    }
    return silu_mul_fast(gate, up);
}

// The workgroup's (entry, tile) of n_entries x tiles: each XCD takes a run of the entries with all
// their tiles (an expert's entries and an entry's tiles share an L2). False: none is left for it.
__device__ __forceinline__ bool grouped_work(const int* n_entries, int tiles, int& entry, int& tile) {
    const int total = uniform(*n_entries) * tiles, lin = (int)blockIdx.x, xcd = lin & 7, q8 = total >> 3, rem = total & 7;
    if ((lin >> 3) >= q8 + (xcd < rem ? 1 : 0)) return false;
    const int wid = xcd * q8 + (xcd < rem ? xcd : rem) + (lin >> 3);
    entry = wid / tiles;
    tile = wid % tiles;
    return true;
}

// The weighted sums over each token's experts: the assignments' outputs yk [T k, H] in float32.
struct MoeCombine {
    const int32_t* idx;
    const float* wts;
    const int32_t* expert_slot;
    int64_t E, n_slots;
    int T, k, H;
    const float* yk;
    void* y;
    int y_dtype;
};

// y[t] = sum_j w[t, j] yk[t k + j], in order of j; a thread 8 values of a row.
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeCombine p) {
    const int H = p.H, per = H / 8;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)p.T * per) return;
    const int t = (int)(at / per), c = (int)(at % per);
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int AHEAD = 4;  // outputs on their way together
    for (int j0 = 0; j0 < p.k; j0 += AHEAD) {
        int sl[AHEAD];
        float w[AHEAD], v[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t a = (int64_t)t * p.k + (j0 + u < p.k ? j0 + u : j0);
            const int e = p.idx[a];
            w[u] = p.wts[a];
            sl[u] = j0 + u < p.k && e >= 0 && e < p.E ? p.expert_slot[e] : -1;
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {  // not resident: nothing was written there, and any row is read
            const bool live = sl[u] >= 0 && sl[u] < p.n_slots;
            f8_load8<TSA_F32>(p.yk + (live ? (int64_t)t * p.k + j0 + u : 0) * H, c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r] = sl[u] >= 0 && sl[u] < p.n_slots ? fmaf(w[u], v[u][r], s[r]) : s[r];
    }
    const int64_t o = (int64_t)t * H + 8 * c;
    if (p.y_dtype == TSA_BF16 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + o) =
            make_uint4(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]), pack_bf16x2(s[6], s[7]));
        return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) store_out(p.y, p.y_dtype, o + r, s[r]);
}

inline int launch_combine(const MoeCombine& p, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)p.T * (p.H / 8) + 255) / 256));
    hipLaunchKernelGGL(moe_combine_kernel, grid, dim3(256), 0, st, p);
    TSA_LAUNCH_CHECK();
    return TSA_OK;
}

inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

constexpr int64_t MOE_ASSIGNMENTS = 131072;  // at a time: bounds the workspace (1.1 GiB of outputs at hidden 2048)

// Tokens at a time for at most `most` assignments.
inline int64_t group_tokens(int64_t T, int k, int64_t most) {
    const int64_t c = most / k > 0 ? most / k : 1;
    return T < c ? T : c;
}

}  // namespace
}  // namespace tsa
