// MoE layers over FP8 experts (e4m3 codes with a float32 scale per 128 x 128 block).
//
// Definition, per token: x quantised per 128 values (fp8_common.h); for each selected expert
// h = act(Wg x, Wu x) in float32, quantised the same way; y = sum_j w_j Wd h, rounded once.
//
// Few tokens: two launches ordered by the stream. gate_up: one workgroup per (token, expert) pair
// and 16 channels; down: one per token and 16 outputs, over all the token's experts, so every
// output has one writer. Each is a stream of weights into the A operands of
// v_mfma_f32_16x16x128_f8f6f4 (one column of B in use: the matrix cores are idle otherwise, and the
// codes need no conversion).
#include "fp8_common.h"

namespace tsa {
namespace {

struct F8Moe {
    tsa_expert_layout L;
    const uint8_t* pool;
    int64_t n_slots;
    const int32_t* slots;
    const float* wts;
    const void* logits;
    int logits_dtype, route_mode;
    const int32_t* expert_slot;
    int E, k;
    int32_t* idx_out;
    float* w_out;
    int32_t* tab_slot;
    float* tab_w;
    const void* x;
    float* h;  // [T k, I]
    void* y;
    int y_dtype;
    int chunk;  // down: experts staged in LDS at a time
};

constexpr int F8A_NW = 4, F8A_D = 4;  // gate_up: waves, K blocks in flight per wave
constexpr int F8D_NW = 8, F8D_D = 6;  // down

__device__ __forceinline__ float f8_act(const tsa_expert_layout& L, float gate, float up) {
    if (L.act == TSA_ACT_SWIGLU_OAI) return swiglu_oai_fast(L, gate, up);
    return silu_mul_fast(gate, up);
}

template <int XT>
__global__ void __launch_bounds__(64 * F8A_NW) fp8_gate_up_kernel(F8Moe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, G = (int)f8_blocks(H);
    const int a = blockIdx.y, t = a / k, jj = a % k, n0 = (int)blockIdx.x * 16;
    uint8_t* xc = smem;
    float* xs = reinterpret_cast<float*>(smem + G * F8B);
    float* red = xs + G;  // [wave][gate / up][row]

    int64_t slot = -1;
    if (p.logits) {
        // every wave selects the pair's expert (round jj of the top-k); wave 0 of the token's first
        // workgroup makes all the selections and writes the table that the down launch reads
        float lg[4];
        int es[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) es[j] = p.expert_slot[min(lane + 64 * j, p.E - 1)];
        load4(p.logits, p.logits_dtype, (int64_t)t * p.E, p.E, lane, lg);
        if (blockIdx.x == 0 && jj == 0 && wave == 0) {
            __shared__ int s_slot[FUSED_MAXK];
            __shared__ float s_w[FUSED_MAXK];
            const int sel = route_token_v(p, 0, lane, lg, es, s_slot, s_w);
            if (lane < k) {
                if (p.idx_out) p.idx_out[t * k + lane] = sel;
                if (p.w_out) p.w_out[t * k + lane] = s_w[lane];
                p.tab_slot[t * k + lane] = s_slot[lane];  // written by this lane
                p.tab_w[t * k + lane] = s_w[lane];
            }
            slot = uniform(s_slot[0]);  // lane 0's own write
        } else {
            uint32_t myk;
            int mysel, myslot;
            select_topk(p, lane, lg, es, jj + 1, myk, mysel, myslot);
            slot = __builtin_amdgcn_readlane(myslot, jj);
        }
    } else {
        slot = uniform(p.slots[a]);
    }
    if (slot < 0 || slot >= p.n_slots) return;  // every wave of the workgroup: the pair's h is never read

    const uint8_t* base = p.pool + slot * L.slot_bytes;
    const int64_t records = (int64_t)(I - n0 < 16 ? I - n0 : 16) * H;
    const __amdgpu_buffer_rsrc_t rg = f8_buf(base + L.gate_off + (int64_t)n0 * H, records);
    const __amdgpu_buffer_rsrc_t ru = f8_buf(base + L.up_off + (int64_t)n0 * H, records);
    const float* sg = reinterpret_cast<const float*>(base + L.gate_scales_off) + n0 / F8B * G;
    const float* su = sg + f8_blocks(I) * G;
    u32x4 A[F8A_D][2][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < F8A_D; ++d) {
            const uint32_t o = (uint32_t)(F8B * (wave + F8A_NW * (j0 + d)) + 16 * q);
            const uint32_t o0 = f8_off((uint32_t)(i * H), o, (uint32_t)H), o1 = f8_off((uint32_t)(i * H), o + 64, (uint32_t)H);
            A[d][0][0] = f8_ld(rg, o0);
            A[d][0][1] = f8_ld(rg, o1);
            A[d][1][0] = f8_ld(ru, o0);
            A[d][1][1] = f8_ld(ru, o1);
        }
    };
    load(0);
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    f8_stage_row<XT>(static_cast<const uint8_t*>(p.x) + (int64_t)t * H * ES, H, xc, xs, tid, 64 * F8A_NW);
    __syncthreads();
    v4f acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    const int steps = (G + F8A_NW - 1) / F8A_NW;
    for (int j0 = 0; j0 < steps; j0 += F8A_D) {
        if (j0) load(j0);
#pragma unroll
        for (int d = 0; d < F8A_D; ++d) {
            const int b = wave + F8A_NW * (j0 + d);
            if (b >= G) break;
            u32x4 Bv[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
            if (i == 0) {
                Bv[0] = *reinterpret_cast<const u32x4*>(xc + F8B * b + 16 * q);
                Bv[1] = *reinterpret_cast<const u32x4*>(xc + F8B * b + 64 + 16 * q);
            }
            const float sx = xs[b], s[2] = {sg[b] * sx, su[b] * sx};
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const v4f part = f8_mfma(A[d][m], Bv);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(s[m], part[r], acc[m][r]);
            }
        }
    }
    if (i == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[(wave * 2 + m) * 16 + 4 * q + r] = acc[m][r];
    }
    __syncthreads();
    if (tid < 16 && n0 + tid < I) {
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < F8A_NW; ++w) g += red[(2 * w) * 16 + tid], u += red[(2 * w + 1) * 16 + tid];
        p.h[(int64_t)a * I + n0 + tid] = f8_act(L, g, u);
    }
}

__global__ void __launch_bounds__(64 * F8D_NW) fp8_down_kernel(F8Moe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, G = (int)f8_blocks(I);
    const int t = blockIdx.y, n0 = (int)blockIdx.x * 16;
    __shared__ float red[F8D_NW * 16];
    uint8_t* hc = smem;                                              // [expert of the chunk][G 128]
    float* hs = reinterpret_cast<float*>(smem + p.chunk * G * F8B);  // [expert of the chunk][G]
    const int32_t* slots = p.slots + (int64_t)t * k;
    const float* wts = p.wts + (int64_t)t * k;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < k; c0 += p.chunk) {  // workgroup-uniform
        const int nc = k - c0 < p.chunk ? k - c0 : p.chunk, units = nc * G;
        // unit u: K block u % G of the chunk's expert u / G, one wave's
        auto live = [&](int j) {
            const int s = uniform(slots[c0 + j]);
            return s >= 0 && s < p.n_slots ? s : -1;
        };
        u32x4 A[F8D_D][2];
        float sc[F8D_D];
        auto load = [&](int u0) {
#pragma unroll
            for (int d = 0; d < F8D_D; ++d) {
                const int u = u0 + F8D_NW * d;
                sc[d] = 0.0f;
                if (u >= units) continue;
                const int j = u / G, b = u % G, s = live(j);
                if (s < 0) continue;
                const uint8_t* base = p.pool + s * L.slot_bytes;
                const __amdgpu_buffer_rsrc_t r =
                    f8_buf(base + L.down_off + (int64_t)n0 * I, (int64_t)(H - n0 < 16 ? H - n0 : 16) * I);
                const uint32_t o = (uint32_t)(F8B * b + 16 * q);
                A[d][0] = f8_ld(r, f8_off((uint32_t)(i * I), o, (uint32_t)I));
                A[d][1] = f8_ld(r, f8_off((uint32_t)(i * I), o + 64, (uint32_t)I));
                sc[d] = wts[c0 + j] * reinterpret_cast<const float*>(base + L.down_scales_off)[n0 / F8B * G + b];
            }
        };
        load(wave);
        if (c0) __syncthreads();  // the chunk before is used up
        for (int j = 0; j < nc; ++j)
            if (live(j) >= 0)
                f8_stage_row<TSA_F32>(p.h + ((int64_t)t * k + c0 + j) * I, I, hc + j * G * F8B, hs + j * G, tid, 64 * F8D_NW);
        __syncthreads();
        for (int u0 = wave; u0 < units; u0 += F8D_NW * F8D_D) {
            if (u0 != wave) load(u0);
#pragma unroll
            for (int d = 0; d < F8D_D; ++d) {
                const int u = u0 + F8D_NW * d;
                if (u >= units || live(u / G) < 0) continue;
                u32x4 Bv[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
                if (i == 0) {
                    Bv[0] = *reinterpret_cast<const u32x4*>(hc + F8B * u + 16 * q);
                    Bv[1] = *reinterpret_cast<const u32x4*>(hc + F8B * u + 64 + 16 * q);
                }
                const float s = sc[d] * hs[u];
                const v4f part = f8_mfma(A[d], Bv);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] = fmaf(s, part[r], acc[r]);
            }
        }
    }
    if (i == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wave * 16 + 4 * q + r] = acc[r];
    }
    __syncthreads();
    if (tid < 16 && n0 + tid < H) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < F8D_NW; ++w) v += red[16 * w + tid];
        store_out(p.y, p.y_dtype, (int64_t)t * H + n0 + tid, v);
    }
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// h [T k, I] fp32, then the routed selection.
int64_t f8_decode_ws_bytes(const tsa_expert_layout& L, int64_t T, int k) {
    return align256(T * k * L.inter * 4) + 2 * align256(T * k * 4);
}

// Calls whose routing runs inside the gate_up kernel.
bool f8_routes(int64_t T, int64_t E, int k) { return E <= 256 && k <= FUSED_MAXK && T * k <= 65535; }

int f8_decode(const tsa_expert_layout& L, const uint8_t* pool, int64_t n_slots, const int32_t* slots, const float* wts,
              const void* logits, int logits_dtype, int mode, const int32_t* expert_slot, int64_t E, int32_t* idx_out,
              float* w_out, int64_t T, int k, const void* x, int x_dtype, void* y, int y_dtype, uint8_t* ws,
              int64_t ws_bytes, hipStream_t st) {
    TSA_REQUIRE(T >= 1 && T * k <= 65535 && (!logits || f8_routes(T, E, k)), TSA_ERR_SHAPE, "FP8 decode: T %lld, k %d, E %lld",
                (long long)T, k, (long long)E);
    TSA_REQUIRE(ws_bytes >= f8_decode_ws_bytes(L, T, k), TSA_ERR_WORKSPACE, "workspace too small for the FP8 decode");
    TSA_REQUIRE(((reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(ws)) & 15) == 0,
                TSA_ERR_INVALID_ARG, "FP8 experts: pool, x and workspace must be 16-byte aligned");
    F8Moe p{};
    p.L = L;
    p.pool = pool;
    p.n_slots = n_slots;
    p.slots = slots;
    p.wts = wts;
    p.logits = logits;
    p.logits_dtype = logits_dtype;
    p.route_mode = mode;
    p.expert_slot = expert_slot;
    p.E = (int)E;
    p.k = k;
    p.idx_out = idx_out;
    p.w_out = w_out;
    p.x = x;
    p.h = reinterpret_cast<float*>(ws);
    p.tab_slot = reinterpret_cast<int32_t*>(ws + align256(T * k * L.inter * 4));
    p.tab_w = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.tab_slot) + align256(T * k * 4));
    p.y = y;
    p.y_dtype = y_dtype;
    const int GH = (int)f8_blocks(L.hidden), GI = (int)f8_blocks(L.inter), row = GI * (F8B + 4);
    p.chunk = k * row <= 60 * 1024 ? k : 60 * 1024 / row;  // at least 3 rows of 16384
    const int lds_a = GH * (F8B + 4) + F8A_NW * 32 * 4, lds_b = p.chunk * row;
    const void* fa = x_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_F32>)
                     : x_dtype == TSA_F16 ? reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_F16>)
                                          : reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_BF16>);
    void* args[] = {&p};
    TSA_HIP_CHECK(hipLaunchKernel(fa, dim3((unsigned)((L.inter + 15) / 16), (unsigned)(T * k)), dim3(64 * F8A_NW), args, lds_a, st));
    F8Moe pb = p;  // the down launch reads the routed table, or the caller's
    if (logits) {
        pb.slots = p.tab_slot;
        pb.wts = p.tab_w;
    }
    void* args_b[] = {&pb};
    TSA_HIP_CHECK(hipLaunchKernel(reinterpret_cast<const void*>(&fp8_down_kernel), dim3((unsigned)((L.hidden + 15) / 16), (unsigned)T),
                                  dim3(64 * F8D_NW), args_b, lds_b, st));
    return TSA_OK;
}

// Requirements beyond the common ones of validate_layout: "" if met.
const char* f8_unsupported(const tsa_expert_layout& L) {
    if (L.gate_bias_off >= 0 || L.down_bias_off >= 0) return "FP8 experts carry no biases";
    if ((L.slot_bytes | L.gate_off | L.up_off | L.down_off) & 15) return "FP8 slots and matrices must start on multiples of 16 bytes";
    if ((L.gate_scales_off | L.down_scales_off) & 3) return "FP8 scales must start on multiples of 4 bytes";
    return "";
}

}  // namespace tsa
