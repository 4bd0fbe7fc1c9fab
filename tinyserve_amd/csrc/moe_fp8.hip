// MoE layers over FP8 experts (e4m3 codes with a float32 scale per 128 x 128 block).
//
// Definition, per token: x quantised per 128 values (fp8_common.h); for each selected expert
// h = act(Wg x, Wu x) in float32, quantised the same way; y = sum_j w_j Wd h, rounded once.
//
// Few tokens: two launches ordered by the stream. gate_up: one workgroup per (token, expert) pair
// and 8 channels; down: one per token and 8 outputs, over all the token's experts, so every
// output has one writer. Each is a stream of weights into the A operands of matrix
// instructions (one or two columns of B in use: the matrix cores are idle otherwise).
//
// Gate and up are summed to float32 accuracy (f8_mfma's WIDE), here and for many tokens: their result is
// quantised again, and a sum off by 1e-5 takes some 3 codes in 10000 to another side, off by 6% each.
// A layer's bf16 result is then off by its own rounding (0.0017 rms over 12 to 785 tokens), with the FP8
// instructions by 0.0018 to 0.0032. us, float32 accuracy / FP8 instructions: hidden 2880, 32 experts top-4,
// 8 layers of 4 tokens 632 / 613, a layer of 2048 570 / 490; hidden 2048, 128 experts top-8, 24 tokens 58 / 57,
// 1024 tokens 210 / 187. Down is summed so where the layer's result is float32; for 16-bit ones the FP8
// instructions' sums are far below the last rounding. A layer's us for float32 / bf16 results: hidden 2880, 32
// experts top-4, 4 and 2048 tokens 74 / 71 and 605 / 568; hidden 2048, 128 experts top-8, 1, 24 and 1024 tokens
// 15.7 / 15.3, 48.5 / 47.0 and 220 / 208.
#include "fp8_gemm.h"
#include "moe_group.h"

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

constexpr int F8A_NW = 8, F8A_D = 3, F8A_XC = 1;  // gate_up: waves; K blocks in flight per wave; chunks of x held per thread
constexpr int F8D_NW = 8, F8D_D = 3, F8D_HC = 2;  // down: the same with its units and h

__device__ __forceinline__ float f8_act(const tsa_expert_layout& L, float gate, float up) {
    if (L.act == TSA_ACT_SWIGLU_OAI) {
        // the limits by comparisons: a minimum or maximum would give its other operand for a NaN
        const float lim = L.swiglu_limit, g = gate > lim ? lim : gate, u = up > lim ? lim : up < -lim ? -lim : up;
        const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * (L.swiglu_alpha * g));
        return (u + 1.0f) * g * __builtin_amdgcn_rcpf(1.0f + e);
    }
    return silu_mul_fast(gate, up);
}

// One workgroup per (token, expert) pair and 8 channels: rows 0 .. 7 of the tile are the channels' gate
// rows, 8 .. 15 their up rows, so one pair gives enough workgroups (768 at inter 768 and top-8, three
// whole rounds of the CUs; tiles of 16 channels give 384, one and a half: 9.5 us against 7.7, both with the
// FP8 instructions; 8.1 with the widened products). Loads
// go out in the order of their use: x, the routing's inputs, then every weight of the tile; x is
// quantised while the weights are on their way.
template <int XT>
__global__ void __launch_bounds__(64 * F8A_NW) fp8_gate_up_kernel(F8Moe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, G = (int)f8_blocks(H), GI = (int)f8_blocks(I);
    const int a = blockIdx.y, t = a / k, jj = a % k, n0 = (int)blockIdx.x * 8;
    uint8_t* xc = smem;
    float* xs = reinterpret_cast<float*>(smem + G * F8B);
    float* red = reinterpret_cast<float*>(smem + (G * (F8B + 4) + 15) / 16 * 16);  // [wave][gate / up][channel]
    constexpr int ES = XT == TSA_F32 ? 4 : 2, NT = 64 * F8A_NW;
    const uint8_t* xrow = static_cast<const uint8_t*>(p.x) + (int64_t)t * H * ES;
    float xv[F8A_XC][8];
#pragma unroll
    for (int c = 0; c < F8A_XC; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) xv[c][e] = 0.0f;
        if (8 * (tid + NT * c) < H) f8_load8<XT>(xrow, tid + NT * c, xv[c]);
    }
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
    const __amdgpu_buffer_rsrc_t r = f8_buf(base, L.slot_bytes);
    const uint32_t row = n0 + (i & 7) < I ? (uint32_t)((i >> 3) ? L.up_off : L.gate_off) + (uint32_t)(n0 + (i & 7)) * (uint32_t)H
                                          : 0x80000000u;
    const uint32_t scale = (uint32_t)L.gate_scales_off + 4u * (uint32_t)(((q >> 1) * GI + n0 / F8B) * G);
    u32x4 A[F8A_D][2];
    float ws[F8A_D];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < F8A_D; ++d) {
            const int b = wave + F8A_NW * (j0 + d);
            if (b >= G) break;
            const uint32_t o = (uint32_t)(F8B * b + 16 * q);
            A[d][0] = f8_ld(r, o < (uint32_t)H ? row + o : 0x80000000u);
            A[d][1] = f8_ld(r, o + 64 < (uint32_t)H ? row + o + 64 : 0x80000000u);
            ws[d] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (int)(scale + 4u * (uint32_t)b), 0, 0));
        }
    };
    load(0);
#pragma unroll
    for (int c = 0; c < F8A_XC; ++c)
        if (tid + NT * c < 16 * G) f8_put8<XT == TSA_F32>(xv[c], tid + NT * c, xc, xs);
    for (int c = tid + NT * F8A_XC; c < 16 * G; c += NT) {  // the rest of a long row
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (8 * c < H) f8_load8<XT>(xrow, c, v);
        f8_put8<XT == TSA_F32>(v, c, xc, xs);
    }
    __syncthreads();
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
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
            const float s = ws[d] * xs[b];
            const v4f part = f8_mfma<true>(A[d], Bv);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(s, part[e], acc[e]);
        }
    }
    if (i == 0) *reinterpret_cast<v4f*>(red + wave * 16 + 4 * q) = acc;
    __syncthreads();
    if (tid < 8 && n0 + tid < I) {
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < F8A_NW; ++w) g += red[16 * w + tid], u += red[16 * w + 8 + tid];
        p.h[(int64_t)a * I + n0 + tid] = f8_act(L, g, u);
    }
}

__device__ const uint32_t f8_zeros[4] = {0, 0, 0, 0};  // what lanes past a matrix read

// One workgroup per token and 8 outputs, over all the token's experts: rows 0 .. 7 of a tile are the
// outputs' rows of an even expert, 8 .. 15 those of the next, which meet columns 0 and 1 (their h); a
// unit is a K block of such a pair, and the waves take the units in turn.
template <bool WIDE>
__global__ void __launch_bounds__(64 * F8D_NW, 4) fp8_down_kernel(F8Moe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, G = (int)f8_blocks(I);
    const int t = blockIdx.y, n0 = (int)blockIdx.x * 8;
    constexpr int NT = 64 * F8D_NW;
    __shared__ __align__(16) float red[F8D_NW * 16];
    uint8_t* hc = smem;                                              // [expert of the chunk][G 128]
    float* hs = reinterpret_cast<float*>(smem + p.chunk * G * F8B);  // [expert of the chunk][G]
    // lane j: the token's j-th slot (-1: none) and weight
    int my_slot = -1;
    float my_w = 0.0f;
    if (lane < k) {
        my_slot = p.slots[(int64_t)t * k + lane];
        my_w = p.wts[(int64_t)t * k + lane];
    }
    my_slot = my_slot < p.n_slots ? my_slot : -1;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < k; c0 += p.chunk) {  // workgroup-uniform
        const int nc = k - c0 < p.chunk ? k - c0 : p.chunk, units = (nc + 1) / 2 * G, tasks = nc * G * 16;
        // h of the chunk: [expert][group][16 chunks of 8], a dead expert's as zeros
        const float* hrow = p.h + ((int64_t)t * k + c0) * I;
        auto load_h = [&](int c, float (&v)[8]) {
            const int j = c / (G * 16), o = 8 * (c % (G * 16));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            const int slot = __shfl(my_slot, (c0 + j) & 63, 64);  // outside the condition: every lane takes part
            if (c < tasks && o < I && slot >= 0) f8_load8<TSA_F32>(hrow + (int64_t)j * I, o / 8, v);
        };
        float hv[F8D_HC][8];
#pragma unroll
        for (int c = 0; c < F8D_HC; ++c) load_h(tid + NT * c, hv[c]);
        u32x4 A[F8D_D][2];
        float sc[F8D_D];
        auto load = [&](int u0) {
#pragma unroll
            for (int d = 0; d < F8D_D; ++d) {
                const int u = u0 + F8D_NW * d, pair = u / G, b = u % G;
                if (u >= units) break;
                const int ja = 2 * pair + (i >> 3), js = 2 * pair + (q >> 1);  // of the lane's row of A, of its sums
                // every lane takes part in the shuffles: one that is off has 0 (a slot) read from it
                const int la = __shfl(my_slot, (c0 + ja) & 63, 64), ls = __shfl(my_slot, (c0 + js) & 63, 64);
                const float w = __shfl(my_w, (c0 + js) & 63, 64);
                const int sa = ja < nc ? la : -1, ss = js < nc ? ls : -1;
                const int o = F8B * b + 16 * q, row = n0 + (i & 7);
                const uint8_t* at = p.pool + (int64_t)sa * L.slot_bytes + L.down_off + (int64_t)row * I + o;
                const bool ok = sa >= 0 && row < H;
                const void* z = f8_zeros;
                A[d][0] = *static_cast<const u32x4*>(ok && o < I ? at : z);
                A[d][1] = *static_cast<const u32x4*>(ok && o + 64 < I ? at + 64 : z);
                const float* sp = reinterpret_cast<const float*>(p.pool + (int64_t)ss * L.slot_bytes + L.down_scales_off) + n0 / F8B * G + b;
                const float ws = *(ss >= 0 ? sp : static_cast<const float*>(z));
                sc[d] = ss >= 0 ? w * ws : 0.0f;  // a dead expert's weight may be anything
            }
        };
        load(wave);
        if (c0) __syncthreads();  // the chunk before is used up
#pragma unroll
        for (int c = 0; c < F8D_HC; ++c)
            if (tid + NT * c < tasks) f8_put8<false>(hv[c], tid + NT * c, hc, hs);
        for (int c = tid + NT * F8D_HC; c < (tasks + 63) / 64 * 64; c += NT) {  // whole waves: load_h shuffles
            float v[8];
            load_h(c, v);
            if (c < tasks) f8_put8<false>(v, c, hc, hs);
        }
        __syncthreads();
        for (int u0 = wave; u0 < units; u0 += F8D_NW * F8D_D) {
            if (u0 != wave) load(u0);
#pragma unroll
            for (int d = 0; d < F8D_D; ++d) {
                const int u = u0 + F8D_NW * d;
                if (u >= units) break;
                const int pair = u / G, b = u % G, j = 2 * pair + i, js = 2 * pair + (q >> 1);
                u32x4 Bv[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
                if (i < 2 && j < nc) {
                    Bv[0] = *reinterpret_cast<const u32x4*>(hc + F8B * (j * G + b) + 16 * q);
                    Bv[1] = *reinterpret_cast<const u32x4*>(hc + F8B * (j * G + b) + 64 + 16 * q);
                }
                const float s = js < nc ? sc[d] * hs[js * G + b] : 0.0f;
                const v4f part = f8_mfma<WIDE>(A[d], Bv);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(s, part[e], acc[e]);
            }
        }
    }
    if (i == (q >> 1)) *reinterpret_cast<v4f*>(red + wave * 16 + 4 * q) = acc;  // an expert's rows in its own column
    __syncthreads();
    if (tid < 8 && n0 + tid < H) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < F8D_NW; ++w) v += red[16 * w + tid] + red[16 * w + 8 + tid];
        store_out(p.y, p.y_dtype, (int64_t)t * H + n0 + tid, v);
    }
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// ---------------------------------------------------------------- many tokens
// Four launches: (1) the assignments grouped by expert with a table of token tiles (workgroup 0), x
// quantised (the others); (2) gate_up over the tiles: 128 channels of gate and of up per workgroup, so
// the epilogue holds whole groups of h and quantises them; (3) down, each assignment's output in
// float32 at the assignment's place; (4) the weighted sums. (Outputs rounded to bf16 between (3) and (4)
// save 12 us at 1024 tokens, 128 experts top-8, and add an error of 0.0019 to the result, more than its own
// rounding's.)
struct F8Group {
    tsa_expert_layout L;
    const uint8_t* pool;
    int64_t n_slots;
    const int32_t* expert_slot;
    int64_t E;
    const int32_t* idx;
    const float* wts;
    int T, k;
    const void* x;
    void* y;
    int y_dtype;
    int32_t *counts, *offsets, *perm;
    int* n_entries;
    int4* table;  // (slot, first sorted row, rows, -)
    int tile_rows;
    uint8_t* xq;
    float* xs;
    uint8_t* hq;  // [sorted row, I]
    float* hs;
    float* yk;  // [T k, H]
};

constexpr int F8P_ROWS = 4;  // rows of x per quantising workgroup, 128 threads each

template <int XT>
__global__ void __launch_bounds__(GROUP_THREADS) fp8_prepare_kernel(F8Group p) {
    extern __shared__ __align__(16) unsigned char gsm[];
    if (blockIdx.x == 0) {
        const GroupTiles tiles{p.expert_slot, p.n_slots, p.tile_rows, p.n_entries, p.table};
        group_assignments<true>(p.idx, (int64_t)p.T * p.k, (int)p.E, p.counts, p.offsets, p.perm, tiles, GROUP_WAVES, gsm);
        return;
    }
    const int H = (int)p.L.hidden, tasks = (int)f8_blocks(H) * 16, tid = (int)threadIdx.x & 127;
    const int t = ((int)blockIdx.x - 1) * F8P_ROWS + ((int)threadIdx.x >> 7);
    if (t >= p.T) return;
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const uint8_t* row = static_cast<const uint8_t*>(p.x) + (int64_t)t * H * ES;
    for (int c = tid; c < tasks; c += 128) {
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (8 * c < H) f8_load8<XT>(row, c, v);
        const float s = f8_scale(f8_group_max(v));
        const uint2 o = f8_codes8<XT == TSA_F32>(v, s);
        if (8 * c < H) *reinterpret_cast<uint2*>(p.xq + (int64_t)t * H + 8 * c) = o;
        if ((c & 15) == 0) p.xs[(int64_t)t * (tasks >> 4) + (c >> 4)] = s;
    }
}

// The workgroup's (entry, tile) of n_entries x tiles: each XCD takes a run of the entries with all
// their tiles (an expert's entries and an entry's tiles share an L2). False: none is left for it.
__device__ __forceinline__ bool f8_work(const int* n_entries, int tiles, int& entry, int& tile) {
    const int total = uniform(*n_entries) * tiles, lin = (int)blockIdx.x, xcd = lin & 7, q8 = total >> 3, rem = total & 7;
    if ((lin >> 3) >= q8 + (xcd < rem ? 1 : 0)) return false;
    const int wid = xcd * q8 + (xcd < rem ? xcd : rem) + (lin >> 3);
    entry = wid / tiles;
    tile = wid % tiles;
    return true;
}

template <class C>
__global__ void __launch_bounds__(C::THREADS) fp8_group_gate_up_kernel(F8Group p) {
    extern __shared__ __align__(16) uint8_t smem[];
    static_assert(C::RN == 2 * F8B && C::LDS >= C::TM * (F8B + 4 * C::WR), "one group of h per workgroup");
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, GH = (int)f8_blocks(H), GI = (int)f8_blocks(I);
    int entry, tile;
    if (!f8_work(p.n_entries, GI, entry, tile)) return;
    const int4 e = p.table[entry];
    const int slot = uniform(e.x), row0 = uniform(e.y), tn = uniform(e.z), c0 = tile * F8B;
    const uint8_t* base = p.pool + (int64_t)slot * L.slot_bytes;
    const float* sg = reinterpret_cast<const float*>(base + L.gate_scales_off) + (int64_t)tile * GH;
    F8Operands<2> o;
    o.w[0] = base + L.gate_off + (int64_t)c0 * H;
    o.w[1] = base + L.up_off + (int64_t)c0 * H;
    o.w_rows = I - c0;
    o.ws[0] = sg;
    o.ws[1] = sg + (int64_t)GI * GH;
    o.x = p.xq;
    o.xs = p.xs;
    o.x_records = (uint32_t)p.T * (uint32_t)H;
    o.xs_records = (uint32_t)p.T * (uint32_t)GH * 4u;
    o.K = H;
    o.G = GH;
    v4f acc[C::MR][C::MT];
    f8_tile<C, 2, true>(o, smem, tn, [&](int r) { return r < tn ? p.perm[row0 + r] / p.k : -1; }, acc);

    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    constexpr int MP = C::MR / 2;
    uint8_t* stage = smem;                                              // [token][channel]
    uint32_t* top = reinterpret_cast<uint32_t*>(smem + C::TM * F8B);    // [wr][token]
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < MP; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                acc[j][t][r] = f8_act(L, acc[j][t][r], acc[MP + j][t][r]);
                m = max(m, __float_as_uint(acc[j][t][r]) & 0x7FFFFFFFu);
            }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if (q == 0) top[wr * C::TM + 16 * (C::MT * wt + t) + i] = m;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
        const int tk = 16 * (C::MT * wt + t) + i;
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < C::WR; ++w) m = max(m, top[w * C::TM + tk]);
        const float s = f8_scale(m);
#pragma unroll
        for (int j = 0; j < MP; ++j)
            *reinterpret_cast<uint32_t*>(stage + tk * F8B + 16 * (wr * MP + j) + 4 * q) = f8_codes4(acc[j][t], s);
        if (wr == 0 && q == 0 && tk < tn) p.hs[(int64_t)(row0 + tk) * GI + tile] = s;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < tn * 8; c += C::THREADS) {
        const int tk = c >> 3, col = 16 * (c & 7);
        if (c0 + col < I)
            *reinterpret_cast<u32x4*>(p.hq + (int64_t)(row0 + tk) * I + c0 + col) = *reinterpret_cast<const u32x4*>(stage + tk * F8B + col);
    }
}

template <class C, bool WIDE>
__global__ void __launch_bounds__(C::THREADS) fp8_group_down_kernel(F8Group p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, GI = (int)f8_blocks(I);
    int entry, tile;
    if (!f8_work(p.n_entries, (H + C::RN - 1) / C::RN, entry, tile)) return;
    const int4 e = p.table[entry];
    const int slot = uniform(e.x), row0 = uniform(e.y), tn = uniform(e.z), n0 = tile * C::RN;
    const uint8_t* base = p.pool + (int64_t)slot * L.slot_bytes;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR, nw = n0 + wr * C::MR * 16;
    static_assert(F8B % (C::MR * 16) == 0, "a wave's rows share their scales");
    F8Operands<1> o;
    o.w[0] = base + L.down_off + (int64_t)n0 * I;
    o.w_rows = H - n0;
    o.ws[0] = reinterpret_cast<const float*>(base + L.down_scales_off) + (int64_t)(nw < H ? nw / F8B : 0) * GI;
    o.x = p.hq + (int64_t)row0 * I;
    o.xs = p.hs + (int64_t)row0 * GI;
    o.x_records = (uint32_t)tn * (uint32_t)I;
    o.xs_records = (uint32_t)tn * (uint32_t)GI * 4u;
    o.K = I;
    o.G = GI;
    v4f acc[C::MR][C::MT];
    f8_tile<C, 1, WIDE>(o, smem, tn, [&](int r) { return r < tn ? r : -1; }, acc);
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
        const int tk = 16 * (C::MT * wt + t) + i;
        if (tk >= tn) continue;
        float* dst = p.yk + (int64_t)p.perm[row0 + tk] * H;
#pragma unroll
        for (int m = 0; m < C::MR; ++m) {
            const int n = nw + 16 * m + 4 * q;  // H % 32 == 0: all four or none
            if (n < H) *reinterpret_cast<v4f*>(dst + n) = acc[m][t];
        }
    }
}

// y[t] = sum_j w[t, j] yk[t k + j], in order of j; a thread 8 values of a row.
__global__ void __launch_bounds__(256) fp8_combine_kernel(F8Group p) {
    const int H = (int)p.L.hidden, per = H / 8;
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

using GateUp128 = F8Tile<4, 2, 4, 4, 3>;  // 128 channels x 128 tokens, 8 waves
using GateUp64 = F8Tile<4, 2, 4, 2, 3>;   // x 64
using Down128 = F8Tile<4, 2, 4, 4, 3>;    // 256 rows x 128 tokens
using Down64 = F8Tile<4, 1, 2, 4, 3>;     // 128 x 64, two workgroups per CU

constexpr int64_t F8_CHUNK = 131072;  // assignments at a time: bounds the workspace (1.1 GiB at hidden 2048)

int64_t group_tokens(int64_t T, int k) {
    const int64_t c = F8_CHUNK / k > 0 ? F8_CHUNK / k : 1;
    return T < c ? T : c;
}

struct F8Places {
    int64_t counts, offsets, perm, n_entries, table, xq, xs, hq, hs, yk, bytes;
};

F8Places group_places(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    const int64_t n = T * k, H = L.hidden, I = L.inter;
    F8Places w;
    int64_t at = 0;
    auto take = [&](int64_t b) {
        const int64_t r = at;
        at += align256(b);
        return r;
    };
    w.counts = take(E * 4);
    w.offsets = take((E + 1) * 4);
    w.perm = take(n * 4);
    w.n_entries = take(4);
    w.table = take((n / 64 + E) * 16);
    w.xq = take(T * H);
    w.xs = take(T * f8_blocks(H) * 4);
    w.hq = take(n * I);
    w.hs = take(n * f8_blocks(I) * 4);
    w.yk = take(n * H * 4);
    w.bytes = at;
    return w;
}

template <class GU, class DN>
int group_gemms(const F8Group& p, int64_t entries, hipStream_t st) {
    F8Group q = p;
    void* args[] = {&q};
    const void* fg = reinterpret_cast<const void*>(&fp8_group_gate_up_kernel<GU>);
    const void* fd = p.y_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_group_down_kernel<DN, true>)
                                          : reinterpret_cast<const void*>(&fp8_group_down_kernel<DN, false>);
    TSA_HIP_CHECK(ensure_dynamic_lds(fg, GU::LDS));
    TSA_HIP_CHECK(ensure_dynamic_lds(fd, DN::LDS));
    static_assert(GU::TM == DN::TM, "one table of token tiles");
    const int64_t tg = f8_blocks(p.L.inter), td = (p.L.hidden + DN::RN - 1) / DN::RN;
    auto grid = [](int64_t n) { return dim3((unsigned)((n + 7) / 8 * 8)); };  // whole rounds of XCDs
    TSA_HIP_CHECK(hipLaunchKernel(fg, grid(entries * tg), dim3(GU::THREADS), args, GU::LDS, st));
    TSA_HIP_CHECK(hipLaunchKernel(fd, grid(entries * td), dim3(DN::THREADS), args, DN::LDS, st));
    return TSA_OK;
}

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
    const int lds_a = (GH * (F8B + 4) + 15) / 16 * 16 + F8A_NW * 16 * 4, lds_b = p.chunk * row;
    const void* fa = x_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_F32>)
                     : x_dtype == TSA_F16 ? reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_F16>)
                                          : reinterpret_cast<const void*>(&fp8_gate_up_kernel<TSA_BF16>);
    void* args[] = {&p};
    TSA_HIP_CHECK(hipLaunchKernel(fa, dim3((unsigned)((L.inter + 7) / 8), (unsigned)(T * k)), dim3(64 * F8A_NW), args, lds_a, st));
    F8Moe pb = p;  // the down launch reads the routed table, or the caller's
    if (logits) {
        pb.slots = p.tab_slot;
        pb.wts = p.tab_w;
    }
    void* args_b[] = {&pb};
    const void* fb = y_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_down_kernel<true>)
                                        : reinterpret_cast<const void*>(&fp8_down_kernel<false>);
    TSA_HIP_CHECK(hipLaunchKernel(fb, dim3((unsigned)((L.hidden + 7) / 8), (unsigned)T), dim3(64 * F8D_NW), args_b, lds_b, st));
    return TSA_OK;
}

// Calls that the grouped kernels take (us of a layer grouped / as pairs: hidden 2048, 128 experts top-8, 5 / 8 /
// 24 tokens 36 / 38 / 52 and 42 / 59 / 153; hidden 2880, 32 experts top-4, 5 / 8 tokens 74 / 76 and 98 / 142).
bool f8_group_supported(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    return L.format == TSA_EXPERT_FP8 && T > F8_PAIR_TOKENS && E <= MAX_GROUP_E && k <= 64;
}

int64_t f8_group_workspace_bytes(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    return group_places(L, group_tokens(T, k), k, E).bytes;
}

int f8_group_prefill(const tsa_expert_layout& L, const uint8_t* pool, int64_t n_slots, const int32_t* expert_slot, int64_t E,
                     const int32_t* idx, const float* weights, int64_t T, int k, const void* x, int x_dtype, void* y,
                     int y_dtype, uint8_t* ws, hipStream_t st) {
    const int64_t step = group_tokens(T, k), H = L.hidden;
    const F8Places w = group_places(L, step, k, E);
    const int lds = group_lds_bytes((int)E);
    const void* fp = x_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_prepare_kernel<TSA_F32>)
                     : x_dtype == TSA_F16 ? reinterpret_cast<const void*>(&fp8_prepare_kernel<TSA_F16>)
                                          : reinterpret_cast<const void*>(&fp8_prepare_kernel<TSA_BF16>);
    TSA_HIP_CHECK(ensure_dynamic_lds(fp, lds));
    for (int64_t t0 = 0; t0 < T; t0 += step) {
        F8Group p{};
        p.L = L;
        p.pool = pool;
        p.n_slots = n_slots;
        p.expert_slot = expert_slot;
        p.E = E;
        p.T = (int)(T - t0 < step ? T - t0 : step);
        p.k = k;
        p.idx = idx + t0 * k;
        p.wts = weights + t0 * k;
        p.x = static_cast<const uint8_t*>(x) + t0 * H * dtype_size(x_dtype);
        p.y = static_cast<uint8_t*>(y) + t0 * H * dtype_size(y_dtype);
        p.y_dtype = y_dtype;
        p.counts = reinterpret_cast<int32_t*>(ws + w.counts);
        p.offsets = reinterpret_cast<int32_t*>(ws + w.offsets);
        p.perm = reinterpret_cast<int32_t*>(ws + w.perm);
        p.n_entries = reinterpret_cast<int*>(ws + w.n_entries);
        p.table = reinterpret_cast<int4*>(ws + w.table);
        p.xq = ws + w.xq;
        p.xs = reinterpret_cast<float*>(ws + w.xs);
        p.hq = ws + w.hq;
        p.hs = reinterpret_cast<float*>(ws + w.hs);
        p.yk = reinterpret_cast<float*>(ws + w.yk);
        const int64_t n = (int64_t)p.T * k;
        // Few tokens per expert fill tiles of 64 better, many read each weight for 128: us of a layer
        // with tiles of 64 / 128, hidden 2048, 128 experts top-8, 24 / 300 / 600 / 1024 tokens 52 / 124 /
        // 162 / 211 and 56 / 140 / 167 / 210; hidden 2880, 32 experts top-4, 100 / 300 / 700 / 2048 tokens
        // 195 / 246 / 359 / 729 and 206 / 252 / 359 / 581. (Tiles of 32 measured 8 to 60% slower from 24 tokens.)
        p.tile_rows = n <= 48 * E ? 64 : 128;
        const int64_t entries = n / p.tile_rows + (E < n ? E : n);
        void* args[] = {&p};
        TSA_HIP_CHECK(hipLaunchKernel(fp, dim3((unsigned)(1 + (p.T + F8P_ROWS - 1) / F8P_ROWS)), dim3(GROUP_THREADS), args, lds, st));
        const int rc = p.tile_rows == 64 ? group_gemms<GateUp64, Down64>(p, entries, st) : group_gemms<GateUp128, Down128>(p, entries, st);
        if (rc) return rc;
        const dim3 grid((unsigned)(((int64_t)p.T * (H / 8) + 255) / 256));
        hipLaunchKernelGGL(fp8_combine_kernel, grid, dim3(256), 0, st, p);
        TSA_LAUNCH_CHECK();
    }
    return TSA_OK;
}

// Requirements beyond the common ones of validate_layout: "" if met.
const char* f8_unsupported(const tsa_expert_layout& L) {
    if (L.gate_bias_off >= 0 || L.down_bias_off >= 0) return "FP8 experts carry no biases";
    if ((L.slot_bytes | L.gate_off | L.up_off | L.down_off) & 15) return "FP8 slots and matrices must start on multiples of 16 bytes";
    if (L.slot_bytes >= ((int64_t)1 << 31)) return "FP8 slots of 2^31 bytes and more are not supported";
    if ((L.gate_scales_off | L.down_scales_off) & 3) return "FP8 scales must start on multiples of 4 bytes";
    return "";
}

}  // namespace tsa
