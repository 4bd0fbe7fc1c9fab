// MoE layers over experts in bfloat16, float16 or int8 (a float32 scale for each row).
//
// Definition, per token: for each selected expert h = act(Wg x, Wu x) in float32; 16 bits: h rounded to the weights'
// type, which x has too; int8: x and h quantised per token (int8_common.h); y = sum_j w_j Wd h in float32, rounded
// once.
//
// Few tokens: two launches ordered by the stream. gate_up: one workgroup per (token, expert) pair and 8 channels; down:
// one per token and 8 outputs, over all the token's experts, so every output has one writer. Each is a stream of
// weights into the A operands of matrix instructions (one or two columns of B in use).
#include "int8_common.h"
#include "mm_epilogue.h"
#include "moe_grouped.h"

namespace tsa {
int i8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st);

namespace {

template <class E>
constexpr bool is_int8 = std::is_same<E, MmI8>::value;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(int v) { return (float)v; }

struct DenseMoe {
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
    void* h;  // [T k, I]: 16 bits, or float32 (int8 experts)
    void* y;
    int y_dtype;
    int chunk;  // down, int8: experts staged in LDS at a time
};

constexpr int DMA_NW = 8, DMA_D = 4;  // gate_up: waves; steps of 128 bytes in flight per wave
constexpr int DMD_NW = 8, DMD_D = 4;  // down

// The slot of assignment a (token t, its jj-th), selected by every wave; the token's first workgroup writes all the
// selections for the down launch.
__device__ __forceinline__ int64_t dense_slot(const DenseMoe& p, int a, int t, int jj, int lane, int wave) {
    if (!p.logits) return uniform(p.slots[a]);
    const int k = p.k;
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
        return uniform(s_slot[0]);  // lane 0's own write
    }
    uint32_t myk;
    int mysel, myslot;
    select_topk(p, lane, lg, es, jj + 1, myk, mysel, myslot);
    return __builtin_amdgcn_readlane(myslot, jj);
}

// One workgroup per (token, expert) pair and 8 channels: rows 0 .. 7 of the tile are the channels' gate rows, 8 .. 15
// their up rows. int8: x (XT) is quantised in LDS while the weights are on their way; 16 bits: it goes from memory
// into the B operand's first column.
template <class E, int XT>
__global__ void __launch_bounds__(64 * DMA_NW) dense_gate_up_kernel(DenseMoe p) {
    extern __shared__ __align__(16) uint8_t smem[];  // int8: the codes of x
    __shared__ uint32_t top[DMA_NW];
    __shared__ __align__(16) float red[DMA_NW * 16];  // [wave][gate / up][channel]
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, KB = H * E::ES, steps = (KB + MMB - 1) / MMB;
    const int a = blockIdx.y, t = a / k, jj = a % k, n0 = (int)blockIdx.x * 8;
    constexpr int XS = is_int8<E> ? (XT == TSA_F32 ? 4 : 2) : E::ES;
    const uint8_t* xrow = static_cast<const uint8_t*>(p.x) + (int64_t)t * H * XS;
    float xv[1][8];
    if constexpr (is_int8<E>) i8_row_load<XT, true, DMA_NW, 1>(xrow, H, tid, xv);
    const int64_t slot = dense_slot(p, a, t, jj, lane, wave);
    if (slot < 0 || slot >= p.n_slots) return;  // every wave of the workgroup: the pair's h is never read

    const uint8_t* base = p.pool + slot * L.slot_bytes;
    const __amdgpu_buffer_rsrc_t r = f8_buf(base, L.slot_bytes), rx = f8_buf(xrow, is_int8<E> ? 0 : KB);
    const uint32_t row = (uint32_t)((i >> 3) ? L.up_off : L.gate_off) + (uint32_t)(n0 + (i & 7)) * (uint32_t)KB;
    u32x4 A[DMA_D][2], Bv[DMA_D][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < DMA_D; ++d) {
            const int b = wave + DMA_NW * (j0 + d);
            if (b >= steps) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t o = (uint32_t)(MMB * b + 64 * h + 16 * q);
                if constexpr (!is_int8<E>) Bv[d][h] = f8_ld(rx, i == 0 ? f8_off(0, o, (uint32_t)KB) : 0x80000000u);
                A[d][h] = f8_ld(r, f8_off(row, o, (uint32_t)KB));
            }
        }
    };
    load(0);
    float sx = 1.0f;
    if constexpr (is_int8<E>) {
        sx = i8_row_codes<XT, true, DMA_NW, 1>(xrow, H, tid, xv, smem, top);
        __syncthreads();
    }
    typename E::acc acc = {0, 0, 0, 0};
    for (int j0 = 0; j0 < (steps + DMA_NW - 1) / DMA_NW; j0 += DMA_D) {
        if (j0) load(j0);
#pragma unroll
        for (int d = 0; d < DMA_D; ++d) {
            const int b = wave + DMA_NW * (j0 + d);
            if (b >= steps) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (is_int8<E>) {  // (past the row: weights that are zeros meet whatever lies there)
                    Bv[d][h] = u32x4{0, 0, 0, 0};
                    if (i == 0) Bv[d][h] = *reinterpret_cast<const u32x4*>(smem + MMB * b + 64 * h + 16 * q);
                }
                acc = E::mfma(A[d][h], Bv[d][h], acc);
            }
        }
    }
    if (i == 0) *reinterpret_cast<v4f*>(red + wave * 16 + 4 * q) = v4f{to_f32(acc[0]), to_f32(acc[1]), to_f32(acc[2]), to_f32(acc[3])};
    __syncthreads();
    if (tid < 8) {
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < DMA_NW; ++w) g += red[16 * w + tid], u += red[16 * w + 8 + tid];
        const int64_t at = (int64_t)a * I + n0 + tid;
        if constexpr (is_int8<E>) {
            const float* sg = reinterpret_cast<const float*>(base + L.gate_scales_off) + n0 + tid;
            static_cast<float*>(p.h)[at] = moe_act(L, g * (sx * sg[0]), u * (sx * sg[I]));
        } else {
            store_out(p.h, std::is_same<E, MmBf16>::value ? TSA_BF16 : TSA_F16, at, moe_act(L, g, u));
        }
    }
}

__device__ const uint32_t dense_zeros[4] = {0, 0, 0, 0};  // what lanes past a matrix read

// One workgroup per token and 8 outputs, over all the token's experts: rows 0 .. 7 of a tile are the outputs' rows of
// an even expert, 8 .. 15 those of the next, which meet columns 0 and 1 (their h); a unit is a step of 128 bytes of
// such a pair, and the waves take the units in turn. int8: the experts' h are quantised in LDS.
template <class E>
__global__ void __launch_bounds__(64 * DMD_NW) dense_down_kernel(DenseMoe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, KB = I * E::ES, G = (KB + MMB - 1) / MMB;
    const int t = blockIdx.y, n0 = (int)blockIdx.x * 8;
    __shared__ __align__(16) float red[DMD_NW * 16];
    __shared__ float hs[64];
    // lane j: the token's j-th slot (-1: none) and weight
    int my_slot = -1;
    float my_w = 0.0f;
    if (lane < k) {
        my_slot = p.slots[(int64_t)t * k + lane];
        my_w = p.wts[(int64_t)t * k + lane];
    }
    my_slot = my_slot < p.n_slots ? my_slot : -1;
    const uint8_t* hrows = static_cast<const uint8_t*>(p.h) + (int64_t)t * k * I * (is_int8<E> ? 4 : 2);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < k; c0 += p.chunk) {  // workgroup-uniform
        const int nc = k - c0 < p.chunk ? k - c0 : p.chunk, units = (nc + 1) / 2 * G;
        u32x4 A[DMD_D][2], Bv[DMD_D][2];
        v4f sc[DMD_D];
        auto load = [&](int u0) {
#pragma unroll
            for (int d = 0; d < DMD_D; ++d) {
                const int u = u0 + DMD_NW * d, pair = u / G, b = u % G;
                if (u >= units) break;
                const int ja = 2 * pair + (i >> 3), js = 2 * pair + (q >> 1), jb = 2 * pair + (i & 1);
                // every lane takes part in the shuffles: one that is off has 0 (a slot) read from it
                const int la = __shfl(my_slot, (c0 + ja) & 63, 64), ls = __shfl(my_slot, (c0 + js) & 63, 64);
                const int lb = __shfl(my_slot, (c0 + jb) & 63, 64);
                const float w = __shfl(my_w, (c0 + js) & 63, 64);
                const int sa = ja < nc ? la : -1, ss = js < nc ? ls : -1, sb = i < 2 && jb < nc ? lb : -1;
                const int o = MMB * b + 16 * q;
                const void* z = dense_zeros;
                if constexpr (!is_int8<E>) {
                    const uint8_t* hr = hrows + (int64_t)(c0 + jb) * KB + o;  // a dead expert's was never written
                    Bv[d][0] = *static_cast<const u32x4*>(sb >= 0 && o < KB ? hr : z);
                    Bv[d][1] = *static_cast<const u32x4*>(sb >= 0 && o + 64 < KB ? hr + 64 : z);
                    const float ws = ss >= 0 ? w : 0.0f;  // a dead expert's weight may be anything
                    sc[d] = v4f{ws, ws, ws, ws};
                } else {
                    const uint8_t* sp = p.pool + (int64_t)ss * L.slot_bytes + L.down_scales_off + 4 * (n0 + 4 * (q & 1));
                    const v4f ws = *static_cast<const v4f*>(ss >= 0 ? static_cast<const void*>(sp) : z);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[d][e] = ss >= 0 ? w * ws[e] : 0.0f;
                }
                const uint8_t* at = p.pool + (int64_t)sa * L.slot_bytes + L.down_off + (int64_t)(n0 + (i & 7)) * KB + o;
                A[d][0] = *static_cast<const u32x4*>(sa >= 0 && o < KB ? at : z);
                A[d][1] = *static_cast<const u32x4*>(sa >= 0 && o + 64 < KB ? at + 64 : z);
            }
        };
        load(wave);
        if constexpr (is_int8<E>) {
            if (c0) __syncthreads();  // the chunk before is used up
            for (int j = wave; j < nc; j += DMD_NW) {  // a wave an expert
                const int slot = __builtin_amdgcn_readlane(my_slot, c0 + j);
                uint8_t* codes = smem + j * G * MMB;
                if (slot < 0) {  // what is there is multiplied by weights of zero
                    for (int c = lane; c < G * MMB / 16; c += 64) *reinterpret_cast<u32x4*>(codes + 16 * c) = u32x4{0, 0, 0, 0};
                    if (lane == 0) hs[j] = 0.0f;
                    continue;
                }
                constexpr int D = 6;
                const uint8_t* hr = hrows + (int64_t)(c0 + j) * I * 4;
                float v[D][8];
                i8_row_load<TSA_F32, true, 1, D>(hr, I, lane, v);
                const float s = i8_row_codes<TSA_F32, true, 1, D>(hr, I, lane, v, codes, nullptr);
                if (lane == 0) hs[j] = s;
            }
            __syncthreads();
        }
        for (int u0 = wave; u0 < units; u0 += DMD_NW * DMD_D) {
            if (u0 != wave) load(u0);
#pragma unroll
            for (int d = 0; d < DMD_D; ++d) {
                const int u = u0 + DMD_NW * d;
                if (u >= units) break;
                v4f s = sc[d];
                if constexpr (is_int8<E>) {
                    const int pair = u / G, b = u % G, j = 2 * pair + i, js = 2 * pair + (q >> 1);
                    Bv[d][0] = Bv[d][1] = u32x4{0, 0, 0, 0};
                    if (i < 2 && j < nc) {
                        Bv[d][0] = *reinterpret_cast<const u32x4*>(smem + MMB * (j * G + b) + 16 * q);
                        Bv[d][1] = *reinterpret_cast<const u32x4*>(smem + MMB * (j * G + b) + 64 + 16 * q);
                    }
                    const float f = js < nc ? hs[js] : 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] = sc[d][e] * f;
                }
                typename E::acc part = {0, 0, 0, 0};
                part = E::mfma(A[d][0], Bv[d][0], part);
                part = E::mfma(A[d][1], Bv[d][1], part);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(s[e], to_f32(part[e]), acc[e]);
            }
        }
    }
    if (i == (q >> 1)) *reinterpret_cast<v4f*>(red + wave * 16 + 4 * q) = acc;  // an expert's rows in its own column
    __syncthreads();
    if (tid < 8) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < DMD_NW; ++w) v += red[16 * w + tid] + red[16 * w + 8 + tid];
        store_out(p.y, p.y_dtype, (int64_t)t * H + n0 + tid, v);
    }
}

// ---------------------------------------------------------------- many tokens
// Launches: the assignments grouped by expert with a table of token tiles (workgroup 0), x quantised (int8, the others);
// gate_up over the tiles, as many channels of gate as of up per workgroup; h quantised (int8); down, each assignment's
// output in float32 at the assignment's place; the weighted sums. (Outputs rounded to 16 bits ahead of the sums would add
// an error larger than the result's own rounding.)
struct DenseGroup {
    tsa_expert_layout L;
    const uint8_t* pool;
    int64_t n_slots;
    const int32_t* expert_slot;
    int64_t E;
    const int32_t* idx;
    int T, k;
    const void* x;
    int32_t *counts, *offsets, *perm;
    int* n_entries;
    int4* table;  // (slot, first sorted row, rows, -)
    int tile_rows;
    const uint8_t* xq;  // what gate_up multiplies: x itself, or its codes
    float* xs;
    void* h;  // [sorted row, I]: 16 bits, or float32
    const uint8_t* hq;  // what down multiplies: h itself, or its codes
    const float* hs;
    float* yk;  // [T k, H]
};

// Workgroup 0: the grouping; the others: 8 rows of x each, a wave a row (QUANT).
template <int XT, bool QUANT>
__global__ void __launch_bounds__(GROUP_THREADS) dense_prepare_kernel(DenseGroup p) {
    extern __shared__ __align__(16) unsigned char gsm[];
    if (blockIdx.x == 0) {
        const GroupTiles tiles{p.expert_slot, p.n_slots, p.tile_rows, p.n_entries, p.table};
        group_assignments<true>(p.idx, (int64_t)p.T * p.k, (int)p.E, p.counts, p.offsets, p.perm, tiles, GROUP_WAVES, gsm);
        return;
    }
    if constexpr (QUANT) {
        const int H = (int)p.L.hidden, lane = (int)threadIdx.x & 63, t = ((int)blockIdx.x - 1) * GROUP_WAVES + ((int)threadIdx.x >> 6);
        if (t >= p.T) return;
        constexpr int ES = XT == TSA_F32 ? 4 : 2, D = 6;
        const uint8_t* row = static_cast<const uint8_t*>(p.x) + (int64_t)t * H * ES;
        float v[D][8];
        i8_row_load<XT, true, 1, D>(row, H, lane, v);
        const float s = i8_row_codes<XT, true, 1, D>(row, H, lane, v, const_cast<uint8_t*>(p.xq) + (int64_t)t * H, nullptr);
        if (lane == 0) p.xs[t] = s;
    }
}

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) dense_group_gate_up_kernel(DenseGroup p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, KB = H * E::ES;
    constexpr int CH = C::RN / 2, MP = C::MR / 2;  // channels of a workgroup
    int entry, tile;
    if (!grouped_work(p.n_entries, (I + CH - 1) / CH, entry, tile)) return;
    const int4 e = p.table[entry];
    const int slot = uniform(e.x), row0 = uniform(e.y), tn = uniform(e.z), c0 = tile * CH;
    const uint8_t* base = p.pool + (int64_t)slot * L.slot_bytes;
    MmOperands<2> o;
    o.w[0] = base + L.gate_off + (int64_t)c0 * KB;
    o.w[1] = base + L.up_off + (int64_t)c0 * KB;
    o.w_rows = I - c0;
    o.x = p.xq;
    o.x_records = (uint32_t)p.T * (uint32_t)KB;
    o.KB = (uint32_t)KB;
    typename E::acc acc[C::MR][C::MT];
    auto token = [&](int r) { return p.perm[row0 + r] / p.k; };
    mm_tile<C, E, 2>(o, smem, tn, token, acc);

    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    v4f sg[MP], su[MP];
    if constexpr (is_int8<E>) {
        const float* s = reinterpret_cast<const float*>(base + L.gate_scales_off);
#pragma unroll
        for (int m = 0; m < MP; ++m) {
            const int c = c0 + (wr * MP + m) * 16 + 4 * q;
            sg[m] = *reinterpret_cast<const v4f*>(s + (c < I ? c : 0));
            su[m] = *reinterpret_cast<const v4f*>(s + I + (c < I ? c : 0));
        }
    }
#pragma unroll
    for (int t = 0; t < C::MT; ++t) {
        const int tk = 16 * (C::MT * wt + t) + i;
        if (tk >= tn) continue;
        float sx = 1.0f;
        if constexpr (is_int8<E>) sx = p.xs[token(tk)];
#pragma unroll
        for (int m = 0; m < MP; ++m) {
            const int c = c0 + (wr * MP + m) * 16 + 4 * q;  // I % 32 == 0: all four or none
            if (c >= I) continue;
            v4f h;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float g = to_f32(acc[m][t][r]), u = to_f32(acc[MP + m][t][r]);
                h[r] = is_int8<E> ? moe_act(L, g * (sx * sg[m][r]), u * (sx * su[m][r])) : moe_act(L, g, u);
            }
            const int64_t at = (int64_t)(row0 + tk) * I + c;
            if constexpr (is_int8<E>) {
                *reinterpret_cast<v4f*>(static_cast<float*>(p.h) + at) = h;
            } else {
                uint16_t* dst = static_cast<uint16_t*>(p.h) + at;
                if constexpr (std::is_same<E, MmBf16>::value)
                    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3]));
                else
                    *reinterpret_cast<uint2*>(dst) = make_uint2((uint32_t)f32_to_f16_bits(h[0]) | (uint32_t)f32_to_f16_bits(h[1]) << 16,
                                                                (uint32_t)f32_to_f16_bits(h[2]) | (uint32_t)f32_to_f16_bits(h[3]) << 16);
            }
        }
    }
}

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) dense_group_down_kernel(DenseGroup p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, KB = (int)L.inter * E::ES;
    int entry, tile;
    if (!grouped_work(p.n_entries, (H + C::RN - 1) / C::RN, entry, tile)) return;
    const int4 e = p.table[entry];
    const int slot = uniform(e.x), row0 = uniform(e.y), tn = uniform(e.z), n0 = tile * C::RN;
    const uint8_t* base = p.pool + (int64_t)slot * L.slot_bytes;
    MmOperands<1> o;
    o.w[0] = base + L.down_off + (int64_t)n0 * KB;
    o.w_rows = H - n0;
    o.x = p.hq + (int64_t)row0 * KB;
    o.x_records = (uint32_t)tn * (uint32_t)KB;
    o.KB = (uint32_t)KB;
    typename E::acc acc[C::MR][C::MT];
    mm_tile<C, E, 1>(o, smem, tn, [](int r) { return r; }, acc);
    const MmOut out = MmOut{p.yk, TSA_F32, H, nullptr, 0, 1};  // H % 32 == 0: rows of whole 16-byte pieces
    mm_store<C>(acc, out, n0, H, tn, [&](int r) { return (int64_t)p.perm[row0 + r]; }, [&](int r) { return p.hs[row0 + r]; },
                reinterpret_cast<const float*>(base + L.down_scales_off));
}

struct DensePlaces {
    int64_t counts, offsets, perm, n_entries, table, xq, xs, h, hq, hs, yk, bytes;
};

DensePlaces dense_places(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    const int64_t n = T * k, H = L.hidden, I = L.inter;
    const bool i8 = L.format == TSA_EXPERT_INT8;
    DensePlaces w;
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
    w.table = take((n / 16 + E) * 16);
    w.xq = take(i8 ? T * H : 0);
    w.xs = take(i8 ? T * 4 : 0);
    w.h = take(n * I * (i8 ? 4 : 2));
    w.hq = take(i8 ? n * I : 0);
    w.hs = take(i8 ? n * 4 : 0);
    w.yk = take(n * H * 4);
    w.bytes = at;
    return w;
}

// Tokens at a time: bounded workspace, and x (whose rows are picked by 32-bit offsets) of at most 2^31 bytes.
int64_t dense_tokens(const tsa_expert_layout& L, int64_t T, int k) {
    const int64_t c = group_tokens(T, k, MOE_ASSIGNMENTS), most = ((int64_t)1 << 31) / (2 * L.hidden);
    return c < most ? c : most;
}

template <class E, class GU, class DN>
int dense_gemms(const DenseGroup& p, int64_t entries, hipStream_t st) {
    DenseGroup q = p;
    void* args[] = {&q};
    const void* fg = reinterpret_cast<const void*>(&dense_group_gate_up_kernel<GU, E>);
    const void* fd = reinterpret_cast<const void*>(&dense_group_down_kernel<DN, E>);
    TSA_HIP_CHECK(ensure_dynamic_lds(fg, GU::LDS));
    TSA_HIP_CHECK(ensure_dynamic_lds(fd, DN::LDS));
    static_assert(GU::TM == DN::TM, "one table of token tiles");
    const int64_t tg = (p.L.inter + GU::RN / 2 - 1) / (GU::RN / 2), td = (p.L.hidden + DN::RN - 1) / DN::RN;
    auto grid = [](int64_t n) { return dim3((unsigned)((n + 7) / 8 * 8)); };  // whole rounds of XCDs
    TSA_HIP_CHECK(hipLaunchKernel(fg, grid(entries * tg), dim3(GU::THREADS), args, GU::LDS, st));
    if (is_int8<E>) {  // every sorted row, also those of experts that are not here (never read)
        const int rc = i8_quantize(p.h, TSA_F32, (int64_t)p.T * p.k, p.L.inter, const_cast<uint8_t*>(p.hq), const_cast<float*>(p.hs), st);
        if (rc) return rc;
    }
    TSA_HIP_CHECK(hipLaunchKernel(fd, grid(entries * td), dim3(DN::THREADS), args, DN::LDS, st));
    return TSA_OK;
}

using Up128 = MmTile<4, 2, 4, 4, 3>;   // 128 channels x 128 tokens, 8 waves
using Up64 = MmTile<4, 1, 2, 4, 3>;    // 64 x 64
using Up16 = MmTile<4, 1, 2, 1, 3>;    // 64 x 16
using Down128 = MmTile<4, 2, 4, 4, 3>; // 256 rows x 128 tokens
using Down64 = MmTile<4, 1, 2, 4, 3>;  // 128 x 64
using Down16 = MmTile<4, 1, 2, 1, 3>;  // 128 x 16

template <class E>
int dense_gemms(const DenseGroup& p, hipStream_t st) {
    const int64_t n = (int64_t)p.T * p.k, entries = n / p.tile_rows + (p.E < n ? p.E : n);
    switch (p.tile_rows) {
        case 16: return dense_gemms<E, Up16, Down16>(p, entries, st);
        case 64: return dense_gemms<E, Up64, Down64>(p, entries, st);
        default: return dense_gemms<E, Up128, Down128>(p, entries, st);
    }
}

}  // namespace

bool dense_format(const tsa_expert_layout& L) { return L.format == TSA_EXPERT_DENSE || L.format == TSA_EXPERT_INT8; }

// h [T k, I] fp32, then the routed selection.
int64_t dense_decode_ws_bytes(const tsa_expert_layout& L, int64_t T, int k) {
    return align256(T * k * L.inter * 4) + 2 * align256(T * k * 4);
}

// Calls whose routing runs inside the gate_up kernel.
bool dense_routes(int64_t T, int64_t E, int k) { return E <= 256 && k <= FUSED_MAXK && T * k <= 65535; }

// What a call needs beyond its layout.
static int check_dense(const tsa_expert_layout& L, const void* pool, const void* x, int x_dtype, const void* ws) {
    TSA_REQUIRE(((reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(ws)) & 15) == 0,
                TSA_ERR_INVALID_ARG, "16-bit and int8 experts: pool, x and workspace must be 16-byte aligned");
    TSA_REQUIRE(L.format == TSA_EXPERT_INT8 || x_dtype == L.gate_type, TSA_ERR_INVALID_ARG,
                "16-bit experts take activations of their own type (weights dtype %d, x %d)", L.gate_type, x_dtype);
    return TSA_OK;
}

int dense_decode(const tsa_expert_layout& L, const uint8_t* pool, int64_t n_slots, const int32_t* slots, const float* wts,
                 const void* logits, int logits_dtype, int mode, const int32_t* expert_slot, int64_t E, int32_t* idx_out,
                 float* w_out, int64_t T, int k, const void* x, int x_dtype, void* y, int y_dtype, uint8_t* ws,
                 int64_t ws_bytes, hipStream_t st) {
    TSA_REQUIRE(T >= 1 && T * k <= 65535 && (!logits || dense_routes(T, E, k)), TSA_ERR_SHAPE, "decode: T %lld, k %d, E %lld",
                (long long)T, k, (long long)E);
    TSA_REQUIRE(ws_bytes >= dense_decode_ws_bytes(L, T, k), TSA_ERR_WORKSPACE, "workspace too small for the decode");
    const int rc = check_dense(L, pool, x, x_dtype, ws);
    if (rc) return rc;
    const bool i8 = L.format == TSA_EXPERT_INT8;
    DenseMoe p{};
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
    p.h = ws;
    p.tab_slot = reinterpret_cast<int32_t*>(ws + align256(T * k * L.inter * 4));
    p.tab_w = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.tab_slot) + align256(T * k * 4));
    p.y = y;
    p.y_dtype = y_dtype;
    const int GH = (int)((L.hidden + MMB - 1) / MMB), GI = (int)((L.inter + MMB - 1) / MMB), row = GI * MMB;
    p.chunk = !i8 || k * row <= 60 * 1024 ? k : 60 * 1024 / row;  // at least 3 rows of 16384
    p.chunk = p.chunk < k ? p.chunk / 2 * 2 : p.chunk;            // whole pairs
    const int lds_a = i8 ? GH * MMB : 0, lds_b = i8 ? p.chunk * row : 0;
    const void* fa = !i8 ? (L.gate_type == TSA_BF16 ? reinterpret_cast<const void*>(&dense_gate_up_kernel<MmBf16, TSA_BF16>)
                                                    : reinterpret_cast<const void*>(&dense_gate_up_kernel<MmF16, TSA_F16>))
                     : x_dtype == TSA_F32 ? reinterpret_cast<const void*>(&dense_gate_up_kernel<MmI8, TSA_F32>)
                     : x_dtype == TSA_F16 ? reinterpret_cast<const void*>(&dense_gate_up_kernel<MmI8, TSA_F16>)
                                          : reinterpret_cast<const void*>(&dense_gate_up_kernel<MmI8, TSA_BF16>);
    void* args[] = {&p};
    TSA_HIP_CHECK(hipLaunchKernel(fa, dim3((unsigned)(L.inter / 8), (unsigned)(T * k)), dim3(64 * DMA_NW), args, lds_a, st));
    DenseMoe pb = p;  // the down launch reads the routed table, or the caller's
    if (logits) {
        pb.slots = p.tab_slot;
        pb.wts = p.tab_w;
    }
    void* args_b[] = {&pb};
    const void* fb = i8 ? reinterpret_cast<const void*>(&dense_down_kernel<MmI8>)
                     : L.gate_type == TSA_BF16 ? reinterpret_cast<const void*>(&dense_down_kernel<MmBf16>)
                                               : reinterpret_cast<const void*>(&dense_down_kernel<MmF16>);
    TSA_HIP_CHECK(hipLaunchKernel(fb, dim3((unsigned)(L.hidden / 8), (unsigned)T), dim3(64 * DMD_NW), args_b, lds_b, st));
    return TSA_OK;
}

// Calls that the grouped kernels take.
bool dense_group_supported(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    return dense_format(L) && T > DENSE_PAIR_TOKENS && E <= MAX_GROUP_E && k <= 64;
}

int64_t dense_group_workspace_bytes(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    return dense_places(L, dense_tokens(L, T, k), k, E).bytes;
}

int dense_group_prefill(const tsa_expert_layout& L, const uint8_t* pool, int64_t n_slots, const int32_t* expert_slot, int64_t E,
                        const int32_t* idx, const float* weights, int64_t T, int k, const void* x, int x_dtype, void* y,
                        int y_dtype, uint8_t* ws, hipStream_t st) {
    int rc = check_dense(L, pool, x, x_dtype, ws);
    if (rc) return rc;
    const bool i8 = L.format == TSA_EXPERT_INT8;
    const int64_t step = dense_tokens(L, T, k), H = L.hidden;
    const DensePlaces w = dense_places(L, step, k, E);
    const int lds = group_lds_bytes((int)E);
    const void* fp = !i8 ? reinterpret_cast<const void*>(&dense_prepare_kernel<TSA_BF16, false>)
                     : x_dtype == TSA_F32 ? reinterpret_cast<const void*>(&dense_prepare_kernel<TSA_F32, true>)
                     : x_dtype == TSA_F16 ? reinterpret_cast<const void*>(&dense_prepare_kernel<TSA_F16, true>)
                                          : reinterpret_cast<const void*>(&dense_prepare_kernel<TSA_BF16, true>);
    TSA_HIP_CHECK(ensure_dynamic_lds(fp, lds));
    for (int64_t t0 = 0; t0 < T; t0 += step) {
        DenseGroup p{};
        p.L = L;
        p.pool = pool;
        p.n_slots = n_slots;
        p.expert_slot = expert_slot;
        p.E = E;
        p.T = (int)(T - t0 < step ? T - t0 : step);
        p.k = k;
        p.idx = idx + t0 * k;
        p.x = static_cast<const uint8_t*>(x) + t0 * H * dtype_size(x_dtype);
        p.counts = reinterpret_cast<int32_t*>(ws + w.counts);
        p.offsets = reinterpret_cast<int32_t*>(ws + w.offsets);
        p.perm = reinterpret_cast<int32_t*>(ws + w.perm);
        p.n_entries = reinterpret_cast<int*>(ws + w.n_entries);
        p.table = reinterpret_cast<int4*>(ws + w.table);
        p.xq = i8 ? ws + w.xq : static_cast<const uint8_t*>(p.x);
        p.xs = reinterpret_cast<float*>(ws + w.xs);
        p.h = ws + w.h;
        p.hq = ws + (i8 ? w.hq : w.h);
        p.hs = reinterpret_cast<float*>(ws + w.hs);
        p.yk = reinterpret_cast<float*>(ws + w.yk);
        const int64_t n = (int64_t)p.T * k;
        p.tile_rows = n <= 12 * E ? 16 : n <= 48 * E ? 64 : 128;
        void* args[] = {&p};
        const unsigned wgs = i8 ? (unsigned)(1 + (p.T + GROUP_WAVES - 1) / GROUP_WAVES) : 1u;
        TSA_HIP_CHECK(hipLaunchKernel(fp, dim3(wgs), dim3(GROUP_THREADS), args, lds, st));
        rc = i8 ? dense_gemms<MmI8>(p, st) : L.gate_type == TSA_BF16 ? dense_gemms<MmBf16>(p, st) : dense_gemms<MmF16>(p, st);
        if (rc) return rc;
        rc = launch_combine(MoeCombine{p.idx, weights + t0 * k, expert_slot, E, n_slots, p.T, k, (int)H, p.yk,
                                       static_cast<uint8_t*>(y) + t0 * H * dtype_size(y_dtype), y_dtype}, st);
        if (rc) return rc;
    }
    return TSA_OK;
}

// Requirements beyond the common ones of validate_layout, with the status they fail with.
int dense_validate(const tsa_expert_layout& L) {
    const bool i8 = L.format == TSA_EXPERT_INT8;
    TSA_REQUIRE(i8 || ((L.gate_type == TSA_BF16 || L.gate_type == TSA_F16) && L.up_type == L.gate_type && L.down_type == L.gate_type),
                TSA_ERR_INVALID_ARG, "16-bit experts: gate, up and down must all be bfloat16 or all float16 (got dtypes %d, %d, %d)",
                L.gate_type, L.up_type, L.down_type);
    TSA_REQUIRE(L.gate_bias_off < 0 && L.down_bias_off < 0, TSA_ERR_INVALID_ARG, "16-bit and int8 experts carry no biases");
    const int64_t H = L.hidden, I = L.inter, m = H * I * (i8 ? 1 : 2);
    const int64_t need[5][2] = {{L.gate_off, m}, {L.up_off, m}, {L.down_off, m}, {L.gate_scales_off, 8 * I}, {L.down_scales_off, 4 * H}};
    for (int j = 0; j < (i8 ? 5 : 3); ++j) {
        TSA_REQUIRE(need[j][0] >= 0 && need[j][0] + need[j][1] <= L.slot_bytes, TSA_ERR_WEIGHT_TOO_SMALL,
                    "tensor at offset %lld (%lld bytes) exceeds slot_bytes %lld", (long long)need[j][0], (long long)need[j][1],
                    (long long)L.slot_bytes);
        TSA_REQUIRE(need[j][0] % 16 == 0, TSA_ERR_INVALID_ARG, "16-bit and int8 experts: tensors must start on multiples of 16 bytes");
    }
    TSA_REQUIRE(L.slot_bytes % 16 == 0 && L.slot_bytes < ((int64_t)1 << 31), TSA_ERR_INVALID_ARG,
                "16-bit and int8 experts: slots must be a multiple of 16 bytes, below 2^31");
    return TSA_OK;
}

}  // namespace tsa
