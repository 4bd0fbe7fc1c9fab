// MoE layers over experts in bfloat16, float16 or int8 (a float32 scale for each row).
//
// Definition, per token: for each selected expert h = act(Wg x, Wu x) in float32; 16 bits: h rounded to the weights'
// type, which x has too; int8: x and h quantised per token (int8_common.h); y = sum_j w_j Wd h in float32, rounded
// once.
//
// Few tokens: two launches ordered by the stream. gate_up: one workgroup per (token, expert) pair and 8 channels; down:
// one per token and 4 outputs, over all the token's experts, so every output has one writer. Each is a stream of
// weights into the A operands of matrix instructions (one or two columns of B in use).
#include "int8_common.h"
#include "mm_epilogue.h"
#include "moe_grouped.h"

namespace tsa {
int i8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st);

namespace {

template <class E>
constexpr bool is_int8 = std::is_same<E, MmI8>::value;

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
constexpr int DMD_NW = 8;             // down
template <class E>
constexpr int dmd_d = is_int8<E> ? 2 : 3;  // (one more: spills, and down takes 2 to 3 times as long)

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
    constexpr int XR = is_int8<E> ? XT : TSA_BF16;
    I8Raw<XR> xv[1];
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

// One workgroup per token and 4 outputs, over all the token's experts: rows 4 e .. 4 e + 3 of a tile are the outputs' rows
// of the e-th of four experts, which meet column e (its h); a unit is a step of 128 bytes of such four, and the waves take
// the units in turn. (Against two experts and 8 outputs, half as many workgroups: 180 us for 189, 8 layers of
// hidden 2048, 128 experts top-8, bf16, one token.) int8: the experts' h are quantised in LDS.
template <class E>
__global__ void __launch_bounds__(64 * DMD_NW, 4) dense_down_kernel(DenseMoe p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const tsa_expert_layout& L = p.L;
    const int H = (int)L.hidden, I = (int)L.inter, k = p.k, KB = I * E::ES, G = (KB + MMB - 1) / MMB;
    const int t = blockIdx.y, n0 = (int)blockIdx.x * 4;
    constexpr int D = dmd_d<E>;
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
    my_w = my_slot >= 0 ? my_w : 0.0f;  // the weight of an expert that is not here may be anything
    const uint8_t* hrows = static_cast<const uint8_t*>(p.h) + (int64_t)t * k * I * (is_int8<E> ? 4 : 2);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < k; c0 += p.chunk) {  // workgroup-uniform
        const int nc = k - c0 < p.chunk ? k - c0 : p.chunk, units = (nc + 3) / 4 * G;
        u32x4 A[D][2], Bv[D][2];
        v4f ws[D];
        float sc[D];
        auto load = [&](int u0) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int u = u0 + DMD_NW * d, four = u / G, b = u - four * G;
                if (u >= units) break;
                const int ja = 4 * four + (i >> 2), js = 4 * four + q, jb = 4 * four + (i & 3);  // of the lane's row of A, its sums, its column
                // every lane takes part in the shuffles: one that is off has 0 (a slot) read from it
                const int la = __shfl(my_slot, (c0 + ja) & 63, 64), ls = __shfl(my_slot, (c0 + js) & 63, 64);
                const float w = __shfl(my_w, (c0 + js) & 63, 64);
                const int sa = ja < nc ? la : -1, ss = js < nc ? ls : -1;
                const int o = MMB * b + 16 * q;
                const void* z = dense_zeros;
                sc[d] = js < nc ? w : 0.0f;
                if constexpr (!is_int8<E>) {
                    const int lb = __shfl(my_slot, (c0 + jb) & 63, 64);
                    const bool live = i < 4 && jb < nc && lb >= 0;  // the h of an expert that is not here was never written
                    const uint8_t* hr = hrows + (int64_t)(c0 + jb) * KB + o;
                    Bv[d][0] = *static_cast<const u32x4*>(live && o < KB ? hr : z);
                    Bv[d][1] = *static_cast<const u32x4*>(live && o + 64 < KB ? hr + 64 : z);
                } else {
                    const uint8_t* sp = p.pool + (int64_t)ss * L.slot_bytes + L.down_scales_off + 4 * n0;
                    ws[d] = *static_cast<const v4f*>(ss >= 0 ? static_cast<const void*>(sp) : z);
                }
                const uint8_t* at = p.pool + (int64_t)sa * L.slot_bytes + L.down_off + (int64_t)(n0 + (i & 3)) * KB + o;
                A[d][0] = *static_cast<const u32x4*>(sa >= 0 && o < KB ? at : z);
                A[d][1] = *static_cast<const u32x4*>(sa >= 0 && o + 64 < KB ? at + 64 : z);
            }
        };
        if constexpr (is_int8<E>) {
            // a wave an expert: the first one's values are loaded ahead of the weights. (Codes of an expert that is not
            // here meet weights of zero.)
            constexpr int HELD = 2;
            auto live = [&](int j) { return j < nc && __builtin_amdgcn_readlane(my_slot, (c0 + j) & 63) >= 0; };
            const int mine = __shfl(my_slot, (c0 + lane) & 63, 64);  // lane j's: the chunk's j-th
            const uint8_t* hr = hrows + (int64_t)(c0 + wave) * I * 4;
            const bool first = live(wave);
            I8Raw<TSA_F32> v[HELD];
            i8_row_load<TSA_F32, true, 1, HELD>(hr, first ? I : 0, lane, v);
            load(wave);
            if (c0) __syncthreads();  // the chunk before is used up
            if (first) {
                const float s = i8_row_codes<TSA_F32, true, 1, HELD>(hr, I, lane, v, smem + wave * G * MMB, nullptr);
                if (lane == 0) hs[wave] = s;
            }
            for (int j = wave + DMD_NW; j < nc; j += DMD_NW) {
                if (!live(j)) continue;
                const uint8_t* row = hrows + (int64_t)(c0 + j) * I * 4;
                i8_row_load<TSA_F32, true, 1, HELD>(row, I, lane, v);
                const float s = i8_row_codes<TSA_F32, true, 1, HELD>(row, I, lane, v, smem + j * G * MMB, nullptr);
                if (lane == 0) hs[j] = s;
            }
            if (wave == 0 && lane < nc && mine < 0) hs[lane] = 0.0f;
            __syncthreads();
        } else {
            load(wave);
        }
        for (int u0 = wave; u0 < units; u0 += DMD_NW * D) {
            if (u0 != wave) load(u0);
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int u = u0 + DMD_NW * d;
                if (u >= units) break;
                v4f s = {sc[d], sc[d], sc[d], sc[d]};
                if constexpr (is_int8<E>) {
                    const int four = u / G, b = u - four * G, j = 4 * four + i, js = 4 * four + q;
                    Bv[d][0] = Bv[d][1] = u32x4{0, 0, 0, 0};
                    if (i < 4 && j < nc) {
                        Bv[d][0] = *reinterpret_cast<const u32x4*>(smem + MMB * (j * G + b) + 16 * q);
                        Bv[d][1] = *reinterpret_cast<const u32x4*>(smem + MMB * (j * G + b) + 64 + 16 * q);
                    }
                    const float f = js < nc ? sc[d] * hs[js] : 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] = f * ws[d][e];
                }
                typename E::acc part = {0, 0, 0, 0};
                part = E::mfma(A[d][0], Bv[d][0], part);
                part = E::mfma(A[d][1], Bv[d][1], part);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(s[e], to_f32(part[e]), acc[e]);
            }
        }
    }
    if (i == q) *reinterpret_cast<v4f*>(red + wave * 16 + 4 * q) = acc;  // an expert's rows in its own column
    __syncthreads();
    if (tid < 4) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < DMD_NW * 4; ++w) v += red[4 * w + tid];
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
        I8Raw<XT> v[D];
        i8_row_load<XT, true, 1, D>(row, H, lane, v);
        const float s = i8_row_codes<XT, true, 1, D>(row, H, lane, v, const_cast<uint8_t*>(p.xq) + (int64_t)t * H, nullptr);
        if (lane == 0) p.xs[t] = s;
    }
}

// A workgroup's tiles (mm_pair's order) of the table's entries.
template <class C>
struct DenseWork {
    const DenseGroup& p;
    const int entries, tiles;  // row tiles of an entry
    MmRuns runs;
    int slot, row0, tn, tile, next_slot, next_row0, next_tn, next_tile;
    __device__ __forceinline__ DenseWork(const DenseGroup& p, int tiles) : p(p), entries(uniform(*p.n_entries)), tiles(tiles), runs(entries * tiles) {}
    __device__ __forceinline__ bool next() {
        if (!runs.next()) return false;
        int entry;
        mm_pair(runs.at, entries, tiles, entry, next_tile);
        const int4 e = p.table[entry];
        next_slot = uniform(e.x), next_row0 = uniform(e.y), next_tn = uniform(e.z);
        return true;
    }
    __device__ __forceinline__ void take() { slot = next_slot, row0 = next_row0, tn = next_tn, tile = next_tile; }
};

template <class C, class E>
struct DenseUp : DenseWork<C> {
    using B = DenseWork<C>;
    static constexpr int CH = C::RN / 2, MP = C::MR / 2, MT = C::MT;  // channels of a tile
    __device__ __forceinline__ explicit DenseUp(const DenseGroup& p) : B(p, ((int)p.L.inter + CH - 1) / CH) {}
    __device__ __forceinline__ int picked(int row) const { return B::p.perm[row] / B::p.k; }
    __device__ __forceinline__ int token(int r) const { return picked(B::next_row0 + r); }
    __device__ __forceinline__ MmOperands<2> operands() const {
        const tsa_expert_layout& L = B::p.L;
        const int KB = (int)L.hidden * E::ES, c0 = B::next_tile * CH;
        const uint8_t* base = B::p.pool + (int64_t)B::next_slot * L.slot_bytes;
        return MmOperands<2>{{base + L.gate_off + (int64_t)c0 * KB, base + L.up_off + (int64_t)c0 * KB}, (int)L.inter - c0, B::p.xq,
                             (uint32_t)B::p.T * (uint32_t)KB, B::next_tn};
    }
    __device__ __forceinline__ void store(const typename E::acc (&acc)[C::MR][MT], uint8_t* out) const {
        const DenseGroup& p = B::p;
        const tsa_expert_layout& L = p.L;
        const int I = (int)L.inter, lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
        const int t0 = wave / C::WR * MT * 16, cw = B::tile * CH + wave % C::WR * MP * 16;
        v4f sg[MP], su[MP];
        float sx[MT];
        if constexpr (is_int8<E>) {
            const float* s = reinterpret_cast<const float*>(p.pool + (int64_t)B::slot * L.slot_bytes + L.gate_scales_off);
#pragma unroll
            for (int m = 0; m < MP; ++m) {  // I % 32 == 0: all four or none
                const int c = cw + 16 * m + 4 * q;
                sg[m] = *reinterpret_cast<const v4f*>(s + (c < I ? c : 0));
                su[m] = *reinterpret_cast<const v4f*>(s + I + (c < I ? c : 0));
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) sx[t] = t0 + 16 * t + i < B::tn ? p.xs[picked(B::row0 + t0 + 16 * t + i)] : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (t0 + 16 * t >= B::tn) continue;  // uniform
            v4f h[MP];
#pragma unroll
            for (int m = 0; m < MP; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float g = to_f32(acc[m][t][r]), u = to_f32(acc[MP + m][t][r]);
                    h[m][r] = is_int8<E> ? moe_act(L, g * (sx[t] * sg[m][r]), u * (sx[t] * su[m][r])) : moe_act(L, g, u);
                }
            if constexpr (is_int8<E>) {
                const int tk = t0 + 16 * t + i;
                float* dst = static_cast<float*>(p.h) + (int64_t)(B::row0 + tk) * I;
#pragma unroll
                for (int m = 0; m < MP; ++m) {
                    const int c = cw + 16 * m + 4 * q;
                    if (tk < B::tn && c < I) *reinterpret_cast<v4f*>(dst + c) = h[m];
                }
            } else {
                uint2 v[MP];
#pragma unroll
                for (int m = 0; m < MP; ++m) v[m] = mm_pack4<std::is_same<E, MmBf16>::value ? TSA_BF16 : TSA_F16>(h[m]);
                mm_rows16<MP>(v, out, [&](int r, int c) -> void* {
                    const int tk = t0 + 16 * t + r, n = cw + 8 * c;
                    return tk < B::tn && n < I ? static_cast<uint16_t*>(p.h) + (int64_t)(B::row0 + tk) * I + n : nullptr;
                });
            }
        }
    }
};

template <class C, class E>
struct DenseDown : DenseWork<C> {
    using B = DenseWork<C>;
    __device__ __forceinline__ explicit DenseDown(const DenseGroup& p) : B(p, ((int)p.L.hidden + C::RN - 1) / C::RN) {}
    __device__ __forceinline__ int token(int r) const { return r; }
    __device__ __forceinline__ MmOperands<1> operands() const {
        const tsa_expert_layout& L = B::p.L;
        const int KB = (int)L.inter * E::ES, n0 = B::next_tile * C::RN;
        return MmOperands<1>{{B::p.pool + (int64_t)B::next_slot * L.slot_bytes + L.down_off + (int64_t)n0 * KB}, (int)L.hidden - n0,
                             B::p.hq + (int64_t)B::next_row0 * KB, (uint32_t)B::next_tn * (uint32_t)KB, B::next_tn};
    }
    __device__ __forceinline__ void store(const typename E::acc (&acc)[C::MR][C::MT], uint8_t* out) const {
        const DenseGroup& p = B::p;
        const int H = (int)p.L.hidden;
        const MmOut o = MmOut{p.yk, TSA_F32, H, nullptr, 0, 1};  // H % 32 == 0: rows of whole 16-byte pieces
        mm_store<C>(acc, o, out, B::tile * C::RN, H, B::tn, [&](int r) { return (int64_t)p.perm[B::row0 + r]; },
                           [&](int r) { return p.hs[B::row0 + r]; },
                           reinterpret_cast<const float*>(p.pool + (int64_t)B::slot * p.L.slot_bytes + p.L.down_scales_off));
    }
};

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) dense_group_gate_up_kernel(DenseGroup p) {
    extern __shared__ __align__(16) uint8_t smem[];
    DenseUp<C, E> work(p);
    mm_run<C, E, 2, true>(work, (uint32_t)p.L.hidden * E::ES, smem);
}

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) dense_group_down_kernel(DenseGroup p) {
    extern __shared__ __align__(16) uint8_t smem[];
    DenseDown<C, E> work(p);
    mm_run<C, E, 1, false>(work, (uint32_t)p.L.inter * E::ES, smem);
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
    w.table = take((n / 64 + E) * 16);
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
int dense_gemms(const DenseGroup& p, int64_t entries, int per, hipStream_t st) {
    DenseGroup q = p;
    void* args[] = {&q};
    const void* fg = reinterpret_cast<const void*>(&dense_group_gate_up_kernel<GU, E>);
    const void* fd = reinterpret_cast<const void*>(&dense_group_down_kernel<DN, E>);
    TSA_HIP_CHECK(ensure_dynamic_lds(fg, GU::LDS));
    TSA_HIP_CHECK(ensure_dynamic_lds(fd, DN::LDS));
    static_assert(GU::TM == DN::TM, "one table of token tiles");
    const int64_t tg = (p.L.inter + GU::RN / 2 - 1) / (GU::RN / 2), td = (p.L.hidden + DN::RN - 1) / DN::RN;
    TSA_HIP_CHECK(hipLaunchKernel(fg, dim3(mm_grid(entries * tg, per)), dim3(GU::THREADS), args, GU::LDS, st));
    if (is_int8<E>) {  // every sorted row, also those of experts that are not here (never read)
        const int rc = i8_quantize(p.h, TSA_F32, (int64_t)p.T * p.k, p.L.inter, const_cast<uint8_t*>(p.hq), const_cast<float*>(p.hs), st);
        if (rc) return rc;
    }
    TSA_HIP_CHECK(hipLaunchKernel(fd, dim3(mm_grid(entries * td, per)), dim3(DN::THREADS), args, DN::LDS, st));
    return TSA_OK;
}

using Up128 = MmTile<4, 2, 4, 4, 3>;   // 128 channels x 128 tokens, 8 waves
using Up64 = MmTile<4, 1, 2, 4, 3>;    // 64 x 64
using Down128 = MmTile<4, 2, 4, 4, 3>; // 256 rows x 128 tokens
using Down64 = MmTile<4, 1, 2, 4, 3>;  // 128 x 64

template <class E>
int dense_gemms(const DenseGroup& p, hipStream_t st) {
    const int64_t n = (int64_t)p.T * p.k, entries = n / p.tile_rows + (p.E < n ? p.E : n);
    return p.tile_rows == 64 ? dense_gemms<E, Up64, Down64>(p, entries, 2, st) : dense_gemms<E, Up128, Down128>(p, entries, 1, st);
}

}  // namespace

bool dense_format(const tsa_expert_layout& L) { return L.format == TSA_EXPERT_DENSE || L.format == TSA_EXPERT_INT8; }

// Tokens up to which a call runs as pairs: two, and more while they are few and their experts' weights, read once for each
// pair, few bytes; the grouped kernels read each expert once, in five or six launches. us of a layer grouped / as pairs, without the
// routing: hidden 2048, 128 experts top-8, 2 / 3 / 4 / 8 tokens, bf16 (9.4 MB an expert) 39 / 43 / 47 / 56 and 34 / 46 / 58 / 105, int8 33 /
// 35 / 38 / 44 and 24 / 32 / 40 / 72; hidden 2880, 32 experts top-4, 2 / 3 / 4 tokens, bf16 (50 MB) 82 / 87 / 91 and 74 / 102 / 130, int8 62 /
// 62 / 65 and 57 / 76 / 96; hidden 1440, 20 experts top-3, int8 (3.2 MB), 6 / 8 tokens 28 / 28 and 27 / 33; hidden 1024, 16 experts top-2, bf16
// (3.1 MB), 12 / 16 tokens 26 / 26 and 27 / 34; hidden 256, 64 experts top-4 (0.25 MB), 16 / 24 tokens 18 / 18 and 12 / 15. (T k stops at
// 64 all the same, where experts as small as the last would gain 3 us more.)
int64_t dense_pair_tokens(const tsa_expert_layout& L, int k) {
    const int64_t expert = 3 * L.hidden * L.inter * (L.format == TSA_EXPERT_INT8 ? 1 : 2), bytes = ((int64_t)72 << 20) / (k * expert), few = 64 / k;
    const int64_t most = bytes < few ? bytes : few;
    return most > 2 ? most : 2;
}

// Pairs: h [T k, I] fp32, then the routed selection. Routed calls of more tokens: the selection, then what the grouped
// kernels need (for any number of experts).
int64_t dense_decode_ws_bytes(const tsa_expert_layout& L, int64_t T, int k) {
    const int64_t pairs = align256(T * k * L.inter * 4), table = 2 * align256(T * k * 4);
    const int64_t grouped = T > dense_pair_tokens(L, k) ? dense_places(L, dense_tokens(L, T, k), k, MAX_GROUP_E).bytes : 0;
    return table + (pairs > grouped ? pairs : grouped);
}

// Calls whose routing runs inside the gate_up kernel.
bool dense_routes(int64_t T, int64_t E, int k) { return E <= 256 && k <= FUSED_MAXK && T * k <= 65535; }

// What a call needs beyond its layout.
int check_dense(const tsa_expert_layout& L, const void* pool, const void* x, int x_dtype, const void* ws) {
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
    p.chunk = p.chunk < k && p.chunk >= 4 ? p.chunk / 4 * 4 : p.chunk;  // whole fours
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
    TSA_HIP_CHECK(hipLaunchKernel(fb, dim3((unsigned)(L.hidden / 4), (unsigned)T), dim3(64 * DMD_NW), args_b, lds_b, st));
    return TSA_OK;
}

// Calls that the grouped kernels take.
bool dense_group_supported(const tsa_expert_layout& L, int64_t T, int k, int64_t E) {
    return dense_format(L) && T > dense_pair_tokens(L, k) && E <= MAX_GROUP_E && k <= 64;
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
        // us of a layer in tiles of 64 / 128 tokens, hidden 2048, 128 experts top-8, 24 / 200 / 700 / 1024 / 2048 tokens:
        // bf16 82 / 151 / 238 / 286 / 426 and 88 / 158 / 239 / 273 / 376, int8 56 / 97 / 158 / 190 / 288 and 61 / 103 / 159 /
        // 188 / 265; hidden 2880, 32 experts top-4, 100 / 200 / 400 / 2048 tokens: bf16 270 / 311 / 355 / 760 and 291 / 322 /
        // 342 / 600, int8 170 / 207 / 244 / 541 and 188 / 216 / 237 / 435. (Tiles of 16: bf16 2 to 5% faster for 24 and 48
        // tokens over 128 experts, else slower.)
        p.tile_rows = n <= 48 * E ? 64 : 128;
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

// Routed calls of more tokens than the pairs take: top-k, then as a prompt.
int dense_routed_batch(const tsa_expert_layout& L, const uint8_t* pool, int64_t n_slots, const void* logits, int logits_dtype, int mode,
                       const int32_t* expert_slot, int64_t E, int32_t* idx_out, float* w_out, int64_t T, int k, const void* x, int x_dtype,
                       void* y, int y_dtype, uint8_t* ws, int64_t ws_bytes, hipStream_t st) {
    TSA_REQUIRE(ws_bytes >= dense_decode_ws_bytes(L, T, k), TSA_ERR_WORKSPACE, "workspace too small for the decode");
    int rc = check_dense(L, pool, x, x_dtype, ws);
    if (rc) return rc;
    int32_t* idx = idx_out ? idx_out : reinterpret_cast<int32_t*>(ws);
    float* w = w_out ? w_out : reinterpret_cast<float*>(ws + align256(T * k * 4));
    rc = tsa_route_topk(logits, logits_dtype, T, E, k, mode, idx, w, st);
    if (rc) return rc;
    return dense_group_prefill(L, pool, n_slots, expert_slot, E, idx, w, T, k, x, x_dtype, y, y_dtype, ws + 2 * align256(T * k * 4), st);
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
