// The tile of the products of int8 and 16-bit matrices over many tokens: RN weight rows x TM tokens of a
// workgroup of WR x WT waves, each MR x MT tiles of 16 x 16.
//
// y[n, t] = sum_k w[n, k] x[t, k], on v_mfma_i32_16x16x64_i8 or v_mfma_f32_16x16x32_{bf16,f16}: all of
// them take 16 bytes a lane of either operand, so the tile counts in bytes. Lane 16 q + i holds bytes 16 q ..
// of row i of A (weights) and of column i of B (tokens); the result's lane 16 q + i holds rows 4 q .. 4 q + 3
// of column i.
//
// K advances 128 bytes at a time, two products deep. A step's rows (weights, then tokens) come into one of S
// stages in LDS by buffer-to-LDS copies; rows and columns past the matrices are offsets past the buffers,
// which copy zeros. The 16-byte chunk c of row r sits in slot c ^ (r / 2 % 8): the 16 rows that a quarter wave
// reads at once then fall on distinct banks. The barrier sits between a step's two products: by then the
// second half's operands are in registers, so the stage is free for the copies of step s + S, which go out
// among the second half's products, as do the LDS reads of step s + 1.
#pragma once

#include "lds_copy.h"
#include "mfma_tile.h"

namespace tsa {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// An element type: its matrix instruction on 16 bytes a lane. Sums of int8 products are exact (int32), those
// of 16-bit ones are held in float32.
struct MmI8 {
    typedef v4i acc;
    static constexpr int ES = 1;
    static __device__ __forceinline__ acc mfma(const u32x4& a, const u32x4& b, const acc& c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, a), __builtin_bit_cast(v4i, b), c, 0, 0, 0);
    }
};
struct MmBf16 {
    typedef v4f acc;
    static constexpr int ES = 2;
    static __device__ __forceinline__ acc mfma(const u32x4& a, const u32x4& b, const acc& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct MmF16 {
    typedef v4f acc;
    static constexpr int ES = 2;
    static __device__ __forceinline__ acc mfma(const u32x4& a, const u32x4& b, const acc& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

constexpr int MMB = 128;  // bytes of a row per step

// WR x WT waves of MR x MT tiles of 16 x 16, S stages.
template <int WR_, int WT_, int MR_, int MT_, int S_>
struct MmTile {
    static constexpr int WR = WR_, WT = WT_, MR = MR_, MT = MT_, S = S_;
    static constexpr int NW = WR * WT, THREADS = 64 * NW, RN = 16 * WR * MR, TM = 16 * WT * MT;
    static constexpr int NXW = RN / 8 / NW, NXT = (TM + 8 * NW - 1) / (8 * NW);  // copies of 8 rows, a wave's
    static constexpr int PER = NXW + NXT;                                        // those of a step
    static constexpr int STAGE = (RN + 8 * NW * NXT) * MMB, LDS = S * STAGE;
    static_assert(RN % (8 * NW) == 0 && (S - 1) * PER < 63 && S >= 2, "tile");
};

// What a tile multiplies. Weight row r of the tile (r < RN) is row r of w[r / (RN / PARTS)] counted
// from that part's first row, w_rows of them (PARTS 2: the gate and the up rows of an expert).
template <int PARTS>
struct MmOperands {
    const uint8_t* w[PARTS];  // first row of the tile
    int w_rows;               // rows there are from it on (those past RN / PARTS are not read)
    const uint8_t* x;
    uint32_t x_records;       // its bytes, below 2^31
    uint32_t KB;              // bytes of a row of either, a multiple of 16
};

// acc[m][t]: rows 4 q .. 4 q + 3 of tile m, token 16 t + i, for lane 16 q + i of the wave. Tile m is
// the wave's m-th: of its MR, the first MR / PARTS belong to part 0. `token(r)`: row of x of the
// tile's token r, -1 from `tokens` on (and for a row of zeros).
template <class C, class E, int PARTS, class Token>
__device__ __forceinline__ void mm_tile(const MmOperands<PARTS>& p, uint8_t* smem, int tokens, Token token,
                                        typename E::acc (&acc)[C::MR][C::MT]) {
    constexpr int MR = C::MR, MT = C::MT, S = C::S, HALF = C::RN / PARTS, MP = MR / PARTS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    const uint32_t KB = p.KB, lds0 = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int steps = (int)((KB + MMB - 1) / MMB);

    // copy j of this wave fills rows 8 (NX wave + j) + lane / 8, slot lane % 8
    buf_v4i rw[PARTS];
#pragma unroll
    for (int h = 0; h < PARTS; ++h) rw[h] = buf_desc(p.w[h], (uint32_t)(p.w_rows < HALF ? p.w_rows : HALF) * KB);
    const buf_v4i rx = buf_desc(p.x, p.x_records);
    uint32_t wo[C::NXW], xo[C::NXT];
    auto chunk = [&](int n) { return (uint32_t)((lane & 7) ^ ((4 * n + (lane >> 4)) & 7)); };  // of copy n's rows
#pragma unroll
    for (int j = 0; j < C::NXW; ++j) {
        const int n = C::NXW * wave + j;
        wo[j] = (uint32_t)(8 * n + (lane >> 3)) % HALF * KB + 16u * chunk(n);
    }
#pragma unroll
    for (int j = 0; j < C::NXT; ++j) {
        const int n = C::NXT * wave + j, r = 8 * n + (lane >> 3), row = r < tokens ? token(r) : -1;
        xo[j] = row < 0 ? 0x80000000u : (uint32_t)row * KB + 16u * chunk(n);
    }
    uint32_t at[2];  // this lane's column in copies of even and odd number
#pragma unroll
    for (int n = 0; n < 2; ++n) at[n] = 16u * chunk(n);
    // copy j (of PER) of step s. Columns past K and steps past the last read zeros, so every step issues as
    // many. (The scalar offset stays inside the buffers: the range check may subtract it from their size.)
    auto issue = [&](int j, int s, int stage) {
        const uint32_t col = (uint32_t)MMB * (uint32_t)s, base = lds0 + (uint32_t)stage * C::STAGE;
        const uint32_t soff = s < steps ? col : 0u;
        const int n = j < C::NXW ? C::NXW * wave + j : C::NXT * wave + j - C::NXW;
        const bool in = col + (n & 1 ? at[1] : at[0]) < KB;
        if (j < C::NXW) lds_copy16(rw[PARTS == 1 ? 0 : 8 * n / HALF], in ? wo[j] : 0x80000000u, soff, base + 1024u * (uint32_t)n);
        else lds_copy16(rx, in ? xo[j - C::NXW] : 0x80000000u, soff, base + (uint32_t)C::RN * MMB + 1024u * (uint32_t)n);
    };

#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[m][t] = typename E::acc{0, 0, 0, 0};

    const int frag = i * MMB + 16 * (q ^ (i >> 1));  // chunk q of row i of a tile; chunk q + 4 is 64 off by xor
    auto read_a = [&](const uint8_t* wl, int m, int h) {
        return *reinterpret_cast<const u32x4*>(wl + (m / MP * HALF + (wr * MP + m % MP) * 16) * MMB + (frag ^ (64 * h)));
    };
    auto read_b = [&](const uint8_t* wl, int t, int h) {
        return *reinterpret_cast<const u32x4*>(wl + (C::RN + (wt * MT + t) * 16) * MMB + (frag ^ (64 * h)));
    };
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int j = 0; j < C::PER; ++j) issue(j, s, s);

    // The steps, for a wave whose first LIVE tiles of tokens hold any.
    auto steps_of = [&](auto live) {
        constexpr int LIVE = decltype(live)::value;
        u32x4 A[2][MR], Bv[2][MT];
        auto fetch = [&](const uint8_t* wl, int m, int h) {  // what row tile m's turn brings of the next half
            if (LIVE == 0) return;
            A[h][m] = read_a(wl, m, h);
#pragma unroll
            for (int t = m * LIVE / MR; t < (m + 1) * LIVE / MR; ++t) Bv[h][t] = read_b(wl, t, h);
        };
        auto products = [&](int m, int h) {
#pragma unroll
            for (int t = 0; t < LIVE; ++t) acc[m][t] = E::mfma(A[h][m], Bv[h][t], acc[m][t]);
        };
        wait_copies_barrier<(S - 1) * C::PER>();
#pragma unroll
        for (int m = 0; m < MR; ++m) fetch(smem, m, 0);
        int stage = 0;
        for (int s = 0; s < steps; ++s) {
            const uint8_t* wl = smem + stage * C::STAGE;
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                fetch(wl, m, 1);
                products(m, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            // every wave has read this stage, and step s + 1 has landed
            wait_copies_barrier<(S - 2) * C::PER>();
            const int next = stage + 1 == S ? 0 : stage + 1;
            const uint8_t* wn = smem + next * C::STAGE;
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                fetch(wn, m, 0);
                products(m, 1);
#pragma unroll
                for (int j = m * C::PER / MR; j < (m + 1) * C::PER / MR; ++j) issue(j, s + S, stage);
                __builtin_amdgcn_sched_barrier(0);
            }
            stage = next;
        }
    };
    // tiles without tokens (a short last tile of a prompt, an expert with few) are left out
    const int live = (tokens - 16 * MT * wt + 15) / 16;
    if (live > (MT + 1) / 2) steps_of(std::integral_constant<int, MT>{});
    else if (MT > 2 && live > (MT + 3) / 4) steps_of(std::integral_constant<int, (MT + 1) / 2>{});
    else if (live > 0) steps_of(std::integral_constant<int, (MT > 2 ? (MT + 3) / 4 : (MT + 1) / 2)>{});
    else steps_of(std::integral_constant<int, 0>{});
    wait_copies_barrier<0>();  // LDS is free
}

// The linear id's place when each of the 8 XCDs (dealt round by id) takes a run: a bijection of [0, total).
__device__ __forceinline__ int xcd_run(int lin, int total) {
    const int xcd = lin & 7, rem = total & 7;
    return xcd * (total >> 3) + (xcd < rem ? xcd : rem) + (lin >> 3);
}

}  // namespace
}  // namespace tsa
