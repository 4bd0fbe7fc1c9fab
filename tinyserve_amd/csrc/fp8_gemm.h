// The tile of the block-scaled FP8 products over many tokens: RN weight rows x TM tokens of a
// workgroup of WR x WT waves, each MR x MT tiles of 16 x 16.
//
// K advances one block of 128 at a time. A block's rows (weights, then tokens; 128 bytes each) come
// into one of S stages in LDS by buffer-to-LDS copies, S - 1 blocks ahead; rows and columns past the
// matrices are offsets past the buffers, which copy zeros. The 16-byte chunk c of row r sits in slot c ^
// (r / 2 % 8): the 16 rows that a quarter wave reads at once then fall on distinct banks. One MFMA
// (v_mfma_f32_16x16x128_f8f6f4; WIDE: four bf16 ones) makes a tile's sum over the block, which joins the
// float32 result times the token's and the weight block's scale: 4 fused multiply-adds beside 32 cycles
// of the matrix core. The tokens' scales of a block travel with it.
#pragma once

#include "fp8_common.h"

namespace tsa {
namespace {

typedef int f8_v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f8_v4i f8_desc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return f8_v4i{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                  __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

// Lane l's 16 (or 4) bytes at buffer offset voff + soff land at LDS byte lds + 16 l (or 4 l).
__device__ __forceinline__ void f8_copy16(const f8_v4i& r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\t" TSA_COPY_WAIT "buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff),
                 "s"(__builtin_amdgcn_readfirstlane((int)lds))
                 : "memory", "m0");
}
__device__ __forceinline__ void f8_copy4(const f8_v4i& r, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\t" TSA_COPY_WAIT "buffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff),
                 "s"(__builtin_amdgcn_readfirstlane((int)lds))
                 : "memory", "m0");
}

// This wave's copies have landed but for the newest N, and its LDS reads are done; then the barrier.
template <int N>
__device__ __forceinline__ void f8_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// WR x WT waves of MR x MT tiles of 16 x 16, S stages.
template <int WR_, int WT_, int MR_, int MT_, int S_>
struct F8Tile {
    static constexpr int WR = WR_, WT = WT_, MR = MR_, MT = MT_, S = S_;
    static constexpr int NW = WR * WT, THREADS = 64 * NW, RN = 16 * WR * MR, TM = 16 * WT * MT;
    static constexpr int NXW = RN / 8 / NW, NXT = TM / 8 / NW;  // copies of 8 rows, a wave's
    static constexpr int NS = 16 * MT / WR;  // tokens whose scales a wave copies
    static_assert(NS * WR == 16 * MT, "tile");
    static constexpr int PER = NXW + NXT + 1;                   // copies a wave issues per block
    static constexpr int STAGE = (RN + TM) * F8B, LDS = S * STAGE + S * NW * 256;
    static_assert(RN % (8 * NW) == 0 && TM % (8 * NW) == 0 && MT <= 4 && (S - 2) * PER < 63, "tile");
};

// What a tile multiplies. Weight row r of the tile (r < RN) is row r of w[r / (RN / PARTS)] counted
// from that part's first row, `rows` of them (PARTS 2: the gate and the up rows of an expert).
template <int PARTS>
struct F8Operands {
    const uint8_t* w[PARTS];  // first row of the tile
    int w_rows;               // rows there are from it on (those past RN / PARTS are not read)
    const float* ws[PARTS];   // the scales of its 128-row block: [G]
    const uint8_t* x;         // codes [., K], scales [., G]
    const float* xs;
    uint32_t x_records, xs_records;  // their bytes
    int K, G;
};

// acc[m][t]: rows 4 q .. 4 q + 3 of tile m, token 16 t + i, for lane 16 q + i of the wave. Tile m is
// the wave's m-th: of its MR, the first MR / PARTS belong to part 0. `token(r)`: row of x of the
// tile's token r, -1 from `tokens` on.
template <class C, int PARTS, bool WIDE, class Token>
__device__ __forceinline__ void f8_tile(const F8Operands<PARTS>& p, uint8_t* smem, int tokens, Token token, v4f (&acc)[C::MR][C::MT]) {
    constexpr int MR = C::MR, MT = C::MT, S = C::S, HALF = C::RN / PARTS;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    const uint32_t K = (uint32_t)p.K, lds0 = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int steps = p.G;

    // copy j of this wave fills rows 8 (NX wave + j) + lane / 8, slot lane % 8
    f8_v4i rw[PARTS];
#pragma unroll
    for (int h = 0; h < PARTS; ++h) rw[h] = f8_desc(p.w[h], (uint32_t)(p.w_rows < HALF ? p.w_rows : HALF) * K);
    const f8_v4i rx = f8_desc(p.x, p.x_records), rs = f8_desc(p.xs, p.xs_records);
    uint32_t wo[C::NXW], xo[C::NXT];
    auto chunk = [&](int n) { return (uint32_t)((lane & 7) ^ ((4 * n + (lane >> 4)) & 7)); };  // of copy n's rows
#pragma unroll
    for (int j = 0; j < C::NXW; ++j) {
        const int n = C::NXW * wave + j;
        wo[j] = (uint32_t)(8 * n + (lane >> 3)) % HALF * K + 16u * chunk(n);
    }
#pragma unroll
    for (int j = 0; j < C::NXT; ++j) {
        const int n = C::NXT * wave + j, r = token(8 * n + (lane >> 3));
        xo[j] = r < 0 ? 0x80000000u : (uint32_t)r * K + 16u * chunk(n);
    }
    uint32_t so;
    {
        // the waves of a token column share its scales' copies: a row's scale is a line of its own
        const int r = lane < C::NS ? token(16 * MT * wt + C::NS * wr + lane) : -1;
        so = r < 0 ? 0x80000000u : (uint32_t)r * (uint32_t)p.G * 4u;
    }
    // copy j (of PER) of block s: the weights', the tokens', the scales'. Columns past K and blocks past
    // the last read zeros, so every step issues as many. (The scalar offset stays inside the buffers:
    // the range check may subtract it from their size.)
    uint32_t at[2];  // this lane's column in copies of even and odd number
#pragma unroll
    for (int n = 0; n < 2; ++n) at[n] = 16u * chunk(n);
    auto issue = [&](int j, int s, int stage) {
        const uint32_t col = (uint32_t)F8B * (uint32_t)s, base = lds0 + (uint32_t)stage * C::STAGE;
        const uint32_t soff = s < steps ? col : 0u;
        if (j < C::NXW) {
            const int n = C::NXW * wave + j;
            const bool in = col + (n & 1 ? at[1] : at[0]) < K;
            f8_copy16(rw[PARTS == 1 ? 0 : 8 * n / HALF], in ? wo[j] : 0x80000000u, soff, base + 1024u * (uint32_t)n);
        } else if (j < C::NXW + C::NXT) {
            const int n = C::NXT * wave + j - C::NXW;
            const bool in = col + (n & 1 ? at[1] : at[0]) < K;
            f8_copy16(rx, in ? xo[j - C::NXW] : 0x80000000u, soff, base + (uint32_t)C::RN * F8B + 1024u * (uint32_t)n);
        } else {
            f8_copy4(rs, s < steps ? so : 0x80000000u, soff / 32,
                     lds0 + (uint32_t)(S * C::STAGE) + 256u * (uint32_t)(C::NW * stage + wave));
        }
    };

#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[m][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    const int frag = i * F8B + 16 * (q ^ (i >> 1));  // chunk q of row i of a tile; chunk q + 4 is 64 off by xor
    auto read = [&](const uint8_t* tile, u32x4 (&v)[2]) {
        v[0] = *reinterpret_cast<const u32x4*>(tile + frag);
        v[1] = *reinterpret_cast<const u32x4*>(tile + (frag ^ 64));
    };
    // the weights' scales, 64 blocks at a time, a lane each, and loaded before anything goes on: a
    // wait for them later would wait for the copies issued in between
    float wsv[PARTS];
    auto load_ws = [&](int s) {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) wsv[h] = p.ws[h][s + lane < p.G ? s + lane : p.G - 1];
#pragma unroll
        for (int h = 0; h < PARTS; ++h) asm volatile("" : "+v"(wsv[h]));
    };
    load_ws(0);
#pragma unroll
    for (int s = 0; s < S - 1; ++s)
#pragma unroll
        for (int j = 0; j < C::PER; ++j) issue(j, s, s);

    // The blocks, for a wave whose first LIVE tiles of tokens hold any.
    auto blocks = [&](auto live) {
        constexpr int LIVE = decltype(live)::value, MP = MR / PARTS;
        u32x4 A[2][2], Bv[MT][2];
        float sc[PARTS][MT];
        v4f part[2][MT];
        auto row_tile = [&](const uint8_t* wl, int m) { return wl + (m / MP * HALF + (wr * MP + m % MP) * 16) * F8B; };
        auto scales = [&](int s, int stage) {
            const float* sl = reinterpret_cast<const float*>(smem + S * C::STAGE + 256 * (C::NW * stage + C::WR * wt));
#pragma unroll
            for (int t = 0; t < LIVE; ++t) {
                const float sx = sl[64 * ((16 * t + i) / C::NS) + (16 * t + i) % C::NS];
#pragma unroll
                for (int h = 0; h < PARTS; ++h)
                    sc[h][t] = sx * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsv[h]), s & 63));
            }
        };
        auto fetch_b = [&](const uint8_t* wl) {
#pragma unroll
            for (int t = 0; t < LIVE; ++t) read(wl + C::RN * F8B + (wt * MT + t) * (16 * F8B), Bv[t]);
        };
        auto join = [&](int m, int t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m][t][r] = fmaf(part[m & 1][t][r], sc[m / MP][t], acc[m][t][r]);
        };
        // The products of a block. A row tile's sums (part) join the results while the next row tile's
        // are made: no multiply-add waits for the matrix core. The copies of block `next` go out between
        // the row tiles: issued at once they hold up the wave until the memory pipe has taken them.
        auto products = [&](const uint8_t* wl, int next, int stage) {
#pragma unroll
            for (int m = 0; m < MR; ++m) {
#pragma unroll
                for (int t = 0; t < LIVE; ++t) {
                    if (t == 0 && m + 1 < MR) read(row_tile(wl, m + 1), A[(m + 1) & 1]);
                    part[m & 1][t] = f8_mfma<WIDE>(A[m & 1], Bv[t]);
                    if (m) join(m - 1, t);
                    if constexpr (!WIDE) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = m * C::PER / MR; j < (m + 1) * C::PER / MR; ++j) issue(j, next, stage);
            }
#pragma unroll
            for (int t = 0; t < LIVE; ++t) join(MR - 1, t);
        };
        int stage = 0;
        for (int s = 0; s < steps; ++s) {
            if ((s & 63) == 0 && s) load_ws(s);
            // block s has landed (every wave's part of it), and the stage read in step s - 1 is free
            f8_wait_barrier<(S - 2) * C::PER>();
            const uint8_t* wl = smem + stage * C::STAGE;
            if (LIVE) read(row_tile(wl, 0), A[0]);
            fetch_b(wl);
            scales(s, stage);
            products(wl, s + S - 1, stage == 0 ? S - 1 : stage - 1);
            stage = stage + 1 == S ? 0 : stage + 1;
        }
    };
    // tiles without tokens (a short last tile of a prompt, an expert with few) are left out
    const int live = (tokens - 16 * MT * wt + 15) / 16;
    if (live >= MT || (MT == 4 && live == 3)) blocks(std::integral_constant<int, MT>{});
    else if (live == 2) blocks(std::integral_constant<int, (MT > 2 ? 2 : MT)>{});
    else if (live == 1) blocks(std::integral_constant<int, 1>{});
    else blocks(std::integral_constant<int, 0>{});
    f8_wait_barrier<0>();  // LDS is free
}

}  // namespace
}  // namespace tsa
