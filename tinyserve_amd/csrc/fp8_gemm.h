// The tile of the block-scaled FP8 products over many tokens: RN weight rows x TM tokens of a
// workgroup of WR x WT waves, each MR x MT tiles of 16 x 16.
//
// K advances one block of 128 at a time. A block's rows (weights, then tokens; 128 bytes each) come
// into one of S stages in LDS by buffer-to-LDS copies, S - 1 blocks ahead; rows and columns past the
// matrices are offsets past the buffers, which copy zeros. The 16-byte chunk c of row r sits in slot c ^
// (r / 2 % 8): the 16 rows that a quarter wave reads at once then fall on distinct banks. One MFMA
// (v_mfma_f32_16x16x128_f8f6f4) makes a tile's sum over the block, which joins the float32 result
// times the token's and the weight block's scale: 4 fused multiply-adds beside 32 cycles of the matrix
// core. The tokens' scales of a block travel with it (a wave copies those of its own tokens).
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

template <int WR_, int WT_, int MR_, int MT_, int S_>
struct F8Tile {
    static constexpr int WR = WR_, WT = WT_, MR = MR_, MT = MT_, S = S_;
    static constexpr int NW = WR * WT, THREADS = 64 * NW, RN = 16 * WR * MR, TM = 16 * WT * MT;
    static constexpr int NXW = RN / 8 / NW, NXT = TM / 8 / NW;  // copies of 8 rows, a wave's
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
// tile's token r, or -1.
template <class C, int PARTS, bool WIDE, class Token>
__device__ __forceinline__ void f8_tile(const F8Operands<PARTS>& p, uint8_t* smem, Token token, v4f (&acc)[C::MR][C::MT]) {
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
        const int r = lane < 16 * MT ? token(16 * MT * wt + lane) : -1;
        so = r < 0 ? 0x80000000u : (uint32_t)r * (uint32_t)p.G * 4u;
    }
    auto issue = [&](int s, int stage) {
        const uint32_t col = (uint32_t)F8B * (uint32_t)s, base = lds0 + (uint32_t)stage * C::STAGE;
        const bool tail = col + F8B > K;  // the row ends in this block
#pragma unroll
        for (int j = 0; j < C::NXW; ++j) {
            const int n = C::NXW * wave + j;
            uint32_t o = wo[j];
            if (tail && col + 16u * chunk(n) >= K) o = 0x80000000u;
            f8_copy16(rw[PARTS == 1 ? 0 : 8 * n / HALF], o, col, base + 1024u * (uint32_t)n);
        }
#pragma unroll
        for (int j = 0; j < C::NXT; ++j) {
            const int n = C::NXT * wave + j;
            uint32_t o = xo[j];
            if (tail && col + 16u * chunk(n) >= K) o = 0x80000000u;
            f8_copy16(rx, o, col, base + (uint32_t)C::RN * F8B + 1024u * (uint32_t)n);
        }
        f8_copy4(rs, so, 4u * (uint32_t)s, lds0 + (uint32_t)(S * C::STAGE) + 256u * (uint32_t)(C::NW * stage + wave));
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
        if (s < steps) issue(s, s);
    int stage = 0;
    for (int s = 0; s < steps; ++s) {
        if ((s & 63) == 0 && s) load_ws(s);
        // block s has landed (every wave's part of it), and the stage read in step s - 1 is free
        if (s + S - 1 <= steps) f8_wait_barrier<(S - 2) * C::PER>();
        else f8_wait_barrier<0>();
        if (s + S - 1 < steps) issue(s + S - 1, stage == 0 ? S - 1 : stage - 1);
        const uint8_t* wl = smem + stage * C::STAGE;
        const uint8_t* xl = wl + C::RN * F8B + wt * (16 * MT * F8B);
        const float* sl = reinterpret_cast<const float*>(smem + S * C::STAGE + 256 * (C::NW * stage + wave));
        u32x4 Bv[MT][2];
        float sc[PARTS][MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            read(xl + t * (16 * F8B), Bv[t]);
            const float sx = sl[16 * t + i];
#pragma unroll
            for (int h = 0; h < PARTS; ++h)
                sc[h][t] = sx * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsv[h]), s & 63));
        }
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            constexpr int MP = MR / PARTS;
            const int h = m / MP;
            u32x4 A[2];
            read(wl + (h * HALF + (wr * MP + m % MP) * 16) * F8B, A);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const v4f part = f8_mfma<WIDE>(A, Bv[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][t][r] = fmaf(part[r], sc[h][t], acc[m][t][r]);
            }
        }
        stage = stage + 1 == S ? 0 : stage + 1;
    }
}

}  // namespace
}  // namespace tsa
