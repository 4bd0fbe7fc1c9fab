// Products of int8 and 16-bit matrices over many tokens: tiles of RN weight rows x TM tokens, each by a workgroup
// of WR x WT waves with MR x MT tiles of 16 x 16.
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
// second half's operands are in registers, so the stage is free for the copies of step s + S. They go out among the
// products of the second half and of the next step's first (with two stages, which are waited for there, of the second
// half alone; all of them there with three: 2% slower, 4096 x 5760 x 2880 int8 90.5 us for 88.3, 8192 rows of 32
// experts of 5760 x 2880 bf16 378 for 371). The LDS reads of a half go out among the products of the half before.
//
// A workgroup works through tiles one after the other, and their steps are one stream: the last S steps of a tile
// issue the copies of the next tile's first, and the results go out while those land.
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
    static constexpr int STAGE = (RN + 8 * NW * NXT) * MMB;
    static constexpr int OUT = 16 * MR * 32;  // a wave's place for 16 tokens' results of 16 bits
    static constexpr int LDS = S * STAGE + NW * OUT;
    static_assert(RN % (8 * NW) == 0 && (S - 1) * PER < 63 && S >= 2 && LDS <= 160 * 1024, "tile");
};

// What a tile multiplies. Weight row r of the tile (r < RN) is row r of w[r / (RN / PARTS)] counted
// from that part's first row, w_rows of them (PARTS 2: the gate and the up rows of an expert).
template <int PARTS>
struct MmOperands {
    const uint8_t* w[PARTS];  // first row of the tile
    int w_rows;               // rows there are from it on (those past RN / PARTS are not read)
    const uint8_t* x;
    uint32_t x_records;       // its bytes, at most 2^31
    int tokens;
};

// Works through `work`'s tiles. KB: bytes of a row of either operand, a multiple of 16.
//   bool work.next(): the next tile becomes work's pending one (uniform); false: there is none
//   MmOperands<PARTS> work.operands(), int work.token(r): of the pending tile; the row of x of its token r (-1: zeros);
//     GATHER false: token r is row r
//   void work.take(): the pending tile becomes the current one
//   void work.store(acc, out): the current tile's results; `out`: this wave's place in LDS
// acc[m][t]: rows 4 q .. 4 q + 3 of tile m, token 16 t + i, for lane 16 q + i of the wave. Tile m is
// the wave's m-th: of its MR, the first MR / PARTS belong to part 0.
template <class C, class E, int PARTS, bool GATHER, class Work>
__device__ __forceinline__ void mm_run(Work& work, uint32_t KB, uint8_t* smem) {
    constexpr int MR = C::MR, MT = C::MT, S = C::S, HALF = C::RN / PARTS, MP = MR / PARTS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(smem);
    const int all = (int)((KB + MMB - 1) / MMB), steps = all > S ? all : S;  // short rows: steps of zeros

    // copy j of this wave fills rows 8 (NX wave + j) + lane / 8, slot lane % 8
    buf_v4i rw[PARTS], rx;
    uint32_t wo[C::NXW], xo[C::NXT];
    auto chunk = [&](int n) { return (uint32_t)((lane & 7) ^ ((4 * n + (lane >> 4)) & 7)); };  // of copy n's rows
#pragma unroll
    for (int j = 0; j < C::NXW; ++j) {
        const int n = C::NXW * wave + j;
        wo[j] = (uint32_t)(8 * n + (lane >> 3)) % HALF * KB + 16u * chunk(n);
    }
#pragma unroll
    for (int j = 0; j < C::NXT; ++j) {
        const int n = C::NXT * wave + j;
        xo[j] = (uint32_t)(8 * n + (lane >> 3)) * KB + 16u * chunk(n);  // past x's records: zeros
    }
    uint32_t at[2];  // this lane's column in copies of even and odd number
#pragma unroll
    for (int n = 0; n < 2; ++n) at[n] = 16u * chunk(n);
    int tokens = 0, pending = 0;  // of the tile whose products run, and of the one whose copies go out
    // the copies' tile becomes work's pending one (none: buffers without bytes)
    auto setup = [&](bool there) {
        if (!there) {
#pragma unroll
            for (int h = 0; h < PARTS; ++h) rw[h] = buf_desc(smem, 0);
            rx = buf_desc(smem, 0);
            return;
        }
        const MmOperands<PARTS> p = work.operands();
        pending = p.tokens;
#pragma unroll
        for (int h = 0; h < PARTS; ++h) rw[h] = buf_desc(p.w[h], (uint32_t)(p.w_rows < HALF ? p.w_rows : HALF) * KB);
        rx = buf_desc(p.x, p.x_records);
        if constexpr (GATHER) {
#pragma unroll
            for (int j = 0; j < C::NXT; ++j) {
                const int n = C::NXT * wave + j, r = 8 * n + (lane >> 3), row = r < p.tokens ? work.token(r) : -1;
                xo[j] = row < 0 ? 0x80000000u : (uint32_t)row * KB + 16u * chunk(n);
            }
        }
    };
    // copy j (of PER) of step s. Columns past K and steps past the last read zeros, so every step issues as
    // many. (The scalar offset stays inside the buffers: the range check may subtract it from their size.)
    auto issue = [&](int j, int s, int stage) {
        const uint32_t col = (uint32_t)MMB * (uint32_t)s, base = lds0 + (uint32_t)stage * C::STAGE;
        const uint32_t soff = s < all ? col : 0u;
        const int n = j < C::NXW ? C::NXW * wave + j : C::NXT * wave + j - C::NXW;
        const bool in = col + (n & 1 ? at[1] : at[0]) < KB;
        if (j < C::NXW) lds_copy16(rw[PARTS == 1 ? 0 : 8 * n / HALF], in ? wo[j] : 0x80000000u, soff, base + 1024u * (uint32_t)n);
        else lds_copy16(rx, in ? xo[j - C::NXW] : 0x80000000u, soff, base + (uint32_t)C::RN * MMB + 1024u * (uint32_t)n);
    };

    const int frag = i * MMB + 16 * (q ^ (i >> 1));  // chunk q of row i of a tile; chunk q + 4 is 64 off by xor
    u32x4 A[2][MR], Bv[2][MT];
    typename E::acc acc[MR][MT];
    auto fetch = [&](const uint8_t* wl, int m, int h) {  // what row tile m's turn brings of the next half
        A[h][m] = *reinterpret_cast<const u32x4*>(wl + (m / MP * HALF + (wr * MP + m % MP) * 16) * MMB + (frag ^ (64 * h)));
#pragma unroll
        for (int t = m * MT / MR; t < (m + 1) * MT / MR; ++t)
            Bv[h][t] = *reinterpret_cast<const u32x4*>(wl + (C::RN + (wt * MT + t) * 16) * MMB + (frag ^ (64 * h)));
    };

    bool more = work.next();
    if (!more) return;
    setup(true);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int j = 0; j < C::PER; ++j) issue(j, s, s);
    wait_copies_barrier<(S - 1) * C::PER>();
    int stage = 0;
    do {
        work.take();
        tokens = pending;
        // (read again after a tile's results: held through them, the operands would take too many registers)
#pragma unroll
        for (int m = 0; m < MR; ++m) fetch(smem + stage * C::STAGE, m, 0);
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[m][t] = typename E::acc{0, 0, 0, 0};
        // token tiles that hold none (a short last tile of a prompt, an expert with few) are left out, by halves
        constexpr int H0 = (MT + 1) / 2;
        const int live = (tokens - 16 * MT * wt + 15) / 16;
        auto products = [&](int m, int h) {
            if (live > 0) {
#pragma unroll
                for (int t = 0; t < H0; ++t) acc[m][t] = E::mfma(A[h][m], Bv[h][t], acc[m][t]);
            }
            if (live > H0) {
#pragma unroll
                for (int t = H0; t < MT; ++t) acc[m][t] = E::mfma(A[h][m], Bv[h][t], acc[m][t]);
            }
        };
        // row tile m's turn of copies [j0, j1)
        auto copies = [&](int m, int j0, int j1, int s, int into) {
#pragma unroll
            for (int j = j0 + m * (j1 - j0) / MR; j < j0 + (m + 1) * (j1 - j0) / MR; ++j) issue(j, s, into);
        };
        auto second = [&](int s, int copied) {  // of step s, and of the copies of step s + S the first `copied`
            const int next = stage + 1 == S ? 0 : stage + 1;
            const uint8_t* wn = smem + next * C::STAGE;
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                fetch(wn, m, 0);
                products(m, 1);
                copies(m, 0, copied, s, stage);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        constexpr int FIRST = S > 2 ? C::PER / 2 : C::PER;
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            fetch(smem + stage * C::STAGE, m, 1);
            products(m, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        wait_copies_barrier<(S - 2) * C::PER>();
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {  // the steps whose copies are this tile's, then those of the next
            if (part) {
                more = work.next();
                setup(more);
            }
            const int s1 = part ? steps - 1 : steps - S, ahead = part ? S - steps : S;
#pragma unroll 1
            for (int s = part ? steps - S : 0; s < s1; ++s) {
                second(s + ahead, FIRST);
                const int free = stage;
                stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    fetch(smem + stage * C::STAGE, m, 1);
                    products(m, 0);
                    copies(m, FIRST, C::PER, s + ahead, free);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // every wave has read this stage, and the next step has landed
                wait_copies_barrier<(S - 2) * C::PER>();
            }
        }
        second(S - 1, C::PER);
        stage = stage + 1 == S ? 0 : stage + 1;
        if (!more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may land after the workgroup's end
        work.store(acc, smem + S * C::STAGE + wave * C::OUT);
    } while (more);
}

// The linear id's place when each of the 8 XCDs (dealt round by id) takes a run: a bijection of [0, total).
__device__ __forceinline__ int xcd_run(int lin, int total) {
    const int xcd = lin & 7, rem = total & 7;
    return xcd * (total >> 3) + (xcd < rem ? xcd : rem) + (lin >> 3);
}

// The places of [0, total) that a workgroup of a grid of whole rounds of XCDs works through: each XCD takes a run, its
// workgroups the places of it in turn.
struct MmRuns {
    int at, end, step;
    __device__ __forceinline__ explicit MmRuns(int total) {
        const int lin = (int)blockIdx.x, xcd = lin & 7, rem = total & 7, first = xcd * (total >> 3) + (xcd < rem ? xcd : rem);
        step = (int)gridDim.x >> 3;
        end = first + (total >> 3) + (xcd < rem ? 1 : 0);
        at = first + (lin >> 3) - step;
    }
    __device__ __forceinline__ bool next() {
        at += step;
        return at < end;
    }
};

// Item `at` of the (entry, row tile) pairs of a grouped product: in bands of 2 row tiles, entry by entry. Each XCD's run is
// then a few row tiles of every expert: a matrix's rows are read by one XCD, which shares them among its entries in
// L2, and experts with few tokens (a stream of weights) and with many (products) are spread over all XCDs alike.
// (8192 rows of 32 uneven experts, 5760 x 2880, bf16: 386 us with runs of whole experts in bands of 8, 366 so; later, bands
// of 1 / 2 / 3 / an eighth of the row tiles 384 / 374 / 383 / 379, 24 tokens of 128 experts 46 / 44 / 49 / 49.)
__device__ __forceinline__ void mm_pair(int at, int entries, int tiles, int& entry, int& tile) {
    constexpr int BAND = 2;
    const int band = at / (BAND * entries), in = at - band * BAND * entries, deep = tiles - BAND * band < BAND ? tiles - BAND * band : BAND;
    entry = in / deep;
    tile = BAND * band + in % deep;
}

// Workgroups for `tiles` tiles where `per` of them run on a CU at a time: whole rounds of XCDs.
inline unsigned mm_grid(int64_t tiles, int per) {
    const int64_t most = (int64_t)(num_cus() >= 8 ? num_cus() : 256) * per;
    return (unsigned)(((tiles < most ? tiles : most) + 7) / 8 * 8);
}

}  // namespace
}  // namespace tsa
