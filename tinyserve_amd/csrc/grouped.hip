// Products grouped by expert: the rows of a batch are sorted by expert, offsets[e] .. offsets[e + 1] - 1 are
// expert e's (any number of them), and
//     y[r, n] = sum_k x[rows[r] / top_k, k] w[e, n, k]  (+ bias[e, n]);
// int8 operands are scaled as the plain product's are. Rows of no expert are zeros.
//
// One launch, nothing read back: the grid holds as many workgroups as any offsets can need, and each finds its
// tile of rows by a prefix sum over the groups (a wave, four groups a lane; about 0.5 us, where a launch ahead
// that writes a table takes 2 and more).
#include "int8_common.h"
#include "mm_epilogue.h"

namespace tsa {
namespace {

struct Grouped {
    const uint8_t* w;
    int64_t w_stride;  // bytes from an expert's matrix to the next
    const float* ws;   // [E, N]
    const uint8_t* x;
    const float* xs;
    int64_t x_rows;
    const int32_t *offsets, *rows;
    int R, E, N, KB, top_k;
    int tiles_n;
    MmOut out;  // its bias: [E, N]
};

// Inclusive prefix sum over the wave's lanes (DPP: row shifts, then the rows' last lanes passed on).
__device__ __forceinline__ int wave_incl_sum(int v) {
    v += dpp_i<0x111, 0xF, 0xF>(v, 0);
    v += dpp_i<0x112, 0xF, 0xF>(v, 0);
    v += dpp_i<0x114, 0xF, 0xF>(v, 0);
    v += dpp_i<0x118, 0xF, 0xF>(v, 0);
    v += dpp_i<0x142, 0xA, 0xF>(v, 0);
    v += dpp_i<0x143, 0xC, 0xF>(v, 0);
    return v;
}

struct GroupedTile {
    int expert;  // -1: rows of none
    int row0, rows, tile;
};

// The tile of this workgroup: of all (rows of TM of a group, tile of N) pairs in order, each XCD takes a run (the
// row tiles of an expert and the tiles of a row tile share an L2). The rows ahead of the first group and behind
// the last are groups of their own, of no expert. Offsets that do not ascend, or leave [0, R], give groups cut to
// it: every row that is touched is one of the R. False: nothing is left for this workgroup.
template <int TM>
__device__ __forceinline__ bool grouped_tile(const Grouped& p, GroupedTile& o) {
    const int lane = (int)threadIdx.x & 63, G = p.E + 2;
    auto bound = [&](int g) {  // where group g starts: 0, offsets[0 .. E], R
        const int v = p.offsets[g < 1 ? 0 : g - 1 > p.E ? p.E : g - 1];
        return g < 1 ? 0 : g > p.E + 1 ? p.R : v < 0 ? 0 : v > p.R ? p.R : v;
    };
    int b[5], n[4], sum;
    auto load = [&](int g0) {
#pragma unroll
        for (int j = 0; j < 5; ++j) b[j] = bound(g0 + 4 * lane + j);
        sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            n[j] = g0 + 4 * lane + j < G && b[j + 1] > b[j] ? (b[j + 1] - b[j] + TM - 1) / TM : 0;
            sum += n[j];
        }
    };
    int total = 0, incl = 0;
    for (int g0 = 0; g0 < G; g0 += 256) {
        load(g0);
        incl = wave_incl_sum(sum);
        total += __builtin_amdgcn_readlane(incl, 63);
    }
    const int all = total * p.tiles_n, lin = (int)blockIdx.x, xcd = lin & 7, q8 = all >> 3, rem = all & 7;
    if ((lin >> 3) >= q8 + (xcd < rem ? 1 : 0)) return false;
    const int wid = xcd * q8 + (xcd < rem ? xcd : rem) + (lin >> 3);
    int entry = wid / p.tiles_n;
    o.tile = wid % p.tiles_n;
    for (int g0 = 0;; g0 += 256) {
        if (G > 256) {
            load(g0);
            incl = wave_incl_sum(sum);
            const int here = __builtin_amdgcn_readlane(incl, 63);
            if (entry >= here) {
                entry -= here;
                continue;
            }
        }
        int left = entry - (incl - sum), g = -1, r0 = 0, end = 0;  // in this lane's groups
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (g < 0 && left < n[j]) {
                g = g0 + 4 * lane + j;
                r0 = b[j] + TM * left;
                end = b[j + 1];
            }
            left -= n[j];
        }
        const int l = __ffsll((unsigned long long)__ballot(incl > entry)) - 1;
        g = __builtin_amdgcn_readlane(g, l);
        o.row0 = __builtin_amdgcn_readlane(r0, l);
        end = __builtin_amdgcn_readlane(end, l);
        o.rows = end - o.row0 < TM ? end - o.row0 : TM;
        o.expert = g >= 1 && g <= p.E ? g - 1 : -1;
        return true;
    }
}

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) grouped_kernel(Grouped p) {
    extern __shared__ __align__(16) uint8_t smem[];
    GroupedTile g;
    if (!grouped_tile<C::TM>(p, g)) return;
    const int n0 = g.tile * C::RN, row0 = g.row0, tn = g.rows;
    if (g.expert < 0) {
        const int cols = p.N - n0 < C::RN ? p.N - n0 : C::RN;
        for (int r = 0; r < tn; ++r)
            for (int c = threadIdx.x; c < cols; c += C::THREADS) store_out(p.out.y, p.out.y_dtype, (int64_t)(row0 + r) * p.out.ldy + n0 + c, 0.0f);
        return;
    }
    auto token = [&](int r) {  // row of x, -1 for one that is not there
        const int a = p.rows[row0 + r];
        return a >= 0 && a / p.top_k < p.x_rows ? a / p.top_k : -1;
    };
    MmOperands<1> o;
    o.w[0] = p.w + g.expert * p.w_stride + (int64_t)n0 * p.KB;
    o.w_rows = p.N - n0;
    o.KB = (uint32_t)p.KB;
    typename E::acc acc[C::MR][C::MT];
    if (p.rows) {
        o.x = p.x;
        o.x_records = (uint32_t)p.x_rows * (uint32_t)p.KB;
    } else {
        o.x = p.x + (int64_t)row0 * p.KB;
        o.x_records = (uint32_t)tn * (uint32_t)p.KB;
    }
    mm_tile<C, E, 1>(o, smem, tn, [&](int r) { return p.rows ? token(r) : r; }, acc);
    MmOut out = p.out;
    if (out.bias) out.bias = static_cast<const uint8_t*>(out.bias) + (int64_t)g.expert * p.N * (out.bias_dtype == TSA_F32 ? 4 : 2);
    auto scale = [&](int r) {
        if (!p.rows) return p.xs[row0 + r];
        const int t = token(r);
        return t >= 0 ? p.xs[t] : 0.0f;
    };
    mm_store<C>(acc, out, n0, p.N, tn, [&](int r) { return (int64_t)(row0 + r); }, scale, p.ws + (int64_t)g.expert * p.N);
}

template <class C, class E>
hipError_t launch_grouped(const Grouped& p, hipStream_t st) {
    const void* fn = reinterpret_cast<const void*>(&grouped_kernel<C, E>);
    const hipError_t e = ensure_dynamic_lds(fn, C::LDS);
    if (e != hipSuccess) return e;
    Grouped q = p;
    q.tiles_n = (p.N + C::RN - 1) / C::RN;
    void* args[] = {&q};
    // a group of n rows has at most n / TM + 1 tiles, and no more than n
    const int64_t groups = (int64_t)p.E + 2 < p.R ? p.E + 2 : p.R, tiles = p.R / C::TM + groups;
    const int64_t grid = (tiles * q.tiles_n + 7) / 8 * 8;
    return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(C::THREADS), args, C::LDS, st);
}

using Grp128 = MmTile<4, 2, 4, 4, 3>;  // 256 rows x 128 tokens
using Grp64 = MmTile<4, 1, 2, 4, 3>;   // 128 x 64
using Grp32 = MmTile<4, 1, 2, 2, 4>;   // 128 x 32
using Grp16 = MmTile<4, 1, 1, 1, 4>;   // 64 x 16

template <class E>
hipError_t pick_grouped(const Grouped& p, hipStream_t st) {
    const int64_t R = p.R, n = p.E;
    if (R > 48 * n) return launch_grouped<Grp128, E>(p, st);
    if (R > 20 * n) return launch_grouped<Grp64, E>(p, st);
    if (R > 8 * n) return launch_grouped<Grp32, E>(p, st);
    return launch_grouped<Grp16, E>(p, st);
}

constexpr int64_t GROUPED_MAX_E = 65536;

int check_grouped(const void* x, int64_t x_rows, int64_t K, int es, const void* w, int64_t w_stride, int64_t E, int64_t N,
                  const int32_t* offsets, const int32_t* rows, int64_t R, int top_k, const void* bias, int bias_dtype,
                  const void* y, int y_dtype) {
    TSA_REQUIRE(valid_dtype(y_dtype), TSA_ERR_INVALID_ARG, "bad dtype (y %d)", y_dtype);
    TSA_REQUIRE(!bias || valid_dtype(bias_dtype), TSA_ERR_INVALID_ARG, "bad dtype (bias %d)", bias_dtype);
    TSA_REQUIRE(R >= 0 && x_rows >= 0 && E >= 1 && N >= 1 && K >= 1 && top_k >= 1, TSA_ERR_SHAPE,
                "bad shape (rows %lld of %lld, experts %lld, N %lld, K %lld, top_k %d)", (long long)R, (long long)x_rows, (long long)E,
                (long long)N, (long long)K, top_k);
    TSA_REQUIRE(K * es % 16 == 0 && K <= I8_MAX_K, TSA_ERR_SHAPE, "K (%lld) must be a multiple of %d of at most %lld", (long long)K,
                16 / es, (long long)I8_MAX_K);
    TSA_REQUIRE(E <= GROUPED_MAX_E && N <= ((int64_t)1 << 24) && R < ((int64_t)1 << 30) && (R / 16 + E + 2) * ((N + 63) / 64) < ((int64_t)1 << 23),
                TSA_ERR_SHAPE, "%lld rows x N %lld x %lld experts are too many", (long long)R, (long long)N, (long long)E);
    TSA_REQUIRE(w_stride >= N * K * es && w_stride % 16 == 0, TSA_ERR_SHAPE, "the experts' matrices (%lld bytes apart) overlap or are not 16-byte aligned",
                (long long)w_stride);
    if (R == 0) return TSA_OK;
    TSA_REQUIRE(x_rows >= 1 && (rows || x_rows >= R), TSA_ERR_SHAPE, "x has %lld rows for %lld", (long long)x_rows, (long long)R);
    TSA_REQUIRE(!rows || x_rows * K * es < ((int64_t)1 << 31), TSA_ERR_SHAPE, "rows picked from x: x of 2^31 bytes and more is not supported");
    TSA_REQUIRE(x && w && offsets && y, TSA_ERR_INVALID_ARG, "null pointer");
    TSA_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0, TSA_ERR_INVALID_ARG,
                "x and the weights must be 16-byte aligned");
    return TSA_OK;
}

Grouped grouped_params(const void* x, const float* xs, int64_t x_rows, int64_t K, int es, const void* w, int64_t w_stride,
                       const float* ws, int64_t E, int64_t N, const int32_t* offsets, const int32_t* rows, int64_t R, int top_k,
                       const void* bias, int bias_dtype, void* y, int y_dtype) {
    Grouped p{};
    p.w = static_cast<const uint8_t*>(w);
    p.w_stride = w_stride;
    p.ws = ws;
    p.x = static_cast<const uint8_t*>(x);
    p.xs = xs;
    p.x_rows = x_rows;
    p.offsets = offsets;
    p.rows = rows;
    p.R = (int)R;
    p.E = (int)E;
    p.N = (int)N;
    p.KB = (int)(K * es);
    p.top_k = top_k;
    p.out = mm_out(y, y_dtype, N, bias, bias_dtype);
    return p;
}

}  // namespace
}  // namespace tsa

using namespace tsa;

extern "C" int tsa_grouped_matmul(const void* x, int dtype, int64_t x_rows, int64_t K, const void* w, int64_t w_stride, int64_t E,
                                  int64_t N, const int32_t* offsets, const int32_t* rows, int64_t R, int top_k, const void* bias,
                                  int bias_dtype, void* y, int y_dtype, void* stream) {
    clear_error();
    TSA_REQUIRE(dtype == TSA_BF16 || dtype == TSA_F16, TSA_ERR_INVALID_ARG, "bad dtype (x and weights %d: bfloat16 or float16)", dtype);
    const int rc = check_grouped(x, x_rows, K, 2, w, w_stride, E, N, offsets, rows, R, top_k, bias, bias_dtype, y, y_dtype);
    if (rc || R == 0) return rc;
    const Grouped p = grouped_params(x, nullptr, x_rows, K, 2, w, w_stride, nullptr, E, N, offsets, rows, R, top_k, bias, bias_dtype, y, y_dtype);
    TSA_HIP_CHECK(dtype == TSA_BF16 ? pick_grouped<MmBf16>(p, as_stream(stream)) : pick_grouped<MmF16>(p, as_stream(stream)));
    return TSA_OK;
}

extern "C" int tsa_int8_grouped_matmul(const void* codes, const float* scales, int64_t x_rows, int64_t K, const void* w, int64_t w_stride,
                                       const float* w_scales, int64_t E, int64_t N, const int32_t* offsets, const int32_t* rows, int64_t R,
                                       int top_k, const void* bias, int bias_dtype, void* y, int y_dtype, void* stream) {
    clear_error();
    const int rc = check_grouped(codes, x_rows, K, 1, w, w_stride, E, N, offsets, rows, R, top_k, bias, bias_dtype, y, y_dtype);
    if (rc || R == 0) return rc;
    TSA_REQUIRE(scales && w_scales, TSA_ERR_INVALID_ARG, "null pointer");
    const Grouped p = grouped_params(codes, scales, x_rows, K, 1, w, w_stride, w_scales, E, N, offsets, rows, R, top_k, bias, bias_dtype, y, y_dtype);
    TSA_HIP_CHECK(pick_grouped<MmI8>(p, as_stream(stream)));
    return TSA_OK;
}
