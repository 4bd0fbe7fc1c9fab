// Products grouped by expert: the rows of a batch are sorted by expert, offsets[e] .. offsets[e + 1] - 1 are
// expert e's (any number of them), and
//     y[r, n] = sum_k x[rows[r] / top_k, k] w[e, n, k]  (+ bias[e, n]);
// int8 operands are scaled as the plain product's are. Rows of no expert are zeros.
//
// One launch, nothing read back: each workgroup finds its tiles by a prefix sum over the groups (a wave, four groups
// a lane).
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

// Over the wave's lanes (DPP: row shifts, then the rows' last lanes passed on): the sum up to this lane, and the largest
// of the lanes before it (0 for none; of numbers that are not negative).
__device__ __forceinline__ int wave_incl_sum(int v) {
    v += dpp_i<0x111, 0xF, 0xF>(v, 0);
    v += dpp_i<0x112, 0xF, 0xF>(v, 0);
    v += dpp_i<0x114, 0xF, 0xF>(v, 0);
    v += dpp_i<0x118, 0xF, 0xF>(v, 0);
    v += dpp_i<0x142, 0xA, 0xF>(v, 0);
    v += dpp_i<0x143, 0xC, 0xF>(v, 0);
    return v;
}
__device__ __forceinline__ int wave_excl_max(int v) {
    v = max(v, dpp_i<0x111, 0xF, 0xF>(v, 0));
    v = max(v, dpp_i<0x112, 0xF, 0xF>(v, 0));
    v = max(v, dpp_i<0x114, 0xF, 0xF>(v, 0));
    v = max(v, dpp_i<0x118, 0xF, 0xF>(v, 0));
    v = max(v, dpp_i<0x142, 0xA, 0xF>(v, 0));
    v = max(v, dpp_i<0x143, 0xC, 0xF>(v, 0));
    return __shfl_up(v, 1, 64) * ((threadIdx.x & 63) != 0);
}

// A workgroup's tiles (mm_pair's order; an entry: up to TM rows of a group). The rows ahead of the first group and
// behind the last are groups of their own, of no expert. Offsets that do not ascend, or leave [0, R], are raised to the
// largest before them and cut to it: each of the R rows is in one group whatever they hold.
template <class C, class E>
struct GroupedWork {
    static constexpr int TM = C::TM;
    const Grouped& p;
    int entries;
    int b[5], n[4], sum, incl;  // this lane's four groups (of the first 256): bounds, entries, their sums
    MmRuns runs;
    int expert, n0, row0, tn, next_expert, next_n0, next_row0, next_tn;

    __device__ __forceinline__ int bound(int g) const {  // where group g starts: 0, offsets[0 .. E], R
        const int v = p.offsets[g < 1 ? 0 : g - 1 > p.E ? p.E : g - 1];
        return g < 1 ? 0 : g > p.E + 1 ? p.R : v < 0 ? 0 : v > p.R ? p.R : v;
    }
    int reached;  // the largest bound of the groups ahead of those that are loaded
    __device__ __forceinline__ void load(int g0) {
        const int lane = (int)threadIdx.x & 63;
        if (g0 == 0) reached = 0;
#pragma unroll
        for (int j = 0; j < 5; ++j) b[j] = bound(g0 + 4 * lane + j);
#pragma unroll
        for (int j = 1; j < 5; ++j) b[j] = max(b[j], b[j - 1]);
        const int before = max(reached, wave_excl_max(b[4]));
#pragma unroll
        for (int j = 0; j < 5; ++j) b[j] = max(b[j], before);
        reached = __builtin_amdgcn_readlane(b[4], 63);
        sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            n[j] = g0 + 4 * lane + j < p.E + 2 && b[j + 1] > b[j] ? (b[j + 1] - b[j] + TM - 1) / TM : 0;
            sum += n[j];
        }
        incl = wave_incl_sum(sum);
    }
    __device__ __forceinline__ int count() {
        entries = 0;
        for (int g0 = 0; g0 < p.E + 2; g0 += 256) {
            load(g0);
            entries += __builtin_amdgcn_readlane(incl, 63);
        }
        return entries * p.tiles_n;
    }
    __device__ __forceinline__ explicit GroupedWork(const Grouped& p) : p(p), runs(count()) {}
    __device__ __forceinline__ bool next() {
        while (runs.next()) {
            int entry, tile;
            mm_pair(runs.at, entries, p.tiles_n, entry, tile);
            next_n0 = tile * C::RN;
            for (int g0 = 0;; g0 += 256) {
                if (p.E + 2 > 256) {
                    load(g0);
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
                        g = g0 + 4 * ((int)threadIdx.x & 63) + j;
                        r0 = b[j] + TM * left;
                        end = b[j + 1];
                    }
                    left -= n[j];
                }
                const int l = __ffsll((unsigned long long)__ballot(incl > entry)) - 1;
                g = __builtin_amdgcn_readlane(g, l);
                next_row0 = __builtin_amdgcn_readlane(r0, l);
                end = __builtin_amdgcn_readlane(end, l);
                next_tn = end - next_row0 < TM ? end - next_row0 : TM;
                next_expert = g >= 1 && g <= p.E ? g - 1 : -1;
                break;
            }
            if (next_expert >= 0) return true;
            // rows of no expert: 16 bytes at a time where y's rows allow it
            const int cols = p.N - next_n0 < C::RN ? p.N - next_n0 : C::RN, es = p.out.y_dtype == TSA_F32 ? 4 : 2;
            uint8_t* y = static_cast<uint8_t*>(p.out.y) + (next_row0 * p.out.ldy + next_n0) * es;
            const int bytes = cols * es, piece = p.out.y_vec ? 16 : 2, per = bytes / piece;
            for (int c = threadIdx.x; c < next_tn * per; c += C::THREADS) {
                uint8_t* at = y + (c / per) * p.out.ldy * es + c % per * piece;
                if (piece == 16) *reinterpret_cast<u32x4*>(at) = u32x4{0, 0, 0, 0};
                else *reinterpret_cast<uint16_t*>(at) = 0;
            }
        }
        return false;
    }
    __device__ __forceinline__ int picked(int row) const {  // row of x, -1 for one that is not there
        const int a = p.rows[row];
        return a >= 0 && a / p.top_k < p.x_rows ? a / p.top_k : -1;
    }
    __device__ __forceinline__ int token(int r) const { return p.rows ? picked(next_row0 + r) : r; }
    __device__ __forceinline__ MmOperands<1> operands() const {
        const uint8_t* w = p.w + next_expert * p.w_stride + (int64_t)next_n0 * p.KB;
        const uint8_t* x = p.rows ? p.x : p.x + (int64_t)next_row0 * p.KB;
        return MmOperands<1>{{w}, p.N - next_n0, x, (uint32_t)(p.rows ? p.x_rows : next_tn) * (uint32_t)p.KB, next_tn};
    }
    __device__ __forceinline__ void take() { expert = next_expert, n0 = next_n0, row0 = next_row0, tn = next_tn; }
    __device__ __forceinline__ void store(const typename E::acc (&acc)[C::MR][C::MT], uint8_t* out) const {
        MmOut o = p.out;
        if (o.bias) o.bias = static_cast<const uint8_t*>(o.bias) + (int64_t)expert * p.N * (o.bias_dtype == TSA_F32 ? 4 : 2);
        auto scale = [&](int r) {
            const int t = p.rows ? picked(row0 + r) : row0 + r;
            return t >= 0 ? p.xs[t] : 0.0f;
        };
        mm_store<C>(acc, o, out, n0, p.N, tn, [&](int r) { return (int64_t)(row0 + r); }, scale, p.ws + (int64_t)expert * p.N);
    }
};

template <class C, class E>
__global__ void __launch_bounds__(C::THREADS) grouped_kernel(Grouped p) {
    extern __shared__ __align__(16) uint8_t smem[];
    GroupedWork<C, E> work(p);
    mm_run<C, E, 1, true>(work, (uint32_t)p.KB, smem);
}

template <class C, class E>
hipError_t launch_grouped(const Grouped& p, int per, hipStream_t st) {
    const void* fn = reinterpret_cast<const void*>(&grouped_kernel<C, E>);
    const hipError_t e = ensure_dynamic_lds(fn, C::LDS);
    if (e != hipSuccess) return e;
    Grouped q = p;
    q.tiles_n = (p.N + C::RN - 1) / C::RN;
    void* args[] = {&q};
    // a group of n rows has at most n / TM + 1 tiles, and no more than n
    const int64_t groups = (int64_t)p.E + 2 < p.R ? p.E + 2 : p.R, tiles = p.R / C::TM + groups;
    return hipLaunchKernel(fn, dim3(mm_grid(tiles * q.tiles_n, per)), dim3(C::THREADS), args, C::LDS, st);
}

using Grp128 = MmTile<4, 2, 4, 4, 3>;  // 256 rows x 128 tokens
using Grp64 = MmTile<4, 1, 2, 4, 3>;   // 128 x 64
using Grp16 = MmTile<4, 1, 1, 1, 4>;   // 64 x 16

// us in tiles of 16 / 64 / 128 rows, groups uneven by a factor of four: 32 experts of 5760 x 2880, 2 / 12 / 32 / 72 / 250 rows each
// on average, int8 103 / 101 / 105, 116 / 106 / 113, 178 / 123 / 121, 290 / 155 / 146 and 804 / 304 / 231, bf16 185 / 186 / 182, 191 /
// 189 / 190, 286 / 209 / 203, 457 / 250 / 226 and 1309 / 480 / 355; 112 experts of 1536 x 2048, 2 / 32 / 72 / 120 rows, int8 63 / 64 /
// 67, 99 / 74 / 78, 170 / 87 / 96 and 262 / 107 / 96. A few rows: 128 experts, 16 rows in all, bf16 16.2 / 17.7 / 24.2; 19 experts of
// 967 x 528, 66 rows 9.4 / 10.1 / 13.5.
template <class E>
hipError_t pick_grouped(const Grouped& p, hipStream_t st) {
    const int64_t R = p.R, n = p.E;
    if (R <= 4 * n) return launch_grouped<Grp16, E>(p, 2, st);
    if (R <= 48 * n) return launch_grouped<Grp64, E>(p, 2, st);
    return launch_grouped<Grp128, E>(p, 1, st);
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
