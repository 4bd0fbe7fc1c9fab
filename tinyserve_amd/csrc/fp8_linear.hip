// FP8 quantisation of activations and the block-scaled FP8 product
//     y[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{k in block b} cx[t, k] cw[n, k]  (+ bias[n]).
#include "fp8_gemm.h"

namespace tsa {
namespace {

// ---------------------------------------------------------------- quantisation
// A thread takes 8 values, 16 lanes a group; rows are handled as one run of groups.
template <int XT, bool VEC>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const void* __restrict__ x, int64_t T, int K,
                                                           uint8_t* __restrict__ codes, float* __restrict__ scales) {
    const int64_t G = f8_blocks(K), task = (int64_t)blockIdx.x * 256 + threadIdx.x, g = task >> 4;
    if (g >= T * G) return;  // the 16 lanes of a group return together
    const int64_t t = g / G;
    const int c = (int)(g - t * G) * 16 + (int)(task & 15);
    const uint32_t col = 8u * (uint32_t)c;  // up to 2^31 + 120
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const uint8_t* row = static_cast<const uint8_t*>(x) + t * K * ES;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (VEC) {
        if (col < (uint32_t)K) f8_load8<XT>(row, c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < (uint32_t)K) v[e] = load_act(row, XT, (int64_t)(col + e));
    }
    const float s = f8_scale(f8_group_max(v));
    const uint2 o = f8_codes8<XT == TSA_F32>(v, s);
    uint8_t* dst = codes + t * K + col;
    if constexpr (VEC) {
        if (col < (uint32_t)K) *reinterpret_cast<uint2*>(dst) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < (uint32_t)K) dst[e] = (uint8_t)((e < 4 ? o.x : o.y) >> (8 * (e & 3)));
    }
    if ((task & 15) == 0) scales[g] = s;
}

// A launch ends at 2^32 threads (2^28 groups): more rows than that go in several.
template <int XT>
hipError_t launch_quantize(const void* x, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
    constexpr uintptr_t AL = 15;
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & AL) == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const int64_t G = f8_blocks(K), step = ((int64_t)1 << 27) / G;  // K < 2^31: 8 rows and more
    for (int64_t t = 0; t < T; t += step) {
        const int64_t n = T - t < step ? T - t : step;
        const uint8_t* xt = static_cast<const uint8_t*>(x) + t * K * ES;
        const dim3 grid((unsigned)((n * G * 16 + 255) / 256));
        if (vec) hipLaunchKernelGGL((fp8_quantize_kernel<XT, true>), grid, dim3(256), 0, st, xt, n, (int)K, codes + t * K, scales + t * G);
        else hipLaunchKernelGGL((fp8_quantize_kernel<XT, false>), grid, dim3(256), 0, st, xt, n, (int)K, codes + t * K, scales + t * G);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---------------------------------------------------------------- few tokens
struct F8Rows {
    const uint8_t* w;
    const float* ws;
    const void* x;    // codes (XT -1) or values
    const float* xs;  // codes: their scales
    const void* bias;
    int bias_dtype;
    void* y;
    int y_dtype;
    int64_t T, N, ldy;  // ldy: y's row, N of the whole product
    int K, G;
    int tiles_n, rows;  // rows: tokens of the largest tile
};

constexpr int F8R_NW = 8, F8R_D = 3;  // waves; K blocks a wave has in flight

// The linear id's place when each of the 8 XCDs (dealt round by id) takes a run: a bijection of [0, total).
__device__ __forceinline__ int f8_run(int lin, int total) {
    const int xcd = lin & 7, rem = total & 7;
    return xcd * (total >> 3) + (xcd < rem ? xcd : rem) + (lin >> 3);
}

// Workgroup = 16 weight rows x 16 MT tokens; its waves take the K blocks in turn and their sums meet in
// LDS. The weights come straight into the A operand's registers (every byte is read by one lane of
// the workgroup), the tokens' codes from memory, or (XT: their dtype, up to 16 tokens) quantised here
// into LDS while the weights are on their way.
template <int XT, int MT, bool WIDE>
__global__ void __launch_bounds__(64 * F8R_NW) fp8_rows_kernel(F8Rows p) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int NT = 64 * F8R_NW;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const int wid = f8_run((int)blockIdx.x, (int)gridDim.x), tt = (int)gridDim.x / p.tiles_n;
    const int64_t n0 = (int64_t)(wid / tt) * 16, t0 = (int64_t)(wid % tt) * (16 * MT);
    const int tn = (int)(p.T - t0 < 16 * MT ? p.T - t0 : 16 * MT), K = p.K, G = p.G;
    const int ld = G * F8B + 16, tasks = G * 16;  // LDS row of codes; pieces of 8 of a token
    static_assert(XT < 0 || MT == 1, "one token tile is quantised here");
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const uint8_t* xrow = static_cast<const uint8_t*>(p.x) + t0 * K * (XT < 0 ? 1 : ES);
    float xv[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (XT >= 0) {  // the first token's values ahead of the weights
        if (8 * tid < K) f8_load8<XT>(xrow, tid, xv);
    }
    const __amdgpu_buffer_rsrc_t rw = f8_buf(p.w + n0 * K, (p.N - n0 < 16 ? p.N - n0 : 16) * K);
    const __amdgpu_buffer_rsrc_t rx = f8_buf(xrow, XT >= 0 ? 0 : (int64_t)tn * K);
    const float* sw = p.ws + n0 / F8B * G;
    const float* xs = p.xs + (XT < 0 ? t0 * G : 0);
    u32x4 A[F8R_D][2], Bv[F8R_D][MT][2];
    float sc[F8R_D][MT];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < F8R_D; ++d) {
            const int b = wave + F8R_NW * (j0 + d);
            if (b >= G) break;
            const uint32_t o = (uint32_t)(F8B * b + 16 * q), row = (uint32_t)(i * K);
            A[d][0] = f8_ld(rw, f8_off(row, o, (uint32_t)K));
            A[d][1] = f8_ld(rw, f8_off(row, o + 64, (uint32_t)K));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (XT < 0) {
                    Bv[d][m][0] = f8_ld(rx, f8_off(row + (uint32_t)(16 * m * K), o, (uint32_t)K));
                    Bv[d][m][1] = f8_ld(rx, f8_off(row + (uint32_t)(16 * m * K), o + 64, (uint32_t)K));
                    sc[d][m] = 16 * m + i < tn ? xs[(int64_t)(16 * m + i) * G + b] : 0.0f;
                }
            }
        }
    };
    load(0);
    uint8_t* xc = smem;
    float* xl = reinterpret_cast<float*>(smem + p.rows * ld);
    if constexpr (XT >= 0) {
        for (int r = 0; r < tn; ++r)
            for (int c = tid; c < tasks; c += NT) {
                float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (r == 0 && c == tid) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = xv[e];
                } else if (8 * c < K) {
                    f8_load8<XT>(xrow + (int64_t)r * K * ES, c, v);
                }
                f8_put8<XT == TSA_F32>(v, c, xc + r * ld, xl + r * G);
            }
        __syncthreads();
    }
    v4f acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (G + F8R_NW - 1) / F8R_NW;
    for (int j0 = 0; j0 < steps; j0 += F8R_D) {
        if (j0) load(j0);
#pragma unroll
        for (int d = 0; d < F8R_D; ++d) {
            const int b = wave + F8R_NW * (j0 + d);
            if (b >= G) break;
            const float s = sw[b];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (XT >= 0) {
                    Bv[d][0][0] = Bv[d][0][1] = u32x4{0, 0, 0, 0};
                    sc[d][0] = 0.0f;
                    if (i < tn) {
                        Bv[d][0][0] = *reinterpret_cast<const u32x4*>(xc + i * ld + F8B * b + 16 * q);
                        Bv[d][0][1] = *reinterpret_cast<const u32x4*>(xc + i * ld + F8B * b + 64 + 16 * q);
                        sc[d][0] = xl[i * G + b];
                    }
                }
                const v4f part = f8_mfma<WIDE>(A[d], Bv[d][m]);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(s * sc[d][m], part[r], acc[m][r]);
            }
        }
    }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // [wave][token][row]
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<v4f*>(red + ((wave * MT + m) * 16 + i) * 16 + 4 * q) = acc[m];
    __syncthreads();
    for (int o = tid; o < 256 * MT; o += NT) {
        const int64_t t = t0 + (o >> 4), n = n0 + (o & 15);
        if (t >= p.T || n >= p.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < F8R_NW; ++w) v += red[w * 256 * MT + o];
        if (p.bias) v += load_act(p.bias, p.bias_dtype, n);
        store_out(p.y, p.y_dtype, t * p.ldy + n, v);
    }
}

int f8r_lds(int xt, int mt, int G, int rows) {
    const int red = F8R_NW * 256 * mt * 4, x = xt >= 0 ? rows * (G * F8B + 16 + G * 4) : 0;
    return x > red ? x : red;
}

template <int XT, int MT>
hipError_t launch_rows(const F8Rows& p, hipStream_t st) {
    const int lds = f8r_lds(XT, MT, p.G, p.rows);
    const void* fn = p.y_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_rows_kernel<XT, MT, true>)
                                          : reinterpret_cast<const void*>(&fp8_rows_kernel<XT, MT, false>);
    const hipError_t e = ensure_dynamic_lds(fn, lds);
    if (e != hipSuccess) return e;
    // a launch ends at 2^32 threads, 2^23 of these workgroups: more rows than that go in several
    const int64_t tiles_t = (p.T + 16 * MT - 1) / (16 * MT), step = ((int64_t)1 << 22) / tiles_t * 16 / F8B * F8B;
    for (int64_t n = 0; n < p.N; n += step) {
        F8Rows q = p;
        q.N = p.N - n < step ? p.N - n : step;
        q.tiles_n = (int)((q.N + 15) / 16);
        q.w = p.w + n * p.K;
        q.ws = p.ws + n / F8B * p.G;
        if (p.bias) q.bias = static_cast<const uint8_t*>(p.bias) + n * dtype_size(p.bias_dtype);
        q.y = static_cast<uint8_t*>(p.y) + n * dtype_size(p.y_dtype);
        void* args[] = {&q};
        const hipError_t l = hipLaunchKernel(fn, dim3((unsigned)(q.tiles_n * tiles_t)), dim3(64 * F8R_NW), args, lds, st);
        if (l != hipSuccess) return l;
    }
    return hipSuccess;
}

hipError_t pick_rows(const F8Rows& p, hipStream_t st) {
    return p.T <= 16 ? launch_rows<-1, 1>(p, st) : launch_rows<-1, 2>(p, st);
}

// ---------------------------------------------------------------- many tokens
struct F8Gemm {
    const uint8_t* w;
    const float* ws;
    const uint8_t* x;
    const float* xs;
    const void* bias;
    int bias_dtype;
    void* y;
    int y_dtype;
    int T, N, K, G, tiles_t;
    int y_vec;  // y rows of whole 4-value pieces
};

template <class C, bool WIDE>
__global__ void __launch_bounds__(C::THREADS) fp8_gemm_kernel(F8Gemm p) {
    extern __shared__ __align__(16) uint8_t smem[];
    // Workgroups are dealt round the 8 XCDs by linear id: renumbered so that each XCD takes a run, and
    // within it bands of 8 row tiles, token tile by token tile (about square pieces of the product at
    // a time share one L2: 3% at 4096 x 5760 against whole rows of token tiles).
    const int total = (int)gridDim.x, wid = f8_run((int)blockIdx.x, total);
    constexpr int BAND = 8;
    const int rows = total / p.tiles_t, band = wid / (BAND * p.tiles_t), in = wid - band * BAND * p.tiles_t;
    const int deep = rows - BAND * band < BAND ? rows - BAND * band : BAND;  // row tiles of the band
    const int n0 = (BAND * band + in % deep) * C::RN, t0 = in / deep * C::TM;
    const int tn = p.T - t0 < C::TM ? p.T - t0 : C::TM;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), q = lane >> 4, i = lane & 15;
    const int wr = wave % C::WR, wt = wave / C::WR;
    const int nw = n0 + wr * C::MR * 16;  // this wave's first row; all of them are in one 128-row block
    static_assert(F8B % (C::MR * 16) == 0, "a wave's rows share their scales");
    F8Operands<1> o;
    o.w[0] = p.w + (int64_t)n0 * p.K;
    o.w_rows = p.N - n0;
    o.ws[0] = p.ws + (int64_t)(nw < p.N ? nw / F8B : 0) * p.G;  // rows past N are not stored
    o.x = p.x + (int64_t)t0 * p.K;
    o.xs = p.xs + (int64_t)t0 * p.G;
    o.x_records = (uint32_t)tn * (uint32_t)p.K;
    o.xs_records = (uint32_t)tn * (uint32_t)p.G * 4u;
    o.K = p.K;
    o.G = p.G;
    v4f acc[C::MR][C::MT];
    f8_tile<C, 1, WIDE>(o, smem, tn, [&](int r) { return r < tn ? r : -1; }, acc);
#pragma unroll
    for (int m = 0; m < C::MR; ++m) {
        const int n = nw + 16 * m + 4 * q;
        float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.bias) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < p.N) b[r] = load_act(p.bias, p.bias_dtype, n + r);
        }
#pragma unroll
        for (int t = 0; t < C::MT; ++t) {
            const int tk = 16 * (C::MT * wt + t) + i;
            if (tk >= tn || n >= p.N) continue;
            const int64_t at = (int64_t)(t0 + tk) * p.N + n;
            const v4f v = acc[m][t] + v4f{b[0], b[1], b[2], b[3]};
            if (p.y_vec && p.y_dtype == TSA_BF16) {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            } else if (p.y_vec && p.y_dtype == TSA_F32) {
                *reinterpret_cast<v4f*>(static_cast<float*>(p.y) + at) = v;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < p.N) store_out(p.y, p.y_dtype, at + r, v[r]);
            }
        }
    }
}

template <class C, bool WIDE>
hipError_t launch_gemm(const F8Gemm& p, hipStream_t st) {
    const void* fn = reinterpret_cast<const void*>(&fp8_gemm_kernel<C, WIDE>);
    const hipError_t e = ensure_dynamic_lds(fn, C::LDS);
    if (e != hipSuccess) return e;
    F8Gemm q = p;
    q.tiles_t = (p.T + C::TM - 1) / C::TM;
    void* args[] = {&q};
    const int64_t grid = (int64_t)((p.N + C::RN - 1) / C::RN) * q.tiles_t;
    return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(C::THREADS), args, C::LDS, st);
}

using TileA = F8Tile<2, 4, 8, 4, 2>;  // 256 rows x 256 tokens
using TileB = F8Tile<4, 2, 4, 4, 3>;  // 256 x 128
using TileC = F8Tile<2, 2, 4, 4, 2>;  // 128 x 128
using TileD = F8Tile<4, 1, 2, 4, 3>;  // 128 x 64
using TileE = F8Tile<4, 1, 1, 2, 4>;  // 64 x 32

// The tile (A .. E as 0 .. 4) with the least rounds x round time, a round being `per` workgroups on
// every CU; -1 if every tile needs more workgroups than a launch takes (2^32 threads).
int gemm_tile(int64_t T, int64_t N, bool wide) {
    struct Tile { int rows, tok, threads, per, cost; };
    constexpr Tile tiles[5] = {{TileA::RN, TileA::TM, TileA::THREADS, 1, 45},
                               {TileB::RN, TileB::TM, TileB::THREADS, 1, 26},
                               {TileC::RN, TileC::TM, TileC::THREADS, 2, 32},
                               {TileD::RN, TileD::TM, TileD::THREADS, 2, 20},
                               {TileE::RN, TileE::TM, TileE::THREADS, 3, 13}};
    const int64_t cus = num_cus() > 0 ? num_cus() : 256;
    int best = -1;
    int64_t least = INT64_MAX;
    for (int i = wide ? 1 : 0; i < 5; ++i) {  // 256 x 256 has no registers for the widened operands
        const int64_t wgs = (N + tiles[i].rows - 1) / tiles[i].rows * ((T + tiles[i].tok - 1) / tiles[i].tok);
        if (wgs * tiles[i].threads >= (int64_t)1 << 32) continue;
        const int64_t cost = (wgs + cus * tiles[i].per - 1) / (cus * tiles[i].per) * tiles[i].cost;
        if (cost < least) least = cost, best = i;
    }
    return best;
}

template <bool WIDE>
hipError_t pick_gemm(const F8Gemm& p, hipStream_t st) {
    switch (gemm_tile(p.T, p.N, WIDE)) {
        case 0:
            if constexpr (!WIDE) return launch_gemm<TileA, WIDE>(p, st);
            return hipErrorInvalidValue;
        case 1: return launch_gemm<TileB, WIDE>(p, st);
        case 2: return launch_gemm<TileC, WIDE>(p, st);
        case 3: return launch_gemm<TileD, WIDE>(p, st);
        default: return launch_gemm<TileE, WIDE>(p, st);
    }
}

constexpr int64_t F8_MAX_K = 1 << 20;  // 32-bit offsets inside a tile of rows

int check_matmul(int64_t T, int64_t K, int64_t N, const void* bias, int bias_dtype, int y_dtype) {
    TSA_REQUIRE(T >= 0 && N >= 1 && K >= 1, TSA_ERR_SHAPE, "bad shape (T %lld, N %lld, K %lld)", (long long)T, (long long)N,
                (long long)K);
    TSA_REQUIRE(K % 16 == 0 && K <= F8_MAX_K, TSA_ERR_SHAPE, "K (%lld) must be a multiple of 16 of at most %lld", (long long)K,
                (long long)F8_MAX_K);
    TSA_REQUIRE(T <= ((int64_t)1 << 30) && N <= ((int64_t)1 << 30) && (T <= 32 || gemm_tile(T, N, y_dtype == TSA_F32) >= 0),
                TSA_ERR_SHAPE, "T %lld x N %lld is too large", (long long)T, (long long)N);
    TSA_REQUIRE(valid_dtype(y_dtype), TSA_ERR_INVALID_ARG, "bad dtype (y %d)", y_dtype);
    TSA_REQUIRE(!bias || valid_dtype(bias_dtype), TSA_ERR_INVALID_ARG, "bad dtype (bias %d)", bias_dtype);
    return TSA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

F8Rows rows_params(const void* x, const float* xs, int64_t T, int64_t K, const void* w, const float* ws, int64_t N,
                   const void* bias, int bias_dtype, void* y, int y_dtype) {
    F8Rows p{};
    p.w = static_cast<const uint8_t*>(w);
    p.ws = ws;
    p.x = x;
    p.xs = xs;
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    p.y = y;
    p.y_dtype = y_dtype;
    p.T = T;
    p.N = N;
    p.K = (int)K;
    p.G = (int)f8_blocks(K);
    p.ldy = N;
    p.rows = (int)(T < 16 ? T : 16);
    return p;
}

}  // namespace

int fp8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
    hipError_t e;
    switch (x_dtype) {
        case TSA_F32: e = launch_quantize<TSA_F32>(x, T, K, codes, scales, st); break;
        case TSA_F16: e = launch_quantize<TSA_F16>(x, T, K, codes, scales, st); break;
        default: e = launch_quantize<TSA_BF16>(x, T, K, codes, scales, st); break;
    }
    TSA_HIP_CHECK(e);
    return TSA_OK;
}

}  // namespace tsa

using namespace tsa;

extern "C" int tsa_fp8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, void* codes, float* scales, void* stream) {
    clear_error();
    TSA_REQUIRE(valid_dtype(x_dtype), TSA_ERR_INVALID_ARG, "bad dtype (x %d)", x_dtype);
    TSA_REQUIRE(T >= 0 && K >= 1 && K < ((int64_t)1 << 31) && T * f8_blocks(K) < ((int64_t)1 << 34), TSA_ERR_SHAPE,
                "bad shape (T %lld, K %lld)", (long long)T, (long long)K);
    if (T == 0) return TSA_OK;
    TSA_REQUIRE(x && codes && scales, TSA_ERR_INVALID_ARG, "null pointer");
    return fp8_quantize(x, x_dtype, T, K, static_cast<uint8_t*>(codes), scales, as_stream(stream));
}

extern "C" int tsa_fp8_matmul(const void* codes, const float* scales, int64_t T, int64_t K, const void* w,
                              const float* w_scales, int64_t N, const void* bias, int bias_dtype, void* y, int y_dtype,
                              void* stream) {
    clear_error();
    int rc = check_matmul(T, K, N, bias, bias_dtype, y_dtype);
    if (rc) return rc;
    if (T == 0) return TSA_OK;
    TSA_REQUIRE(codes && scales && w && w_scales && y, TSA_ERR_INVALID_ARG, "null pointer");
    TSA_REQUIRE(aligned16(codes) && aligned16(w), TSA_ERR_INVALID_ARG, "the codes must be 16-byte aligned");
    if (T > 32) {
        F8Gemm p{};
        p.w = static_cast<const uint8_t*>(w);
        p.ws = w_scales;
        p.x = static_cast<const uint8_t*>(codes);
        p.xs = scales;
        p.bias = bias;
        p.bias_dtype = bias_dtype;
        p.y = y;
        p.y_dtype = y_dtype;
        p.T = (int)T;
        p.N = (int)N;
        p.K = (int)K;
        p.G = (int)f8_blocks(K);
        p.y_vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0;
        TSA_HIP_CHECK(y_dtype == TSA_F32 ? pick_gemm<true>(p, as_stream(stream)) : pick_gemm<false>(p, as_stream(stream)));
        return TSA_OK;
    }
    TSA_HIP_CHECK(pick_rows(rows_params(codes, scales, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype), as_stream(stream)));
    return TSA_OK;
}

// Whether few enough tokens are quantised inside the product's launch: the second launch costs a call that is
// made by itself about 4 us of host time, while every token here adds a load latency to every workgroup. us of
// one launch / two, 2880 x 2880 and 2048 x 4096: calls one by one, 8 tokens 7.4 / 11.2 and 8.2 / 11.6, 16 tokens
// 11.2 / 11.2 and 12.1 / 11.6; inside a graph, 4 tokens 5.3 / 5.9 and 6.1 / 7.3, 8 tokens 7.3 / 6.0 and 8.1 / 7.7,
// 16 tokens 11.4 / 6.5 and 12.2 / 9.0. (The limit is the calls' one by one; a graph's is 4 to 8.)
static bool linear_in_one(int64_t T, int64_t K) { return T <= 16 && f8r_lds(0, 1, (int)f8_blocks(K), (int)T) <= 128 * 1024; }
static int64_t linear_ws(int64_t T, int64_t K) {
    return linear_in_one(T, K) ? 0 : (T * K + 255) / 256 * 256 + T * f8_blocks(K) * 4;
}

extern "C" int tsa_fp8_linear_workspace_size(int64_t T, int64_t K, int64_t* bytes) {
    clear_error();
    TSA_REQUIRE(T >= 0 && K >= 1 && T <= ((int64_t)1 << 30) && K <= F8_MAX_K && bytes, TSA_ERR_INVALID_ARG, "bad T/K/bytes");
    *bytes = linear_ws(T, K);
    return TSA_OK;
}

extern "C" int tsa_fp8_linear(const void* x, int x_dtype, int64_t T, int64_t K, const void* w, const float* w_scales,
                              int64_t N, const void* bias, int bias_dtype, void* y, int y_dtype, void* workspace,
                              int64_t workspace_bytes, void* stream) {
    clear_error();
    TSA_REQUIRE(valid_dtype(x_dtype), TSA_ERR_INVALID_ARG, "bad dtype (x %d)", x_dtype);
    int rc = check_matmul(T, K, N, bias, bias_dtype, y_dtype);
    if (rc) return rc;
    if (T == 0) return TSA_OK;
    TSA_REQUIRE(x && w && w_scales && y, TSA_ERR_INVALID_ARG, "null pointer");
    TSA_REQUIRE(aligned16(x) && aligned16(w), TSA_ERR_INVALID_ARG, "x and the weights must be 16-byte aligned");
    hipStream_t st = as_stream(stream);
    if (linear_in_one(T, K)) {
        const F8Rows p = rows_params(x, nullptr, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype);
        const hipError_t e = x_dtype == TSA_F32 ? launch_rows<TSA_F32, 1>(p, st)
                             : x_dtype == TSA_F16 ? launch_rows<TSA_F16, 1>(p, st) : launch_rows<TSA_BF16, 1>(p, st);
        TSA_HIP_CHECK(e);
        return TSA_OK;
    }
    TSA_REQUIRE(workspace && workspace_bytes >= linear_ws(T, K), TSA_ERR_WORKSPACE,
                "workspace too small: got %lld bytes, need %lld", (long long)workspace_bytes, (long long)linear_ws(T, K));
    TSA_REQUIRE(aligned16(workspace), TSA_ERR_WORKSPACE, "the workspace must be 16-byte aligned");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* scales = reinterpret_cast<float*>(codes + (T * K + 255) / 256 * 256);
    rc = fp8_quantize(x, x_dtype, T, K, codes, scales, st);
    if (rc) return rc;
    return tsa_fp8_matmul(codes, scales, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype, stream);
}
