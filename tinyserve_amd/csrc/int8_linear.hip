// int8 quantisation of activations and the int8 product
//     y[t, n] = sx[t] sw[n] sum_k cx[t, k] cw[n, k]  (+ bias[n]),
// a float32 scale for each token and each weight row. The sum is exact (int32; K is bounded for it); it is
// rounded to float32 once, and once more times the scales' product.
#include "int8_common.h"
#include "mm_epilogue.h"

namespace tsa {
namespace {

// ---------------------------------------------------------------- quantisation
template <int XT, bool VEC, int W>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const uint8_t* __restrict__ x, int64_t T, int64_t K,
                                                            uint8_t* __restrict__ codes, float* __restrict__ scales) {
    __shared__ uint32_t top[4];
    constexpr int ES = XT == TSA_F32 ? 4 : 2, D = W == 1 ? 8 : 2;
    const int g = (int)threadIdx.x / (64 * W);
    const int64_t t = (int64_t)blockIdx.x * (4 / W) + g;
    if (W == 1 && t >= T) return;
    const int tid = (int)threadIdx.x - 64 * W * g;
    I8Raw<XT> v[D];
    i8_row_load<XT, VEC, W, D>(x + t * K * ES, K, tid, v);
    const float s = i8_row_codes<XT, VEC, W, D>(x + t * K * ES, K, tid, v, codes + t * K, top + W * g);
    if (tid == 0) scales[t] = s;
}

template <int XT, bool VEC>
hipError_t launch_quantize(const void* x, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
    const uint8_t* xb = static_cast<const uint8_t*>(x);
    constexpr int64_t STEP = (int64_t)1 << 25;  // rows of a launch, which ends at 2^32 threads
    for (int64_t t = 0; t < T; t += STEP) {
        const int64_t n = T - t < STEP ? T - t : STEP;
        const uint8_t* xt = xb + t * K * (XT == TSA_F32 ? 4 : 2);
        if (n < 1024) hipLaunchKernelGGL((int8_quantize_kernel<XT, VEC, 4>), dim3((unsigned)n), dim3(256), 0, st, xt, n, K, codes + t * K, scales + t);
        else hipLaunchKernelGGL((int8_quantize_kernel<XT, VEC, 1>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, xt, n, K, codes + t * K, scales + t);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int XT>
hipError_t launch_quantize(const void* x, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
    const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    return vec ? launch_quantize<XT, true>(x, T, K, codes, scales, st) : launch_quantize<XT, false>(x, T, K, codes, scales, st);
}

// ---------------------------------------------------------------- few tokens
struct I8Rows {
    const uint8_t* w;
    const float* ws;
    const void* x;    // codes (XT -1) or values
    const float* xs;  // codes: their scales
    MmOut out;
    int64_t T, N;
    int K, tiles_n, rows;  // rows: tokens of the largest tile
};

constexpr int I8R_NW = 8, I8R_D = 4;  // waves; steps of 128 columns a wave has in flight

// Workgroup = 16 weight rows x 16 MT tokens; its waves take the steps of 128 columns in turn and their sums
// meet in LDS. The weights come straight into the A operand's registers (every byte is read by one lane of
// the workgroup), the tokens' codes from memory, or (XT: their dtype, up to 16 tokens) quantised here
// into LDS while the weights are on their way.
template <int XT, int MT, int HELD>
__global__ void __launch_bounds__(64 * I8R_NW, 4) int8_rows_kernel(I8Rows p) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int NT = 64 * I8R_NW;
    static_assert(XT < 0 || MT == 1, "one token tile is quantised here");
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const int wid = xcd_run((int)blockIdx.x, (int)gridDim.x), tt = (int)gridDim.x / p.tiles_n;
    const int64_t n0 = (int64_t)(wid / tt) * 16, t0 = (int64_t)(wid % tt) * (16 * MT);
    const int tn = (int)(p.T - t0 < 16 * MT ? p.T - t0 : 16 * MT), K = p.K;
    const int steps = (K + MMB - 1) / MMB, ld = steps * MMB + 16;  // LDS row of codes
    const uint8_t* xrow = static_cast<const uint8_t*>(p.x) + t0 * K * (XT < 0 ? 1 : ES);
    const __amdgpu_buffer_rsrc_t rw = f8_buf(p.w + n0 * K, (p.N - n0 < 16 ? p.N - n0 : 16) * K);
    const __amdgpu_buffer_rsrc_t rx = f8_buf(xrow, XT >= 0 ? 0 : (int64_t)tn * K);
    u32x4 A[I8R_D][2], Bv[I8R_D][MT][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < I8R_D; ++d) {
            const int b = wave + I8R_NW * (j0 + d);
            if (b >= steps) break;
            const uint32_t o = (uint32_t)(MMB * b + 16 * q), row = (uint32_t)(i * K);
            A[d][0] = f8_ld(rw, f8_off(row, o, (uint32_t)K));
            A[d][1] = f8_ld(rw, f8_off(row, o + 64, (uint32_t)K));
            if constexpr (XT < 0) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    Bv[d][m][0] = f8_ld(rx, f8_off(row + (uint32_t)(16 * m * K), o, (uint32_t)K));
                    Bv[d][m][1] = f8_ld(rx, f8_off(row + (uint32_t)(16 * m * K), o + 64, (uint32_t)K));
                }
            }
        }
    };
    uint8_t* xc = smem;
    float* xl = reinterpret_cast<float*>(smem + p.rows * ld);  // [token]: the scales
    if constexpr (XT >= 0) {
        // 8 / `many` waves a token, pieces of 512 values in turn; the first HELD are held from the search of the maximum on
        const int many = tn > 4 ? 8 : tn > 2 ? 4 : tn, per = I8R_NW / many, sub = wave % per, pieces = (K + 511) / 512;
        for (int r0 = 0; r0 < tn; r0 += many) {  // workgroup-uniform; one turn where waves share a token
            const int r = r0 + wave / per;
            const uint8_t* row = xrow + (int64_t)(r < tn ? r : 0) * K * ES;
            const int64_t len = r < tn ? K : 0;
            I8Raw<XT> v[HELD];
#pragma unroll
            for (int h = 0; h < HELD; ++h) v[h] = i8_load<XT, true>(row, len, 64 * (sub + per * h) + lane);
            if (r0 == 0) load(0);
            uint32_t m = 0;
#pragma unroll
            for (int h = 0; h < HELD; ++h) m = i8_max<XT>(v[h], m);
            for (int u = sub + per * HELD; u < pieces; u += per) m = i8_max<XT>(i8_load<XT, true>(row, len, 64 * u + lane), m);
            m = wave_max_u32(m);
            if (per > 1) {
                uint32_t* top = reinterpret_cast<uint32_t*>(xl + 16);
                if (lane == 0) top[wave] = m;
                __syncthreads();
                for (int w = 0; w < per; ++w) m = max(m, top[wave - sub + w]);
            }
            if (r >= tn) continue;
            const float s = i8_scale(i8_max_f32<XT>(m));
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int c = 64 * (sub + per * h) + lane;
                if (8 * c < steps * MMB) *reinterpret_cast<uint2*>(xc + r * ld + 8 * c) = i8_codes8<XT>(v[h], s);
            }
            for (int u = sub + per * HELD; u < pieces; u += per) {
                const int c = 64 * u + lane;
                if (8 * c < steps * MMB) *reinterpret_cast<uint2*>(xc + r * ld + 8 * c) = i8_codes8<XT>(i8_load<XT, true>(row, len, c), s);
            }
            if (lane == 0 && sub == 0) xl[r] = s;
        }
        __syncthreads();
    } else {
        load(0);
    }
    v4i acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = v4i{0, 0, 0, 0};
    for (int j0 = 0; j0 < (steps + I8R_NW - 1) / I8R_NW; j0 += I8R_D) {
        if (j0) load(j0);
#pragma unroll
        for (int d = 0; d < I8R_D; ++d) {
            const int b = wave + I8R_NW * (j0 + d);
            if (b >= steps) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (XT >= 0) {
                        Bv[d][0][h] = u32x4{0, 0, 0, 0};
                        if (i < tn) Bv[d][0][h] = *reinterpret_cast<const u32x4*>(xc + i * ld + MMB * b + 64 * h + 16 * q);
                    }
                    acc[m] = MmI8::mfma(A[d][h], Bv[d][m][h], acc[m]);
                }
        }
    }
    float sc[MT];  // the scales of this thread's tokens: read before LDS is used again
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int t = (tid + NT * m) >> 4;  // of output tid + NT m, below
        if constexpr (XT >= 0) sc[m] = t < tn ? xl[t] : 0.0f;
        else sc[m] = t < tn ? p.xs[t0 + t] : 0.0f;
    }
    __syncthreads();
    int* red = reinterpret_cast<int*>(smem);  // [wave][token][row]
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<v4i*>(red + ((wave * MT + m) * 16 + i) * 16 + 4 * q) = acc[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int o = tid + NT * m;  // 256 MT outputs
        const int64_t t = t0 + (o >> 4), n = n0 + (o & 15);
        if (o >= 256 * MT || t >= p.T || n >= p.N) continue;
        int v = 0;
#pragma unroll
        for (int w = 0; w < I8R_NW; ++w) v += red[w * 256 * MT + o];
        float y = (float)v * (sc[m] * p.ws[n]);
        if (p.out.bias) y += load_act(p.out.bias, p.out.bias_dtype, n);
        store_out(p.out.y, p.out.y_dtype, t * p.out.ldy + n, y);
    }
}

int i8r_lds(int xt, int mt, int64_t K, int rows) {
    const int red = I8R_NW * 256 * mt * 4, x = xt >= 0 ? rows * (int)((K + MMB - 1) / MMB * MMB + 16) + 128 : 0;
    return x > red ? x : red;
}

template <int XT, int MT, int HELD>
hipError_t launch_rows(const I8Rows& p, hipStream_t st) {
    const int lds = i8r_lds(XT, MT, p.K, p.rows);
    const void* fn = reinterpret_cast<const void*>(&int8_rows_kernel<XT, MT, HELD>);
    const hipError_t e = ensure_dynamic_lds(fn, lds);
    if (e != hipSuccess) return e;
    // a launch ends at 2^32 threads, 2^23 of these workgroups: more rows than that go in several
    const int64_t tiles_t = (p.T + 16 * MT - 1) / (16 * MT), step = ((int64_t)1 << 22) / tiles_t * 16;
    for (int64_t n = 0; n < p.N; n += step) {
        I8Rows q = p;
        q.N = p.N - n < step ? p.N - n : step;
        q.tiles_n = (int)((q.N + 15) / 16);
        q.w = p.w + n * p.K;
        q.ws = p.ws + n;
        if (p.out.bias) q.out.bias = static_cast<const uint8_t*>(p.out.bias) + n * dtype_size(p.out.bias_dtype);
        q.out.y = static_cast<uint8_t*>(p.out.y) + n * dtype_size(p.out.y_dtype);
        void* args[] = {&q};
        const hipError_t l = hipLaunchKernel(fn, dim3((unsigned)(q.tiles_n * tiles_t)), dim3(64 * I8R_NW), args, lds, st);
        if (l != hipSuccess) return l;
    }
    return hipSuccess;
}

// Quantised inside: two pieces a wave held for the fewest tokens, else eight (of float32 values four; more are read twice).
template <int XT>
hipError_t launch_linear(const I8Rows& p, hipStream_t st) {
    const int per = I8R_NW / (p.T > 4 ? 8 : p.T > 2 ? 4 : (int)p.T), pieces = (p.K + 511) / 512;
    return pieces <= 2 * per ? launch_rows<XT, 1, 2>(p, st) : launch_rows<XT, 1, XT == TSA_F32 ? 4 : 8>(p, st);
}

// ---------------------------------------------------------------- many tokens
struct I8Gemm {
    const uint8_t* w;
    const float* ws;
    const uint8_t* x;
    const float* xs;
    MmOut out;
    int T, N, K, tiles_n, tiles_t;
};

// The product's tiles in bands of 8 row tiles, token tile by token tile (about square pieces of the product at a time
// share an XCD's L2).
template <class C>
struct I8Work {
    const I8Gemm& p;
    MmRuns runs;
    int n0, t0, tn, next_n0, next_t0, next_tn;
    __device__ __forceinline__ explicit I8Work(const I8Gemm& p) : p(p), runs(p.tiles_n * p.tiles_t) {}
    __device__ __forceinline__ bool next() {
        if (!runs.next()) return false;
        constexpr int BAND = 8;
        const int band = runs.at / (BAND * p.tiles_t), in = runs.at - band * BAND * p.tiles_t;
        const int deep = p.tiles_n - BAND * band < BAND ? p.tiles_n - BAND * band : BAND;  // row tiles of the band
        next_n0 = (BAND * band + in % deep) * C::RN;
        next_t0 = in / deep * C::TM;
        next_tn = p.T - next_t0 < C::TM ? p.T - next_t0 : C::TM;
        return true;
    }
    __device__ __forceinline__ MmOperands<1> operands() const {
        return MmOperands<1>{{p.w + (int64_t)next_n0 * p.K}, p.N - next_n0, p.x + (int64_t)next_t0 * p.K, (uint32_t)next_tn * (uint32_t)p.K, next_tn};
    }
    __device__ __forceinline__ void take() { n0 = next_n0, t0 = next_t0, tn = next_tn; }
    __device__ __forceinline__ void store(const v4i (&acc)[C::MR][C::MT], uint8_t* out) const {
        mm_store<C>(acc, p.out, out, n0, p.N, tn, [&](int r) { return (int64_t)(t0 + r); }, [&](int r) { return p.xs[t0 + r]; }, p.ws);
    }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS) int8_gemm_kernel(I8Gemm p) {
    extern __shared__ __align__(16) uint8_t smem[];
    I8Work<C> work(p);
    mm_run<C, MmI8, 1, false>(work, (uint32_t)p.K, smem);
}

template <class C>
hipError_t launch_gemm(const I8Gemm& p, int per, hipStream_t st) {
    const void* fn = reinterpret_cast<const void*>(&int8_gemm_kernel<C>);
    const hipError_t e = ensure_dynamic_lds(fn, C::LDS);
    if (e != hipSuccess) return e;
    I8Gemm q = p;
    q.tiles_n = (p.N + C::RN - 1) / C::RN;
    q.tiles_t = (p.T + C::TM - 1) / C::TM;
    void* args[] = {&q};
    return hipLaunchKernel(fn, dim3(mm_grid((int64_t)q.tiles_n * q.tiles_t, per)), dim3(C::THREADS), args, C::LDS, st);
}

using TileA = MmTile<4, 2, 4, 8, 2>;  // 256 rows x 256 tokens
using TileB = MmTile<4, 2, 4, 4, 3>;  // 256 x 128
using TileC = MmTile<2, 2, 4, 4, 2>;  // 128 x 128
using TileD = MmTile<4, 1, 2, 4, 3>;  // 128 x 64

// The tile (A .. D as 0 .. 3) with the least time, where a CU that works on 1 .. `per` tiles at once takes cost[0 .. per - 1]
// for them, and on more in rounds; -1 if every tile gives 2^30 of them or more. (us of a product of K 2880 to 4096. Over the shapes of N 512
// to 8192 and 33 to 8192 tokens that were measured: within 6% of the best tile but for a few of fewer than 100 tokens. K scales
// all four alike but for what a tile costs apart from its steps; other K were not measured.)
struct GemmTile { int rows, tok, per, cost[2]; };
constexpr GemmTile gemm_tiles[4] = {{TileA::RN, TileA::TM, 1, {43}},
                                    {TileB::RN, TileB::TM, 1, {25}},
                                    {TileC::RN, TileC::TM, 2, {21, 28}},
                                    {TileD::RN, TileD::TM, 2, {14, 20}}};

// The tile, and its time.
int gemm_tile(int64_t T, int64_t N, int64_t* time = nullptr) {
    const int64_t cus = num_cus() > 0 ? num_cus() : 256;
    int best = -1;
    int64_t least = INT64_MAX;
    for (int i = 0; i < 4; ++i) {
        const GemmTile& t = gemm_tiles[i];
        const int64_t tiles = (N + t.rows - 1) / t.rows * ((T + t.tok - 1) / t.tok), on = (tiles + cus - 1) / cus;
        if (tiles >= (int64_t)1 << 30) continue;
        const int64_t cost = on / t.per * t.cost[t.per - 1] + (on % t.per ? t.cost[on % t.per - 1] : 0);
        if (cost < least) least = cost, best = i;
    }
    if (time) *time = least;
    return best;
}

// Whether the row kernel takes a product: up to 32 tokens, and more while its rounds of 16 rows x 32 tokens on every CU take
// less than the tiles. us of the row kernel / the tiles, weights from memory: 2880 x 2880, 64 / 128 / 192 tokens 8.3 / 16.8, 10.9 /
// 17.0 and 15.4 / 15.4; 2048 x 4096, 128 / 192 / 256 14.1 / 21.8, 19.3 / 21.8 and 24.4 / 21.9; 5760 x 2880, 64 / 96 / 128 10.9 / 17.0,
// 15.5 / 15.6 and 17.8 / 15.5; 512 x 2048, 512 tokens 8.3 / 12.9. (Past 2^20 tokens, where one 16-row tile's workgroups would near a launch's
// limit, the tiles always.)
bool rows_kernel(int64_t T, int64_t N) {
    if (T <= 32 || T > 1 << 20) return T <= 32;
    const int64_t cus = num_cus() > 0 ? num_cus() : 256, on = ((N + 15) / 16 * ((T + 31) / 32) + cus - 1) / cus;
    int64_t time;
    return gemm_tile(T, N, &time) >= 0 && 3 + 3 * on <= time;
}

hipError_t pick_gemm(const I8Gemm& p, hipStream_t st) {
    const int i = gemm_tile(p.T, p.N), per = gemm_tiles[i].per;
    switch (i) {
        case 0: return launch_gemm<TileA>(p, per, st);
        case 1: return launch_gemm<TileB>(p, per, st);
        case 2: return launch_gemm<TileC>(p, per, st);
        default: return launch_gemm<TileD>(p, per, st);
    }
}

int check_matmul(int64_t T, int64_t K, int64_t N, const void* bias, int bias_dtype, int y_dtype) {
    TSA_REQUIRE(T >= 0 && N >= 1 && K >= 1, TSA_ERR_SHAPE, "bad shape (T %lld, N %lld, K %lld)", (long long)T, (long long)N,
                (long long)K);
    TSA_REQUIRE(K % 16 == 0 && K <= I8_MAX_K, TSA_ERR_SHAPE, "K (%lld) must be a multiple of 16 of at most %lld", (long long)K,
                (long long)I8_MAX_K);
    TSA_REQUIRE(T <= ((int64_t)1 << 30) && N <= ((int64_t)1 << 30) && (T <= 32 || gemm_tile(T, N) >= 0), TSA_ERR_SHAPE,
                "T %lld x N %lld is too large", (long long)T, (long long)N);
    TSA_REQUIRE(valid_dtype(y_dtype), TSA_ERR_INVALID_ARG, "bad dtype (y %d)", y_dtype);
    TSA_REQUIRE(!bias || valid_dtype(bias_dtype), TSA_ERR_INVALID_ARG, "bad dtype (bias %d)", bias_dtype);
    return TSA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

I8Rows rows_params(const void* x, const float* xs, int64_t T, int64_t K, const void* w, const float* ws, int64_t N, const MmOut& out) {
    I8Rows p{};
    p.w = static_cast<const uint8_t*>(w);
    p.ws = ws;
    p.x = x;
    p.xs = xs;
    p.out = out;
    p.T = T;
    p.N = N;
    p.K = (int)K;
    p.rows = (int)(T < 16 ? T : 16);
    return p;
}

}  // namespace

int i8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
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

extern "C" int tsa_int8_quantize(const void* x, int x_dtype, int64_t T, int64_t K, void* codes, float* scales, void* stream) {
    clear_error();
    TSA_REQUIRE(valid_dtype(x_dtype), TSA_ERR_INVALID_ARG, "bad dtype (x %d)", x_dtype);
    TSA_REQUIRE(T >= 0 && K >= 1 && K < ((int64_t)1 << 31) && T <= ((int64_t)1 << 30), TSA_ERR_SHAPE, "bad shape (T %lld, K %lld)",
                (long long)T, (long long)K);
    if (T == 0) return TSA_OK;
    TSA_REQUIRE(x && codes && scales, TSA_ERR_INVALID_ARG, "null pointer");
    return i8_quantize(x, x_dtype, T, K, static_cast<uint8_t*>(codes), scales, as_stream(stream));
}

extern "C" int tsa_int8_matmul(const void* codes, const float* scales, int64_t T, int64_t K, const void* w,
                               const float* w_scales, int64_t N, const void* bias, int bias_dtype, void* y, int y_dtype,
                               void* stream) {
    clear_error();
    int rc = check_matmul(T, K, N, bias, bias_dtype, y_dtype);
    if (rc) return rc;
    if (T == 0) return TSA_OK;
    TSA_REQUIRE(codes && scales && w && w_scales && y, TSA_ERR_INVALID_ARG, "null pointer");
    TSA_REQUIRE(aligned16(codes) && aligned16(w), TSA_ERR_INVALID_ARG, "the codes must be 16-byte aligned");
    const MmOut out = mm_out(y, y_dtype, N, bias, bias_dtype);
    if (!rows_kernel(T, N)) {
        I8Gemm p{};
        p.w = static_cast<const uint8_t*>(w);
        p.ws = w_scales;
        p.x = static_cast<const uint8_t*>(codes);
        p.xs = scales;
        p.out = out;
        p.T = (int)T;
        p.N = (int)N;
        p.K = (int)K;
        TSA_HIP_CHECK(pick_gemm(p, as_stream(stream)));
        return TSA_OK;
    }
    const I8Rows p = rows_params(codes, scales, T, K, w, w_scales, N, out);
    TSA_HIP_CHECK(T <= 16 ? (launch_rows<-1, 1, 0>(p, as_stream(stream))) : (launch_rows<-1, 2, 0>(p, as_stream(stream))));
    return TSA_OK;
}

// Whether few enough tokens are quantised inside the product's launch: the second launch costs a call that is made by
// itself 3.3 us of host time (9.7 to 10 us, whatever the sizes), while every group of 8 tokens here adds a load latency and
// its arithmetic to every workgroup. us of one launch / two: calls one by one, 2880 x 2880, 2048 x 4096 and 5760 x 2880, 8 tokens
// 6.3, 7.2 and 8.0 / 9.7, 12 tokens 7.0, 8.0 and 9.6 / 9.7, 16 tokens 8.0, 9.3 and 10.9 / 9.8; inside a graph, 8 tokens 7.0, 8.0 and
// 8.8 / 7.1, 8.7 and 8.9, 12 tokens 7.8, 8.9 and 10.5 / 7.3, 9.1 and 9.1. The rule goes by calls made one by one: inside a graph it costs
// up to 1.4 us at 12 tokens.
static bool linear_in_one(int64_t T, int64_t K) { return T <= 12 && i8r_lds(0, 1, K, (int)T) <= 128 * 1024; }
static int64_t linear_ws(int64_t T, int64_t K) { return linear_in_one(T, K) ? 0 : (T * K + 255) / 256 * 256 + T * 4; }

extern "C" int tsa_int8_linear_workspace_size(int64_t T, int64_t K, int64_t* bytes) {
    clear_error();
    TSA_REQUIRE(T >= 0 && K >= 1 && T <= ((int64_t)1 << 30) && K <= I8_MAX_K && bytes, TSA_ERR_INVALID_ARG, "bad T/K/bytes");
    *bytes = linear_ws(T, K);
    return TSA_OK;
}

extern "C" int tsa_int8_linear(const void* x, int x_dtype, int64_t T, int64_t K, const void* w, const float* w_scales,
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
        const I8Rows p = rows_params(x, nullptr, T, K, w, w_scales, N, mm_out(y, y_dtype, N, bias, bias_dtype));
        TSA_HIP_CHECK(x_dtype == TSA_F32 ? launch_linear<TSA_F32>(p, st)
                      : x_dtype == TSA_F16 ? launch_linear<TSA_F16>(p, st) : launch_linear<TSA_BF16>(p, st));
        return TSA_OK;
    }
    TSA_REQUIRE(workspace && workspace_bytes >= linear_ws(T, K), TSA_ERR_WORKSPACE,
                "workspace too small: got %lld bytes, need %lld", (long long)workspace_bytes, (long long)linear_ws(T, K));
    TSA_REQUIRE(aligned16(workspace), TSA_ERR_WORKSPACE, "the workspace must be 16-byte aligned");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* scales = reinterpret_cast<float*>(codes + (T * K + 255) / 256 * 256);
    rc = i8_quantize(x, x_dtype, T, K, codes, scales, st);
    if (rc) return rc;
    return tsa_int8_matmul(codes, scales, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype, stream);
}
