// FP8 quantisation of activations and the block-scaled FP8 product
//     y[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{k in block b} cx[t, k] cw[n, k]  (+ bias[n]).
#include "fp8_common.h"

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
    constexpr int ES = XT == TSA_F32 ? 4 : 2;
    const uint8_t* row = static_cast<const uint8_t*>(x) + t * K * ES;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (VEC) {
        if (8 * c < K) f8_load8<XT>(row, c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (8 * c + e < K) v[e] = load_act(row, XT, 8 * c + e);
    }
    const float s = f8_scale(f8_group_max(v));
    const uint2 o = f8_codes8<XT == TSA_F32>(v, s);
    uint8_t* dst = codes + t * K + 8 * c;
    if constexpr (VEC) {
        if (8 * c < K) *reinterpret_cast<uint2*>(dst) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (8 * c + e < K) dst[e] = (uint8_t)((e < 4 ? o.x : o.y) >> (8 * (e & 3)));
    }
    if ((task & 15) == 0) scales[g] = s;
}

template <int XT>
hipError_t launch_quantize(const void* x, int64_t T, int64_t K, uint8_t* codes, float* scales, hipStream_t st) {
    constexpr uintptr_t AL = 15;
    const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & AL) == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const dim3 grid((unsigned)((T * f8_blocks(K) * 16 + 255) / 256));
    if (vec) hipLaunchKernelGGL((fp8_quantize_kernel<XT, true>), grid, dim3(256), 0, st, x, T, (int)K, codes, scales);
    else hipLaunchKernelGGL((fp8_quantize_kernel<XT, false>), grid, dim3(256), 0, st, x, T, (int)K, codes, scales);
    return hipGetLastError();
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
    int64_t T, N;
    int K, G;
    int tiles_n, rows;  // rows: tokens of the largest tile
};

constexpr int F8R_D = 6;  // K blocks a wave has in flight

// Workgroup = 16 weight rows x 16 tokens, its NW waves take the K blocks in turn and their sums meet
// in LDS. The weights come straight into the A operand's registers (every byte is read by one lane
// of the workgroup), the tokens' codes from memory, or quantised here into LDS (XT: the dtype).
template <int XT, int NW, bool WIDE>
__global__ void __launch_bounds__(64 * NW) fp8_rows_kernel(F8Rows p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), q = lane >> 4, i = lane & 15;
    const int64_t n0 = (int64_t)(blockIdx.x % p.tiles_n) * 16, t0 = (int64_t)(blockIdx.x / p.tiles_n) * 16;
    const int tn = (int)(p.T - t0 < 16 ? p.T - t0 : 16), K = p.K, G = p.G;
    const int ld = G * F8B + 16;  // LDS row of codes
    const __amdgpu_buffer_rsrc_t rw = f8_buf(p.w + n0 * K, (p.N - n0 < 16 ? p.N - n0 : 16) * K);
    const float* sw = p.ws + n0 / F8B * G;
    u32x4 A[F8R_D][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int d = 0; d < F8R_D; ++d) {
            const uint32_t o = (uint32_t)(F8B * (wave + NW * (j0 + d)) + 16 * q);
            A[d][0] = f8_ld(rw, f8_off((uint32_t)(i * K), o, (uint32_t)K));
            A[d][1] = f8_ld(rw, f8_off((uint32_t)(i * K), o + 64, (uint32_t)K));
        }
    };
    load(0);
    uint8_t* xc = smem;
    float* xs = reinterpret_cast<float*>(smem + p.rows * ld);
    if constexpr (XT >= 0) {
        constexpr int ES = XT == TSA_F32 ? 4 : 2;
        for (int r = 0; r < tn; ++r)
            f8_stage_row<XT>(static_cast<const uint8_t*>(p.x) + (t0 + r) * K * ES, K, xc + r * ld, xs + r * G, tid, 64 * NW);
        __syncthreads();
    }
    const __amdgpu_buffer_rsrc_t rx = f8_buf(static_cast<const uint8_t*>(p.x) + t0 * K, XT >= 0 ? 0 : (int64_t)tn * K);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (G + NW - 1) / NW;
    for (int j0 = 0; j0 < steps; j0 += F8R_D) {
        if (j0) load(j0);
#pragma unroll
        for (int d = 0; d < F8R_D; ++d) {
            const int b = wave + NW * (j0 + d);
            if (b >= G) break;
            u32x4 Bv[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
            float s = sw[b];
            if constexpr (XT >= 0) {
                if (i < tn) {
                    Bv[0] = *reinterpret_cast<const u32x4*>(xc + i * ld + F8B * b + 16 * q);
                    Bv[1] = *reinterpret_cast<const u32x4*>(xc + i * ld + F8B * b + 64 + 16 * q);
                    s *= xs[i * G + b];
                }
            } else {
                const uint32_t o = (uint32_t)(F8B * b + 16 * q);
                Bv[0] = f8_ld(rx, f8_off((uint32_t)(i * K), o, (uint32_t)K));
                Bv[1] = f8_ld(rx, f8_off((uint32_t)(i * K), o + 64, (uint32_t)K));
                if (i < tn) s *= p.xs[(t0 + i) * G + b];
            }
            const v4f part = f8_mfma<WIDE>(A[d], Bv);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = fmaf(s, part[r], acc[r]);
        }
    }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // [wave][token][row]
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave * 256 + i * 16 + 4 * q + r] = acc[r];
    __syncthreads();
    if (tid < 256) {
        const int64_t t = t0 + (tid >> 4), n = n0 + (tid & 15);
        if (t < p.T && n < p.N) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += red[w * 256 + tid];
            if (p.bias) v += load_act(p.bias, p.bias_dtype, n);
            store_out(p.y, p.y_dtype, t * p.N + n, v);
        }
    }
}

int f8r_lds(int xt, int G, int rows) {
    const int red = 4 * 256 * 4, x = xt >= 0 ? rows * (G * F8B + 16 + G * 4) : 0;
    return x > red ? x : red;
}

template <int XT>
hipError_t launch_rows(const F8Rows& p, hipStream_t st) {
    const int lds = f8r_lds(XT, p.G, p.rows);
    const void* fn = p.y_dtype == TSA_F32 ? reinterpret_cast<const void*>(&fp8_rows_kernel<XT, 4, true>)
                                          : reinterpret_cast<const void*>(&fp8_rows_kernel<XT, 4, false>);
    const hipError_t e = ensure_dynamic_lds(fn, lds);
    if (e != hipSuccess) return e;
    F8Rows q = p;
    void* args[] = {&q};
    return hipLaunchKernel(fn, dim3((unsigned)(p.tiles_n * ((p.T + 15) / 16))), dim3(256), args, lds, st);
}

constexpr int64_t F8_MAX_K = 1 << 20;  // 32-bit offsets inside a tile of rows

int check_matmul(int64_t T, int64_t K, int64_t N, const void* bias, int bias_dtype, int y_dtype) {
    TSA_REQUIRE(T >= 0 && N >= 1 && K >= 1, TSA_ERR_SHAPE, "bad shape (T %lld, N %lld, K %lld)", (long long)T, (long long)N,
                (long long)K);
    TSA_REQUIRE(K % 16 == 0 && K <= F8_MAX_K, TSA_ERR_SHAPE, "K (%lld) must be a multiple of 16 of at most %lld", (long long)K,
                (long long)F8_MAX_K);
    TSA_REQUIRE(T < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && (T + 15) / 16 * ((N + 15) / 16) < ((int64_t)1 << 31),
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
    p.tiles_n = (int)((N + 15) / 16);
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
    TSA_HIP_CHECK(launch_rows<-1>(rows_params(codes, scales, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype),
                                  as_stream(stream)));
    return TSA_OK;
}

static int64_t linear_ws(int64_t T, int64_t K) { return (T * K + 255) / 256 * 256 + T * f8_blocks(K) * 4; }

extern "C" int tsa_fp8_linear_workspace_size(int64_t T, int64_t K, int64_t* bytes) {
    clear_error();
    TSA_REQUIRE(T >= 0 && K >= 1 && T < ((int64_t)1 << 31) && K <= F8_MAX_K && bytes, TSA_ERR_INVALID_ARG, "bad T/K/bytes");
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
    TSA_REQUIRE(workspace && workspace_bytes >= linear_ws(T, K), TSA_ERR_WORKSPACE,
                "workspace too small: got %lld bytes, need %lld", (long long)workspace_bytes, (long long)linear_ws(T, K));
    TSA_REQUIRE(aligned16(workspace), TSA_ERR_WORKSPACE, "the workspace must be 16-byte aligned");
    hipStream_t st = as_stream(stream);
    if (T <= 16 && f8r_lds(0, (int)f8_blocks(K), (int)T) <= 128 * 1024) {
        const F8Rows p = rows_params(x, nullptr, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype);
        TSA_HIP_CHECK(x_dtype == TSA_F32 ? launch_rows<TSA_F32>(p, st)
                                         : x_dtype == TSA_F16 ? launch_rows<TSA_F16>(p, st) : launch_rows<TSA_BF16>(p, st));
        return TSA_OK;
    }
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* scales = reinterpret_cast<float*>(codes + (T * K + 255) / 256 * 256);
    rc = fp8_quantize(x, x_dtype, T, K, codes, scales, st);
    if (rc) return rc;
    return tsa_fp8_matmul(codes, scales, T, K, w, w_scales, N, bias, bias_dtype, y, y_dtype, stream);
}
