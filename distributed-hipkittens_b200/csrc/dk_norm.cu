// Root-mean-square norm with the residual's addition, and its backward pass, for sm_100a.
//
//   r = x + residual, kept in the type of x (r = x without a residual)
//   y = r * rstd * w          rstd = 1 / sqrt(mean(r^2) + eps), one per row
//
//   dk_add_rms_norm       y in the type of x: what the bf16 GEMMs and the MoE layer read
//   dk_add_rms_norm_mx    y as MXFP8, the operand of dk_gemm_mxfp8 (same rule as dk_mx_quant)
//   dk_add_rms_norm_bwd   with n = r * rstd and g = dy * w (all sums in 32 bits):
//                             dx = dr + rstd * (g - n * mean(g * n))     (also the residual's gradient)
//                             dw = sum over rows of dy * n
//
// The rounding of r to the type of x comes BEFORE the norm: r is what is kept, so a backward pass or a
// recomputation, which have r only, see the very numbers that were normed. y is rounded once.
// All of them are bound by HBM.
#include <cuda_fp8.h>

#include "dk_host.h"
#include "dk_ptx.cuh"

namespace dk {

constexpr int NORM_THREADS = 256;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sum over the CTA, the same value in every thread and in the same order for every launch.
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // the last use of `part` is over
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += part[w];
    return s;
}

// One CTA per row: a pass that adds, keeps r and sums the squares, and a pass that writes y. A thread
// meets the same elements in both, so r_out may be the residual's or x's own buffer.
template <typename T, typename W, bool MX>
__global__ void __launch_bounds__(NORM_THREADS)
add_rms_norm_kernel(const T* __restrict__ x, const T* residual, const W* __restrict__ weight, int rows, int H, float eps,
                    T* __restrict__ y, T* r_out, float* __restrict__ rstd_out, uint8_t* __restrict__ q,
                    uint8_t* __restrict__ s_rows, uint8_t* __restrict__ atoms) {
    constexpr int STEP = MX ? 32 : 1;  // consecutive elements of a thread
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t base = static_cast<size_t>(row) * H;
        float ss = 0.f;
        for (int c = threadIdx.x * STEP; c < H; c += NORM_THREADS * STEP)
            for (int i = 0; i < STEP; ++i) {
                float v = to_f32(x[base + c + i]);
                if (residual != nullptr) {
                    const T r = from_f32<T>(v + to_f32(residual[base + c + i]));
                    r_out[base + c + i] = r;
                    v = to_f32(r);
                }
                ss += v * v;
            }
        const float rstd = 1.0f / sqrtf(block_sum(ss) / static_cast<float>(H) + eps);
        if (rstd_out != nullptr && threadIdx.x == 0) rstd_out[row] = rstd;
        const T* r = residual != nullptr ? r_out : x;
        for (int c = threadIdx.x * STEP; c < H; c += NORM_THREADS * STEP) {
            if constexpr (!MX) {
                y[base + c] = from_f32<T>(to_f32(r[base + c]) * rstd * to_f32(weight[c]));
            } else {
                float amax = 0.f;
                for (int i = 0; i < 32; ++i)
                    amax = fmaxf(amax, fabsf(to_f32(r[base + c + i]) * rstd * to_f32(weight[c + i])));
                int e = 0;
                if (amax != 0.f) {
                    int ex;
                    (void)frexpf(amax, &ex);
                    e = min(max(ex - 1 + 127, 0), 254);
                }
                const float inv = ldexpf(1.0f, 127 - e);
                for (int i = 0; i < 32; ++i)
                    q[base + c + i] = __nv_cvt_float_to_fp8(to_f32(r[base + c + i]) * rstd * to_f32(weight[c + i]) * inv,
                                                            __NV_SATFINITE, __NV_E4M3);
                const int kg = c >> 5;
                s_rows[static_cast<size_t>(row) * (H / 32) + kg] = static_cast<uint8_t>(e);
                const int rb = row >> 7, r1 = (row & 127) >> 5, r0 = row & 31;
                atoms[((static_cast<size_t>(rb) * (H / 128) + (kg >> 2)) * 32 + r0) * 16 + r1 * 4 + (kg & 3)] =
                    static_cast<uint8_t>(e);
            }
        }
    }
}

// A CTA takes every gridDim.x-th row and sums its share of dw in its row of `partial`
// [gridDim.x][H], each element by one thread in row order: the same bits on every run.
template <typename T, typename W>
__global__ void __launch_bounds__(NORM_THREADS)
add_rms_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ dr, const T* __restrict__ r,
                        const float* __restrict__ rstd_in, const W* __restrict__ weight, int rows, int H,
                        T* __restrict__ dx, float* __restrict__ partial) {
    float* mine = partial + static_cast<size_t>(blockIdx.x) * H;
    for (int c = threadIdx.x; c < H; c += NORM_THREADS) mine[c] = 0.f;
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t base = static_cast<size_t>(row) * H;
        const float rstd = rstd_in[row];
        float dot = 0.f;
        for (int c = threadIdx.x; c < H; c += NORM_THREADS) {
            const float n = to_f32(r[base + c]) * rstd, d = to_f32(dy[base + c]);
            dot += d * to_f32(weight[c]) * n;
            mine[c] += d * n;
        }
        const float mean = block_sum(dot) / static_cast<float>(H);
        for (int c = threadIdx.x; c < H; c += NORM_THREADS) {
            const float n = to_f32(r[base + c]) * rstd;
            float v = rstd * (to_f32(dy[base + c]) * to_f32(weight[c]) - n * mean);
            if (dr != nullptr) v += to_f32(dr[base + c]);
            dx[base + c] = from_f32<T>(v);
        }
    }
}

// dw[c] = sum of the CTAs' partial sums, in their order.
template <typename W>
__global__ void __launch_bounds__(NORM_THREADS)
add_rms_norm_dw_kernel(const float* __restrict__ partial, int parts, int H, W* __restrict__ dw) {
    const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
    if (c >= H) return;
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += partial[static_cast<size_t>(p) * H + c];
    dw[c] = from_f32<W>(s);
}

// --------------------------------------------------------------------------------------------
// host side

constexpr int NORM_MAX_H = 65536;
constexpr int NORM_BWD_PARTS = 296;  // CTAs of the backward pass at most: two per SM

static int check_norm(const void* x, const void* weight, int x_is_f32, int w_is_f32, int T, int H) {
    DK_REQUIRE(T >= 0, "the number of rows must not be negative");
    DK_REQUIRE(H >= 1 && H <= NORM_MAX_H, "H must be between 1 and 65536");
    DK_REQUIRE(weight != nullptr && (T == 0 || x != nullptr), "null operand");
    DK_REQUIRE(w_is_f32 || !x_is_f32, "a bf16 weight needs bf16 rows");
    return DK_OK;
}

template <bool MX>
static int launch_norm(const void* x, const void* residual, const void* weight, int x_is_f32, int w_is_f32, int T, int H,
                       float eps, void* y, void* r_out, float* rstd, void* q, void* s_rows, void* atoms, cudaStream_t st) {
    const int grid = T < (1 << 20) ? T : (1 << 20);
    auto go = [&](auto tx, auto tw) {
        using TX = decltype(tx);
        using TW = decltype(tw);
        add_rms_norm_kernel<TX, TW, MX><<<grid, NORM_THREADS, 0, st>>>(
            static_cast<const TX*>(x), static_cast<const TX*>(residual), static_cast<const TW*>(weight), T, H, eps,
            static_cast<TX*>(y), static_cast<TX*>(r_out), rstd, static_cast<uint8_t*>(q), static_cast<uint8_t*>(s_rows),
            static_cast<uint8_t*>(atoms));
    };
    if (x_is_f32) go(float{}, float{});
    else if (w_is_f32) go(__nv_bfloat16{}, float{});
    else go(__nv_bfloat16{}, __nv_bfloat16{});
    DK_CUDA_OK(cudaGetLastError());
    return DK_OK;
}

}  // namespace dk

extern "C" int dk_add_rms_norm(const void* x, const void* residual, const void* weight, int x_is_f32, int w_is_f32, int T,
                               int H, float eps, void* y, void* r_out, float* rstd, void* stream) {
    using namespace dk;
    const int rc = check_norm(x, weight, x_is_f32, w_is_f32, T, H);
    if (rc != DK_OK) return rc;
    DK_REQUIRE(eps > 0.f && eps < 1.0e30f, "eps must be positive and finite");
    if (T == 0) return DK_OK;
    DK_REQUIRE(y != nullptr, "null output");
    DK_REQUIRE((residual != nullptr) == (r_out != nullptr), "r_out goes with a residual, and a residual with r_out");
    return launch_norm<false>(x, residual, weight, x_is_f32, w_is_f32, T, H, eps, y, r_out, rstd, nullptr, nullptr, nullptr,
                              static_cast<cudaStream_t>(stream));
}

extern "C" int dk_add_rms_norm_mx(const void* x, const void* residual, const void* weight, int x_is_f32, int w_is_f32, int T,
                                  int H, float eps, void* q, void* s_rows, void* sf_atoms, void* r_out, void* stream) {
    using namespace dk;
    const int rc = check_norm(x, weight, x_is_f32, w_is_f32, T, H);
    if (rc != DK_OK) return rc;
    DK_REQUIRE(eps > 0.f && eps < 1.0e30f, "eps must be positive and finite");
    DK_REQUIRE(H % 128 == 0, "H must be a multiple of 128");
    if (T == 0) return DK_OK;
    DK_REQUIRE(q != nullptr && s_rows != nullptr && sf_atoms != nullptr, "null output");
    DK_REQUIRE((residual != nullptr) == (r_out != nullptr), "r_out goes with a residual, and a residual with r_out");
    DK_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(s_rows) | reinterpret_cast<uintptr_t>(sf_atoms)) & 15) == 0,
               "q, s_rows and sf_atoms must be 16-byte aligned");
    // rows of the last 128-row block that do not exist get scale byte 0
    if (T % 128 != 0)
        DK_CUDA_OK(cudaMemsetAsync(static_cast<uint8_t*>(sf_atoms) + static_cast<size_t>(T / 128) * (H / 128) * 512, 0,
                                   static_cast<size_t>(H / 128) * 512, static_cast<cudaStream_t>(stream)));
    return launch_norm<true>(x, residual, weight, x_is_f32, w_is_f32, T, H, eps, nullptr, r_out, nullptr, q, s_rows, sf_atoms,
                             static_cast<cudaStream_t>(stream));
}

extern "C" size_t dk_add_rms_norm_bwd_workspace_bytes(int T, int H) {
    using namespace dk;
    if (T < 0 || H < 1 || H > NORM_MAX_H) return 0;
    return static_cast<size_t>(T < NORM_BWD_PARTS ? T : NORM_BWD_PARTS) * H * sizeof(float);
}

extern "C" int dk_add_rms_norm_bwd(const void* dy, const void* dr, const void* r, const float* rstd, const void* weight,
                                   int x_is_f32, int w_is_f32, int T, int H, void* dx, void* dw, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    using namespace dk;
    const int rc = check_norm(r, weight, x_is_f32, w_is_f32, T, H);
    if (rc != DK_OK) return rc;
    DK_REQUIRE(dw != nullptr, "null output");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        DK_CUDA_OK(cudaMemsetAsync(dw, 0, static_cast<size_t>(H) * (w_is_f32 ? 4 : 2), st));
        return DK_OK;
    }
    DK_REQUIRE(dy != nullptr && rstd != nullptr, "null operand");
    DK_REQUIRE(dx != nullptr, "null output");
    DK_REQUIRE(workspace != nullptr && workspace_bytes >= dk_add_rms_norm_bwd_workspace_bytes(T, H), "workspace too small");
    DK_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
    const int parts = T < NORM_BWD_PARTS ? T : NORM_BWD_PARTS;
    float* partial = static_cast<float*>(workspace);
    auto go = [&](auto tx, auto tw) {
        using TX = decltype(tx);
        using TW = decltype(tw);
        add_rms_norm_bwd_kernel<TX, TW><<<parts, NORM_THREADS, 0, st>>>(
            static_cast<const TX*>(dy), static_cast<const TX*>(dr), static_cast<const TX*>(r), rstd,
            static_cast<const TW*>(weight), T, H, static_cast<TX*>(dx), partial);
        add_rms_norm_dw_kernel<TW><<<(H + NORM_THREADS - 1) / NORM_THREADS, NORM_THREADS, 0, st>>>(partial, parts, H,
                                                                                                  static_cast<TW*>(dw));
    };
    if (x_is_f32) go(float{}, float{});
    else if (w_is_f32) go(__nv_bfloat16{}, float{});
    else go(__nv_bfloat16{}, __nv_bfloat16{});
    DK_CUDA_OK(cudaGetLastError());
    return DK_OK;
}
