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
#include "dk_launch.cuh"
#include "dk_ptx.cuh"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace dk {

constexpr int NORM_THREADS = 256;  // of the kernels that loop over wide rows

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as they lie in memory, a multiple of 16 bytes.
template <typename T, int V>
struct Pack {
    static constexpr int N16 = V * static_cast<int>(sizeof(T)) / 16;
    static_assert(N16 > 0 && V * sizeof(T) % 16 == 0, "whole 16-byte vectors");
    union {
        uint4 v[N16];
        T e[V];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N16; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < N16; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N16; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
    }
};

// The vectors of a row and the threads that have them: vector i begins at element i * V - shift of the row. Where every row
// starts on 16 bytes (RAGGED == false) shift is 0 and vectors are whole. Otherwise rows start `shift` elements behind a
// 16-byte boundary, their first and last vectors are partial (done element by element), all others are whole all the same.
// Element r * H lies (r * H) % V behind a boundary; a CTA's rows are a multiple of V apart, so shift is the same for all of
// them and what a thread keeps (the weight, its columns of dw) stays in place.
template <int V, bool RAGGED>
struct RowVectors {
    int H, shift, count;
    __device__ __forceinline__ RowVectors(int first_row, int H_) : H(H_) {
        shift = RAGGED ? static_cast<int>(static_cast<int64_t>(first_row) * H_ % V) : 0;
        count = RAGGED ? (H + shift + V - 1) / V : H / V;
    }
    __device__ __forceinline__ bool whole(int i) const { return !RAGGED || (i * V >= shift && (i + 1) * V - shift <= H); }
    __device__ __forceinline__ bool has(int i, int k) const {
        const int c = i * V + k - shift;
        return !RAGGED || (c >= 0 && c < H);
    }
    // `row`: the row's first element
    template <typename T>
    __device__ __forceinline__ void load(Pack<T, V>& p, const T* row, int i) const {
        const T* at = row + (static_cast<int64_t>(i) * V - shift);
        if (whole(i)) {
            p.load(at);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (has(i, k)) p.e[k] = at[k];
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(const Pack<T, V>& p, T* row, int i) const {
        T* at = row + (static_cast<int64_t>(i) * V - shift);
        if (whole(i)) {
            p.store(at);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (has(i, k)) at[k] = p.e[k];
        }
    }
    // the weight lies on a boundary whatever the row does
    template <typename W>
    __device__ __forceinline__ void load_weight(Pack<W, V>& p, const W* weight, int i) const {
        if constexpr (!RAGGED) {
            p.load(weight + static_cast<int64_t>(i) * V);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (has(i, k)) p.e[k] = weight[i * V + k - shift];
        }
    }
};

// a + b, rounded once. Pairs of bf16 are added as such: the fp32 sum of two bf16 values, rounded to bf16, is the same
// (what fp32 cannot hold of the smaller one lies below a 2^-8 part of the last place of bf16).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> added(const Pack<T, V>& a, const Pack<T, V>& b) {
    Pack<T, V> r;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            reinterpret_cast<__nv_bfloat162*>(r.e)[i] =
                __hadd2(reinterpret_cast<const __nv_bfloat162*>(a.e)[i], reinterpret_cast<const __nv_bfloat162*>(b.e)[i]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) r.e[k] = from_f32<T>(to_f32(a.e[k]) + to_f32(b.e[k]));
    }
    return r;
}

// Sum over the threads that share a row (a warp, or the first `threads` of the CTA), the same value in every one of
// them and in the same order on every run. `part` is used in turn by consecutive calls (which = 0, 1, 0, ...), so that
// one barrier a call is enough: between two uses of a half lies the barrier of the other.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float (&part)[2][32], int which, int threads) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (WARP) return v;
    if ((threadIdx.x & 31) == 0) part[which][threadIdx.x >> 5] = v;
    named_bar_sync(1, threads);
    float s = 0.f;
    for (int w = 0; w < (threads >> 5); ++w) s += part[which][w];
    return s;
}

// How the values of a row reach the threads of a backward pass.
//   FROM_REGS   each thread loads its own 16-byte vectors, those of the next row as soon as it has added
//               up this row's: they are in flight during the reduction and the writing
//   FROM_WARP   the same, a row to a warp: no barrier
//   FROM_RING   one thread has whole rows copied into a ring in shared memory (cp.async.bulk), as many rows ahead as
//               fit: up to 200 KB in flight on an SM instead of what registers hold (8192 rows of 7168: 97 -> 80 us)
// The forward pass stays with registers and two CTAs an SM: half the arrays and more arithmetic after the reduction, so
// more warps are worth more than bytes in flight (a ring took 203 us instead of 182 for 16384 rows of 8192 with two CTAs,
// 181 with one; 311 and 402 instead of 302 for 32768 rows of 7168 to MXFP8).
enum : int { FROM_REGS = 0, FROM_WARP = 1, FROM_RING = 2 };
constexpr int RING_STAGES = 12;
constexpr int RING_SM_BYTES = 200 * 1024;  // rings of all CTAs of an SM
enum : unsigned { SITE_NORM_ROW = 121 };
struct Ring {
    int stages, stage_bytes;  // a stage: the CTA's row of each array
    unsigned* status;
};
struct RingShared {
    uint64_t full[RING_STAGES];
    int abort;
};
// The CTA's rows first, first + stride, ... of `n` arrays, a stage each. There is no barrier for empty stages: a thread
// takes all it needs of a row into registers before the row's reduction, and the reduction's barrier then frees the stage.
template <typename T, int N>
struct RowRing {
    RingShared& sh;
    const Ring ring;
    uint8_t* smem;
    const T* const (&src)[N];
    int n, stride, rows, H;
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void copy(int s, int row) {  // one thread
        const uint32_t full = smem_u32(&sh.full[s]), bytes = static_cast<uint32_t>(H) * sizeof(T);
        mbar_expect_tx(full, n * bytes);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n)
                bulk_load_1d(smem_u32(smem) + s * ring.stage_bytes + i * bytes, src[i] + static_cast<size_t>(row) * H, bytes,
                             full);
    }
    __device__ __forceinline__ void start(int first) {
        if (threadIdx.x == 0) {
            sh.abort = 0;
            for (int i = 0; i < ring.stages; ++i) mbar_init(smem_u32(&sh.full[i]), 1);
            fence_mbar_init();
            for (int i = 0; i < ring.stages && first + static_cast<int64_t>(i) * stride < rows; ++i) copy(i, first + i * stride);
        }
        __syncthreads();
    }
    // The row is there. A wait that gives up is recorded and the loop goes on: every thread still takes part in every
    // barrier, the result is void.
    __device__ __forceinline__ const T* wait(int row) {
        const WaitCtx wc{ring.status, &sh.abort};
        mbar_wait(smem_u32(&sh.full[stage]), phase, wc, SITE_NORM_ROW, row);
        return reinterpret_cast<const T*>(smem + stage * ring.stage_bytes);
    }
    // A wait has given up: copies that are still in flight get time to land before the shared memory goes away.
    __device__ __forceinline__ void finish() {
        if (*static_cast<volatile int*>(&sh.abort)) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) {
            }
        }
    }
    // After the row's reduction: the stage takes the row that is `stages` turns ahead.
    __device__ __forceinline__ void next(int row) {
        const int64_t ahead = row + static_cast<int64_t>(ring.stages) * stride;
        if (threadIdx.x == 0 && ahead < rows) copy(stage, static_cast<int>(ahead));
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

__device__ __forceinline__ float rstd_of(float sum_sq, int H, float eps) {
    return 1.0f / sqrtf(sum_sq / static_cast<float>(H) + eps);
}
// e8m0 byte of a block maximum: floor(log2(amax)) + 127 within 0..254, which is the exponent field itself
__device__ __forceinline__ int mx_scale(float amax) { return min(static_cast<int>(__float_as_uint(amax) >> 23), 254); }
// 2^(127 - e)
__device__ __forceinline__ float mx_inverse(int e) {
    return __uint_as_float(e == 254 ? 0x00400000u : static_cast<unsigned>(254 - e) << 23);
}
__device__ __forceinline__ size_t mx_atom_offset(int row, int group4, int KB) {
    const int rb = row >> 7, r1 = (row & 127) >> 5, r0 = row & 31;
    return ((static_cast<size_t>(rb) * KB + group4) * 32 + r0) * 16 + r1 * 4;
}

// Scale words of the last 128-row block's rows that do not exist: 0.
__device__ __forceinline__ void mx_clear_padding(uint8_t* atoms, int rows, int H, int threads) {
    const int left = rows & 127, words = H / 128 * 128;
    if (left == 0) return;
    uint32_t* block = reinterpret_cast<uint32_t*>(atoms) + static_cast<size_t>(rows >> 7) * words;
    for (int i = blockIdx.x * threads + threadIdx.x; i < words; i += gridDim.x * threads) {
        const int w = i & 127;  // word 4 * (row % 32) + row / 32 of an atom
        if ((w >> 2) + 32 * (w & 3) >= left) block[i] = 0u;
    }
}

struct NormOut {
    void* y;      // rows, or null with MX
    float* rstd;  // may be null
    uint8_t *q, *s_rows, *atoms;
};

// Rows that fit into registers: VPT vectors of V elements a thread, a row to a CTA (or to a warp where rows are
// narrow). CTAs are persistent: the weight is read once, and the next row's loads are issued as soon as this row's values
// have been added up, so that they are in flight during the reduction and the writing of y. Every element is read once
// and written once. NT: most threads that share a row.
template <typename T, typename W, int VPT, int NT, bool WARP, bool RAGGED, bool MX>
__global__ void __launch_bounds__(NT)
add_rms_norm_kernel(const T* x, const T* residual, const W* weight, int rows, int H, float eps, T* r_out,
                    const NormOut out) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float part[2][32];
    next_may_begin();
    previous_done();
    const int per_row = WARP ? 32 : blockDim.x;  // threads of a row
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int first = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int stride = WARP ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const RowVectors<V, RAGGED> at(first, H);
    Pack<W, V> w[VPT];
    Pack<T, V> a[VPT], b[VPT];
    auto fetch = [&](int row) {
        const T* xr = x + static_cast<size_t>(row) * H;
        const T* rr = residual + static_cast<size_t>(row) * H;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = j * per_row + tid;
            if (i < at.count) {
                at.load(a[j], xr, i);
                if (residual != nullptr) at.load(b[j], rr, i);
            }
        }
    };
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        a[j].zero();
        b[j].zero();
        w[j].zero();
    }
    if (first < rows) fetch(first);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
        if (j * per_row + tid < at.count) at.load_weight(w[j], weight, j * per_row + tid);
    if constexpr (MX) mx_clear_padding(out.atoms, rows, H, WARP ? blockDim.x : per_row);
    int which = 0;
    for (int row = first; row < rows; row += stride, which ^= 1) {
        Pack<T, V> r[VPT];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            r[j] = residual != nullptr ? added(a[j], b[j]) : a[j];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float v = to_f32(r[j].e[k]);
                ss += v * v;
            }
        }
        if (row + stride < rows) fetch(row + stride);
        const size_t base = static_cast<size_t>(row) * H;
        if (residual != nullptr) {
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (j * per_row + tid < at.count) at.store(r[j], r_out + base, j * per_row + tid);
        }
        const float rstd = rstd_of(row_sum<WARP>(ss, part, which, per_row), H, eps);
        if (out.rstd != nullptr && tid == 0) out.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = j * per_row + tid;
            if constexpr (!MX) {
                if (i < at.count) {
                    Pack<T, V> y;
#pragma unroll
                    for (int k = 0; k < V; ++k) y.e[k] = from_f32<T>(to_f32(r[j].e[k]) * rstd * to_f32(w[j].e[k]));
                    at.store(y, static_cast<T*>(out.y) + base, i);
                }
            } else {
                // 32 / V lanes hold a block of 32 values, 128 / V lanes the four blocks whose scale bytes are one
                // word of s_rows and of the atoms. H % 128 == 0, so such lanes are all inside the row or all outside.
                constexpr int BLOCK = 32 / V, WORD = 128 / V;
                float f[V], amax = 0.f;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    f[k] = to_f32(r[j].e[k]) * to_f32(w[j].e[k]);
                    amax = fmaxf(amax, fabsf(f[k]));
                }
#pragma unroll
                for (int o = 1; o < BLOCK; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const int e = mx_scale(amax * rstd);
                // y * 2^(127 - e) with one product: rstd times a power of two is exact while it stays clear of the ends of
                // fp32 (rstd lies between 2^-64 and 2^64); outside, and for blocks of zeros, with two
                float inv = rstd * mx_inverse(e);
                if (e < 96 || e > 158) {
                    inv = mx_inverse(e);
#pragma unroll
                    for (int k = 0; k < V; ++k) f[k] *= rstd;
                }
                uint32_t word = e;  // of the first lane of four blocks
                word |= __shfl_down_sync(0xffffffffu, word, BLOCK) << 8;
                word |= __shfl_down_sync(0xffffffffu, word, 2 * BLOCK) << 16;
                const int lane = threadIdx.x & 31, lead = lane & ~(WORD - 1);
                if (i < at.count) {
                    uint32_t p[V / 4];
#pragma unroll
                    for (int k = 0; k < V / 4; ++k) {
                        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * k] * inv, f[4 * k + 1] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * k + 2] * inv, f[4 * k + 3] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        p[k] = lo | (hi << 16);
                    }
                    uint8_t* dst = out.q + base + static_cast<size_t>(i) * V;
                    if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(p[0], p[1]);
                    else *reinterpret_cast<uint32_t*>(dst) = p[0];
                    if (lane == lead) {
                        const int g4 = i / WORD;
                        *reinterpret_cast<uint32_t*>(out.s_rows + static_cast<size_t>(row) * (H / 32) + 4 * g4) = word;
                        *reinterpret_cast<uint32_t*>(out.atoms + mx_atom_offset(row, g4, H / 128)) = word;
                    }
                }
            }
        }
    }
}

// Rows of more than 2048 vectors, and tensors that do not start on 16 bytes: a pass that adds, keeps r and sums the squares,
// and a pass that writes y. A thread meets the same elements in both, so r_out may be the residual's or x's own buffer.
template <typename T, typename W, bool MX>
__global__ void __launch_bounds__(NORM_THREADS)
add_rms_norm_wide_kernel(const T* x, const T* residual, const W* weight, int rows, int H, float eps, T* r_out,
                         const NormOut out) {
    __shared__ float part[2][32];
    constexpr int STEP = MX ? 32 : 1;  // consecutive elements of a thread
    next_may_begin();
    previous_done();
    if constexpr (MX) mx_clear_padding(out.atoms, rows, H, NORM_THREADS);
    int which = 0;
    for (int row = blockIdx.x; row < rows; row += gridDim.x, which ^= 1) {
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
        const float rstd = rstd_of(row_sum<false>(ss, part, which, NORM_THREADS), H, eps);
        if (out.rstd != nullptr && threadIdx.x == 0) out.rstd[row] = rstd;
        const T* r = residual != nullptr ? r_out : x;
        for (int c = threadIdx.x * STEP; c < H; c += NORM_THREADS * STEP) {
            if constexpr (!MX) {
                static_cast<T*>(out.y)[base + c] = from_f32<T>(to_f32(r[base + c]) * rstd * to_f32(weight[c]));
            } else {
                float amax = 0.f;
                for (int i = 0; i < 32; ++i)
                    amax = fmaxf(amax, fabsf(to_f32(r[base + c + i]) * rstd * to_f32(weight[c + i])));
                const int e = mx_scale(amax);
                const float inv = mx_inverse(e);
                for (int i = 0; i < 32; ++i)
                    out.q[base + c + i] = __nv_cvt_float_to_fp8(to_f32(r[base + c + i]) * rstd * to_f32(weight[c + i]) * inv,
                                                                __NV_SATFINITE, __NV_E4M3);
                const int kg = c >> 5;
                out.s_rows[static_cast<size_t>(row) * (H / 32) + kg] = static_cast<uint8_t>(e);
                out.atoms[mx_atom_offset(row, kg >> 2, H / 128) + (kg & 3)] = static_cast<uint8_t>(e);
            }
        }
    }
}

// Backward pass on the same plan, with the thread's columns of dw summed in registers over the CTA's rows. Each CTA
// leaves one row of `partial` [gridDim.x][H]; every element is summed by one thread in row order: the same bits on
// every run.
template <typename T, typename W, int VPT, int NT, int FROM, bool RAGGED>
__global__ void __launch_bounds__(NT)
add_rms_norm_bwd_kernel(const T* dy, const T* dr, const T* r,
                        const float* rstd_in, const W* weight, int rows, int H,
                        T* dx, float* partial, const Ring ring) {
    constexpr int V = 16 / sizeof(T);
    constexpr bool WARP = FROM == FROM_WARP, RING = FROM == FROM_RING;
    static_assert(!(RING && RAGGED), "the ring copies rows that start on 16 bytes");
    __shared__ float part[2][32];
    __shared__ float warp_dw[WARP ? NT / 32 : 1][WARP ? 32 * VPT * V : 1];
    __shared__ RingShared sh;
    extern __shared__ __align__(128) uint8_t rows_smem[];
    const int per_row = WARP ? 32 : blockDim.x;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int first = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int stride = WARP ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const RowVectors<V, RAGGED> at(first, H);
    next_may_begin();
    previous_done();
    const T* const src[3] = {dy, r, dr};
    RowRing<T, 3> in{sh, ring, rows_smem, src, dr != nullptr ? 3 : 2, stride, rows, H};
    if constexpr (RING) in.start(first);
    Pack<W, V> w[VPT];
    Pack<T, V> a[VPT], b[VPT], c[VPT];
    float next_rstd = 0.f;
    float dw[VPT][V];
    auto fetch = [&](const T* p, const T* q) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = j * per_row + tid;
            if (i < at.count) {
                at.load(a[j], p, i);
                at.load(b[j], q, i);
            }
        }
    };
    auto fetch_above = [&](const T* p) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (j * per_row + tid < at.count) at.load(c[j], p, j * per_row + tid);
    };
    auto fetch_row = [&](int row) {
        fetch(dy + static_cast<size_t>(row) * H, r + static_cast<size_t>(row) * H);
        next_rstd = rstd_in[row];
    };
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        a[j].zero();
        b[j].zero();
        c[j].zero();
        w[j].zero();
#pragma unroll
        for (int k = 0; k < V; ++k) dw[j][k] = 0.f;
    }
    if (RING && first < rows) next_rstd = rstd_in[first];
    if (!RING && first < rows) fetch_row(first);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
        if (j * per_row + tid < at.count) at.load_weight(w[j], weight, j * per_row + tid);
    int which = 0;
    for (int row = first; row < rows; row += stride, which ^= 1) {
        const size_t base = static_cast<size_t>(row) * H;
        const float rstd = next_rstd;
        if constexpr (RING) {
            if (row + stride < rows) next_rstd = rstd_in[row + stride];
            const T* row_in = in.wait(row);
            fetch(row_in, row_in + H);
            if (dr != nullptr) fetch_above(row_in + 2 * H);
        } else if (dr != nullptr) {
            fetch_above(dr + base);
        }
        Pack<T, V> d[VPT], h[VPT];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            d[j] = a[j];
            h[j] = b[j];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float dn = to_f32(d[j].e[k]) * (to_f32(h[j].e[k]) * rstd);
                dot += dn * to_f32(w[j].e[k]);
                dw[j][k] += dn;
            }
        }
        if (!RING && row + stride < rows) fetch_row(row + stride);
        const float mean = row_sum<WARP>(dot, part, which, per_row) / static_cast<float>(H);
        if constexpr (RING) in.next(row);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = j * per_row + tid;
            if (i < at.count) {
                Pack<T, V> o;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float n = to_f32(h[j].e[k]) * rstd;
                    float v = rstd * (to_f32(d[j].e[k]) * to_f32(w[j].e[k]) - n * mean);
                    if (dr != nullptr) v += to_f32(c[j].e[k]);
                    o.e[k] = from_f32<T>(v);
                }
                at.store(o, dx + base, i);
            }
        }
    }
    if constexpr (RING) in.finish();
    float* mine = partial + static_cast<size_t>(blockIdx.x) * H;
    if constexpr (WARP) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                // element (j * 32 + tid) * V + k - shift; a warp's shift is its own
                const int col = (j * 32 + tid) * V + k - at.shift;
                if (col >= 0 && col < H) warp_dw[threadIdx.x >> 5][col] = first < rows ? dw[j][k] : 0.f;
            }
        __syncthreads();
        for (int col = threadIdx.x; col < H; col += blockDim.x) {
            float s = 0.f;
            for (int q = 0; q < NT / 32; ++q) s += warp_dw[q][col];
            mine[col] = s;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (j * per_row + tid < at.count) {
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (at.has(j * per_row + tid, k)) mine[(j * per_row + tid) * V + k - at.shift] = dw[j][k];
            }
    }
}

// The same rows, backward.
template <typename T, typename W>
__global__ void __launch_bounds__(NORM_THREADS)
add_rms_norm_bwd_wide_kernel(const T* dy, const T* dr, const T* r,
                             const float* rstd_in, const W* weight, int rows, int H,
                             T* dx, float* partial) {
    __shared__ float part[2][32];
    next_may_begin();
    previous_done();
    float* mine = partial + static_cast<size_t>(blockIdx.x) * H;
    for (int c = threadIdx.x; c < H; c += NORM_THREADS) mine[c] = 0.f;
    int which = 0;
    for (int row = blockIdx.x; row < rows; row += gridDim.x, which ^= 1) {
        const size_t base = static_cast<size_t>(row) * H;
        const float rstd = rstd_in[row];
        float dot = 0.f;
        for (int c = threadIdx.x; c < H; c += NORM_THREADS) {
            const float dn = to_f32(dy[base + c]) * (to_f32(r[base + c]) * rstd);
            dot += dn * to_f32(weight[c]);
            mine[c] += dn;
        }
        const float mean = row_sum<false>(dot, part, which, NORM_THREADS) / static_cast<float>(H);
        for (int c = threadIdx.x; c < H; c += NORM_THREADS) {
            const float n = to_f32(r[base + c]) * rstd;
            float v = rstd * (to_f32(dy[base + c]) * to_f32(weight[c]) - n * mean);
            if (dr != nullptr) v += to_f32(dr[base + c]);
            dx[base + c] = from_f32<T>(v);
        }
    }
}

// Few rows, backward in one launch: dw needs the rows' rstd but not their sums, so the first `rows` CTAs make dx, a row each, and
// the others dw, 64 columns each, reading dy and r once more (from L2). A step of 7 rows of 4176 with its forward pass
// takes 18.6 us instead of 22.4, which are the host's: a launch and a buffer less. WIDE: rows that do not fit into
// registers, and tensors that do not start on 16 bytes.
template <typename T, typename W, int VPT, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(1024)
add_rms_norm_bwd_few_kernel(const T* dy, const T* dr, const T* r, const float* rstd_in, const W* weight, int rows, int H, T* dx,
                            W* dw) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float part[2][32];
    __shared__ float sum[32][64];
    next_may_begin();
    previous_done();
    const int tid = threadIdx.x, threads = blockDim.x;
    if (static_cast<int>(blockIdx.x) < rows) {
        const int row = blockIdx.x;
        const size_t base = static_cast<size_t>(row) * H;
        const float rstd = rstd_in[row];
        if constexpr (WIDE) {
            float dot = 0.f;
            for (int c = tid; c < H; c += threads) dot += to_f32(dy[base + c]) * to_f32(weight[c]) * (to_f32(r[base + c]) * rstd);
            const float mean = row_sum<false>(dot, part, 0, threads) / static_cast<float>(H);
            for (int c = tid; c < H; c += threads) {
                const float n = to_f32(r[base + c]) * rstd;
                float v = rstd * (to_f32(dy[base + c]) * to_f32(weight[c]) - n * mean);
                if (dr != nullptr) v += to_f32(dr[base + c]);
                dx[base + c] = from_f32<T>(v);
            }
        } else {
            const RowVectors<V, RAGGED> at(row, H);
            Pack<T, V> d[VPT], h[VPT], above[VPT];
            Pack<W, V> w[VPT];
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int i = j * threads + tid;
                d[j].zero();
                h[j].zero();
                above[j].zero();
                w[j].zero();
                if (i < at.count) {
                    at.load(d[j], dy + base, i);
                    at.load(h[j], r + base, i);
                    if (dr != nullptr) at.load(above[j], dr + base, i);
                    at.load_weight(w[j], weight, i);
                }
            }
#pragma unroll
            for (int j = 0; j < VPT; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    dot += to_f32(d[j].e[k]) * (to_f32(h[j].e[k]) * rstd) * to_f32(w[j].e[k]);
            const float mean = row_sum<false>(dot, part, 0, threads) / static_cast<float>(H);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int i = j * threads + tid;
                if (i < at.count) {
                    Pack<T, V> o;
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float n = to_f32(h[j].e[k]) * rstd;
                        float v = rstd * (to_f32(d[j].e[k]) * to_f32(w[j].e[k]) - n * mean);
                        if (dr != nullptr) v += to_f32(above[j].e[k]);
                        o.e[k] = from_f32<T>(v);
                    }
                    at.store(o, dx + base, i);
                }
            }
        }
        return;
    }
    // warp w adds up rows w, w + warps, ...; the warps' sums are added up in order
    const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    const int c0 = (blockIdx.x - rows) * 64 + lane, c1 = c0 + 32;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
    for (int row = warp; row < rows; row += warps) {
        const size_t base = static_cast<size_t>(row) * H;
        const float rstd = rstd_in[row];
        if (c0 < H) s0 += to_f32(dy[base + c0]) * (to_f32(r[base + c0]) * rstd);
        if (c1 < H) s1 += to_f32(dy[base + c1]) * (to_f32(r[base + c1]) * rstd);
    }
    sum[warp][lane] = s0;
    sum[warp][lane + 32] = s1;
    __syncthreads();
    const int c = (blockIdx.x - rows) * 64 + tid;
    if (tid < 64 && c < H) {
        float v = 0.f;
        for (int q = 0; q < warps; ++q) v += sum[q][tid];
        dw[c] = from_f32<W>(v);
    }
}

// dw[c] = sum of the CTAs' partial sums: 32 columns to a CTA, its eight warps each take every eighth part, and
// their sums are added up in order. Launched while the backward pass still runs (its CTAs fit beside that one's), it
// waits for its end on the device.
template <typename W>
__global__ void __launch_bounds__(256)
add_rms_norm_dw_kernel(const float* partial, int parts, int H, W* __restrict__ dw) {
    __shared__ float sum[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    next_may_begin();
    previous_done();
    float s = 0.f;
    if (c < H) {
#pragma unroll 16
        for (int p = warp; p < parts; p += 8) s += partial[static_cast<size_t>(p) * H + c];
    }
    sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < H) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += sum[q][lane];
        dw[c] = from_f32<W>(v);
    }
}

// --------------------------------------------------------------------------------------------
// host side

constexpr int NORM_MAX_H = 65536;
constexpr int NORM_MAX_T = 1 << 30;  // a row index plus the rows of a turn stays an int
constexpr int NORM_MAX_SMS = 160;
// CTAs of a backward pass on one SM at most, each with a row of `partial`: two, and for narrow rows as many as have
// 32 KB of partial sums between them
static int norm_bwd_ctas(int H) { return std::max(2, std::min(8, 8192 / H)); }
// Up to so many rows a backward pass is one launch without partial sums. In device time, bf16: 128 rows of 8192 5.4 us
// instead of 7.8 + 7.5 in two overlapping launches, of 4176 4.6 instead of 5.0 + 5.0; 512 rows of 4176 12.7 instead of
// 8.7 + 8.3: a column's rows are added up by one CTA here.
constexpr int NORM_BWD_FEW = 128;
static int norm_bwd_parts(int T, int H) { return T <= NORM_BWD_FEW ? 0 : std::min(T, NORM_MAX_SMS * norm_bwd_ctas(H)); }

static int check_norm(const void* x, const void* weight, int x_is_f32, int w_is_f32, int T, int H) {
    DK_REQUIRE(T >= 0 && T <= NORM_MAX_T, "the number of rows must be between 0 and 2^30");
    DK_REQUIRE(H >= 1 && H <= NORM_MAX_H, "H must be between 1 and 65536");
    DK_REQUIRE(weight != nullptr && (T == 0 || x != nullptr), "null operand");
    DK_REQUIRE(w_is_f32 || !x_is_f32, "a bf16 weight needs bf16 rows");
    return DK_OK;
}
// Every element on its own size: what any path needs. (16 bytes only choose the faster one.)
static int check_elements(int x_is_f32, int w_is_f32, std::initializer_list<const void*> rows, const void* weight,
                          std::initializer_list<const void*> f32) {
    uintptr_t row_bits = 0, f32_bits = 0;
    for (const void* p : rows) row_bits |= reinterpret_cast<uintptr_t>(p);
    for (const void* p : f32) f32_bits |= reinterpret_cast<uintptr_t>(p);
    DK_REQUIRE((row_bits & (x_is_f32 ? 3 : 1)) == 0 && (reinterpret_cast<uintptr_t>(weight) & (w_is_f32 ? 3 : 1)) == 0 &&
                   (f32_bits & 3) == 0, "a tensor does not start on a whole element");
    return DK_OK;
}

// How a pass over T rows of H elements is cut up. n: vectors a row may span.
//   FEW      at most `few` rows, no more than a row for each SM: as many threads to a row as it can use (latency)
//   MANY     four vectors a thread, so that a CTA has enough bytes in flight (bandwidth)
//   WARP     rows of at most 4 vectors a lane: a row to a warp, no barrier
//   WIDE     a row that does not fit into the registers of 512 threads, or tensors that do not start on 16 bytes
enum class NormPlan { FEW, FEW2, MANY, MANY512, WARP, WIDE };
static NormPlan norm_plan(bool aligned, int n, int T, int few) {
    if (!aligned || n > 2048) return NormPlan::WIDE;
    if (T <= few) return n <= 1024 ? NormPlan::FEW : NormPlan::FEW2;
    if (n <= 128) return NormPlan::WARP;
    return n <= 1024 ? NormPlan::MANY : NormPlan::MANY512;
}
// Launch shape of a ring kernel: threads that share a row, CTAs on an SM and the ring of each.
struct RingShape {
    int threads, ctas, smem;
    Ring ring;
};
static int ring_shape(int nvec, int H, int elem, int arrays, RingShape* out) {
    const int threads = ((nvec + 3) / 4 + 31) / 32 * 32;
    out->threads = threads;
    out->ctas = std::max(1, 256 / threads);
    out->ring.stage_bytes = arrays * H * elem;
    out->ring.stages = std::max(2, std::min(RING_STAGES, RING_SM_BYTES / out->ctas / out->ring.stage_bytes));
    out->smem = out->ring.stages * out->ring.stage_bytes;
    return device_status_ptr(&out->ring.status);
}
template <typename K>
static int allow_smem(K kernel, bool (&done)[64]) {
    int dev = 0;
    DK_CUDA_OK(cudaGetDevice(&dev));
    if (!done[dev & 63]) {
        DK_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_SM_BYTES));
        done[dev & 63] = true;
    }
    return DK_OK;
}
static int round_threads(int n, int vpt) { return ((n + vpt - 1) / vpt + 31) / 32 * 32; }
static bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t bits = 0;
    for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
    return (bits & 15) == 0;
}

template <typename T, typename W, bool MX>
static int launch_norm(const void* x, const void* residual, const void* weight, int rows, int H, float eps, void* r_out,
                       const NormOut& out, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const bool ragged = H % V != 0;
    const int n = ragged ? (H + 2 * V - 2) / V : H / V;
    const NormPlan plan = norm_plan(aligned16({x, residual, weight, r_out, out.y}), n, rows, sms);
    auto go = [&](auto kernel, int threads, int rows_per_cta, int ctas_per_sm) {
        const int need = (rows + rows_per_cta - 1) / rows_per_cta, most = ragged ? sms * ctas_per_sm / V * V : sms * ctas_per_sm;
        return launch_early(kernel, dim3(need < most ? need : most), threads, 0, 0, st, static_cast<const T*>(x),
                            static_cast<const T*>(residual), static_cast<const W*>(weight), rows, H, eps,
                            static_cast<T*>(r_out), out);
    };
    auto planned = [&](auto is_ragged) {
        constexpr bool R = decltype(is_ragged)::value;
        switch (plan) {
            case NormPlan::FEW: return go(add_rms_norm_kernel<T, W, 1, 1024, false, R, MX>, round_threads(n, 1), 1, 1);
            case NormPlan::FEW2: return go(add_rms_norm_kernel<T, W, 2, 1024, false, R, MX>, round_threads(n, 2), 1, 1);
            case NormPlan::MANY:
                return go(add_rms_norm_kernel<T, W, 4, 256, false, R, MX>, round_threads(n, 4), 1, 512 / round_threads(n, 4));
            case NormPlan::MANY512: return go(add_rms_norm_kernel<T, W, 4, 512, false, R, MX>, round_threads(n, 4), 1, 1);
            default: return go(add_rms_norm_kernel<T, W, 4, 256, true, R, MX>, 256, 8, 2);
        }
    };
    if (plan != NormPlan::WIDE) {
        if (!ragged) return planned(std::false_type{});
        if constexpr (!MX) return planned(std::true_type{});
    }
    return go(add_rms_norm_wide_kernel<T, W, MX>, NORM_THREADS, 1, 8);
}
template <bool MX>
static int launch_norm(const void* x, const void* residual, const void* weight, int x_is_f32, int w_is_f32, int T, int H,
                       float eps, void* r_out, const NormOut& out, cudaStream_t st) {
    if (x_is_f32) return launch_norm<float, float, MX>(x, residual, weight, T, H, eps, r_out, out, st);
    if (w_is_f32) return launch_norm<__nv_bfloat16, float, MX>(x, residual, weight, T, H, eps, r_out, out, st);
    return launch_norm<__nv_bfloat16, __nv_bfloat16, MX>(x, residual, weight, T, H, eps, r_out, out, st);
}

template <typename T, typename W>
static int launch_norm_bwd(const void* dy, const void* dr, const void* r, const float* rstd, const void* weight, int rows,
                           int H, void* dx, void* dw, float* partial, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    if (sms > NORM_MAX_SMS) sms = NORM_MAX_SMS;
    const bool ragged = H % V != 0;
    const int n = ragged ? (H + 2 * V - 2) / V : H / V;
    const NormPlan plan = norm_plan(aligned16({dy, dr, r, weight, dx}), n, rows, NORM_BWD_FEW);
    if (rows <= NORM_BWD_FEW) {
        auto few = [&](auto kernel, int threads) {
            // 512 threads at least, for the CTAs that make dw
            return launch_early(kernel, dim3(rows + (H + 63) / 64), std::max(512, threads), 0, 0, st, static_cast<const T*>(dy),
                                static_cast<const T*>(dr), static_cast<const T*>(r), rstd, static_cast<const W*>(weight), rows, H,
                                static_cast<T*>(dx), static_cast<W*>(dw));
        };
        if (plan == NormPlan::WIDE) return few(add_rms_norm_bwd_few_kernel<T, W, 1, false, true>, 1024);
        if (n <= 1024)
            return ragged ? few(add_rms_norm_bwd_few_kernel<T, W, 1, true, false>, round_threads(n, 1))
                          : few(add_rms_norm_bwd_few_kernel<T, W, 1, false, false>, round_threads(n, 1));
        return ragged ? few(add_rms_norm_bwd_few_kernel<T, W, 2, true, false>, round_threads(n, 2))
                      : few(add_rms_norm_bwd_few_kernel<T, W, 2, false, false>, round_threads(n, 2));
    }
    int parts = 0;
    RingShape shape{};
    auto grid = [&](int rows_per_cta, int ctas_per_sm) {
        const int ctas = sms * std::min(ctas_per_sm, norm_bwd_ctas(H));
        const int need = (rows + rows_per_cta - 1) / rows_per_cta, most = ragged ? ctas / V * V : ctas;
        return parts = need < most ? need : most;
    };
    auto go = [&](auto kernel, int threads, int rows_per_cta, int ctas_per_sm) {
        return launch_early(kernel, dim3(grid(rows_per_cta, ctas_per_sm)), threads, shape.smem, 0, st,
                            static_cast<const T*>(dy), static_cast<const T*>(dr), static_cast<const T*>(r), rstd,
                            static_cast<const W*>(weight), rows, H, static_cast<T*>(dx), partial, shape.ring);
    };
    auto planned = [&](auto is_ragged) {
        constexpr bool R = decltype(is_ragged)::value;
        switch (plan) {
            case NormPlan::MANY: {
                if constexpr (R) {
                    return go(add_rms_norm_bwd_kernel<T, W, 4, 256, FROM_REGS, true>, round_threads(n, 4), 1,
                              256 / round_threads(n, 4));
                } else {
                    const auto kernel = add_rms_norm_bwd_kernel<T, W, 4, 256, FROM_RING, false>;
                    static bool allowed[64] = {false};
                    int rc2 = allow_smem(kernel, allowed);
                    if (rc2 == DK_OK) rc2 = ring_shape(n, H, sizeof(T), dr != nullptr ? 3 : 2, &shape);
                    return rc2 != DK_OK ? rc2 : go(kernel, shape.threads, 1, shape.ctas);
                }
            }
            case NormPlan::MANY512: return go(add_rms_norm_bwd_kernel<T, W, 4, 512, FROM_REGS, R>, round_threads(n, 4), 1, 1);
            default: return go(add_rms_norm_bwd_kernel<T, W, 4, 256, FROM_WARP, R>, 256, 8, 2);
        }
    };
    int done_rc;
    if (plan == NormPlan::WIDE)
        done_rc = launch_early(add_rms_norm_bwd_wide_kernel<T, W>, dim3(grid(1, 2)), NORM_THREADS, 0, 0, st,
                               static_cast<const T*>(dy), static_cast<const T*>(dr), static_cast<const T*>(r), rstd,
                               static_cast<const W*>(weight), rows, H, static_cast<T*>(dx), partial);
    else
        done_rc = ragged ? planned(std::true_type{}) : planned(std::false_type{});
    if (done_rc != DK_OK) return done_rc;
    return launch_early(add_rms_norm_dw_kernel<W>, dim3((H + 31) / 32), 256, 0, 0, st, static_cast<const float*>(partial), parts, H,
                        static_cast<W*>(dw));
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
    const int rc2 = check_elements(x_is_f32, w_is_f32, {x, residual, y, r_out}, weight, {rstd});
    if (rc2 != DK_OK) return rc2;
    return launch_norm<false>(x, residual, weight, x_is_f32, w_is_f32, T, H, eps, r_out,
                              NormOut{y, rstd, nullptr, nullptr, nullptr}, static_cast<cudaStream_t>(stream));
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
    const int rc2 = check_elements(x_is_f32, w_is_f32, {x, residual, r_out}, weight, {});
    if (rc2 != DK_OK) return rc2;
    return launch_norm<true>(x, residual, weight, x_is_f32, w_is_f32, T, H, eps, r_out,
                             NormOut{nullptr, nullptr, static_cast<uint8_t*>(q), static_cast<uint8_t*>(s_rows),
                                     static_cast<uint8_t*>(sf_atoms)},
                             static_cast<cudaStream_t>(stream));
}

extern "C" size_t dk_add_rms_norm_bwd_workspace_bytes(int T, int H) {
    using namespace dk;
    if (T < 0 || T > NORM_MAX_T || H < 1 || H > NORM_MAX_H) return 0;
    return static_cast<size_t>(norm_bwd_parts(T, H)) * H * sizeof(float);
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
    const size_t need = dk_add_rms_norm_bwd_workspace_bytes(T, H);
    DK_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small");
    DK_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
    const int rc2 = check_elements(x_is_f32, w_is_f32, {dy, dr, r, dx}, weight, {rstd});
    if (rc2 != DK_OK) return rc2;
    DK_REQUIRE((reinterpret_cast<uintptr_t>(dw) & (w_is_f32 ? 3 : 1)) == 0, "a tensor does not start on a whole element");
    float* partial = static_cast<float*>(workspace);
    if (x_is_f32) return launch_norm_bwd<float, float>(dy, dr, r, rstd, weight, T, H, dx, dw, partial, st);
    if (w_is_f32) return launch_norm_bwd<__nv_bfloat16, float>(dy, dr, r, rstd, weight, T, H, dx, dw, partial, st);
    return launch_norm_bwd<__nv_bfloat16, __nv_bfloat16>(dy, dr, r, rstd, weight, T, H, dx, dw, partial, st);
}
