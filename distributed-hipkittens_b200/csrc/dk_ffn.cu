// Gated feed-forward block and its backward pass, bf16, for sm_100a.
//
//   [g | u] = x W13^T        x [T,H], W13 [2F,H] (F gate rows, then F up rows, as in the MoE layer)
//   h = silu(g) * u          silu(g) = g * s, s = 1 / (1 + exp(-g))
//   y = h W2^T               W2 [H,F]
//
//   dh = dy W2,  dg = dh * u * s * (1 + g * (1 - s)),  du = dh * g * s
//   dx = [dg|du] W13,  dW13 = [dg|du]^T x,  dW2 = dy^T h
//
// One kernel serves all six products, D[M,N] = A B with fp32 accumulation in tensor memory. It is
// instantiated over how the operands lie in memory: K-major ([M,K] and [N,K], the weights of a
// forward pass) or MN-major ([K,M] and [K,N]: W2 and W13 seen from the other side, and the token axis as
// K in the weight gradients), which the tensor core reads through a descriptor of its own, so nothing is
// transposed in memory. What it does with a finished tile:
//   EPI_STORE   bf16 rows of D
//   EPI_GATED   the B tile is 128 gate rows and 128 up rows, so a thread holds g and u of the same
//               place: silu(g) * u leaves as h, and g, u too when a backward pass will follow
//   EPI_DGATED  D is dh: with the kept g, u of the same place, dg and du leave
// h, dg and du are rounded to bf16, the type in which the tensor core takes them up again. g and u are kept in
// 32 bits: dx and dW13 then carry two roundings, [dg|du] and their own (error against 64 bits 0.0024); kept in bf16
// their roundings entered too (0.0030). The price is 8 bytes a value of h instead of 4, written and read beside
// matrix products.
//
//   warp 0      TMA producer: 128-byte-swizzled boxes into a ring of stages
//   warp 1      one thread issues tcgen05.mma into one of two 256-column accumulators
//   warps 2-5   epilogue: tcgen05.ld, swizzled staging in shared memory, TMA stores (which clip the
//               ragged edges)
//
// PAIR = 2: a cluster of two CTAs per 256x256 tile (cta_group::2). Each stages its 128 rows of A and half of
// the B tile (gated: CTA 0 the gate rows, CTA 1 the up rows), so a stage is 32 KiB instead of 48, the ring six
// deep instead of four, and a flop needs two thirds of the shared-memory fill. Both CTAs' loads complete on the
// leader's barrier, the leader issues the MMAs. PAIR = 1: one CTA per 128x256 tile, for row counts whose last pair
// would be half empty.
#include "dk_host.h"
#include "dk_ptx.cuh"

namespace dk {

namespace ffn {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 64;  // 64 bf16 = 128 bytes = one swizzle row
constexpr int UMMA_K = 16;
constexpr int A_BYTES = BM * BK * 2;
constexpr int MN_BLOCK = 64 * BK * 2;  // an MN-major box: 64 elements of M or N (128 bytes) x 64 of K
constexpr int EPI_BUF = 32 * 128;      // 32 rows x 64 bf16
constexpr int EPI_BYTES = 4 * 2 * EPI_BUF;
template <int PAIR>
struct Cfg {
    static constexpr int B_ROWS = BN / PAIR;
    static constexpr int B_BYTES = B_ROWS * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = PAIR == 2 ? 6 : 4;
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_BYTES + 256;
};
constexpr int THREADS = 192;
constexpr int TMEM_COLS = 512;

enum : int { EPI_STORE = 0, EPI_GATED = 1, EPI_DGATED = 2 };
enum : unsigned { SITE_EMPTY = 101, SITE_FULL = 102, SITE_TMEM_EMPTY = 103, SITE_TMEM_FULL = 104 };

struct Maps {
    CUtensorMap a, b;
    CUtensorMap out[3];  // STORE: D; GATED: h, g, u; DGATED: dg, du
};

struct Args {
    int M, N, num_kb;  // N: columns of the output (GATED, DGATED: F)
    int tiles_m, tiles_n, group_m;  // tiles of 128 * PAIR rows
    int save;                 // GATED: g and u leave too
    const float* gu;          // DGATED: kept [g|u], [M, 2N]
    unsigned* status;
};

// Descriptor of an MN-major operand in boxes of 64 (M or N) x 64 (K) with the 128-byte swizzle: the
// leading offset leads from one 64-element box to the next, the stride offset from eight K rows to
// the next eight.
__device__ __forceinline__ uint64_t desc_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3ffff) >> 4);
    d |= static_cast<uint64_t>(MN_BLOCK >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Column tiles run slowest inside a group of group_m row tiles, so that CTAs running together share
// operand tiles in L2.
__device__ __forceinline__ void tile_coords(int t, const Args& g, int& m, int& n) {
    const int per_group = g.group_m * g.tiles_n;
    const int grp = t / per_group;
    const int first = grp * g.group_m;
    const int gsz = min(g.tiles_m - first, g.group_m);
    const int r = t - grp * per_group;
    m = first + r % gsz;
    n = r / gsz;
}

__device__ __forceinline__ float sigmoid_f(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// 32 packed columns (64 bytes) of this lane's row into half `hi` of a swizzled 32x64 staging buffer.
__device__ __forceinline__ void stage_half(uint32_t buf, int lane, int hi, const uint32_t (&p)[16]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t addr = buf + lane * 128 + (((hi * 4 + j) ^ (lane & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(p[4 * j]), "r"(p[4 * j + 1]),
                     "r"(p[4 * j + 2]), "r"(p[4 * j + 3])
                     : "memory");
    }
}
__device__ __forceinline__ void pack32(const float (&f)[32], uint32_t (&p)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void ld_acc(uint32_t taddr, float (&f)[32]) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(taddr, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}
// 32 fp32 of global memory; columns at or beyond `n` (a multiple of 8) count as 0
__device__ __forceinline__ void ld_row32(const float* p, int col, int n, bool ok, float (&f)[32]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ok && col + 4 * j < n) v = __ldg(reinterpret_cast<const float4*>(p) + j);
        f[4 * j] = v.x;
        f[4 * j + 1] = v.y;
        f[4 * j + 2] = v.z;
        f[4 * j + 3] = v.w;
    }
}

template <bool A_MN, bool B_MN, int EPI, int PAIR>
__global__ void __launch_bounds__(THREADS, 1) ffn_gemm_kernel(const __grid_constant__ Maps maps, const Args g) {
    constexpr int STAGES = Cfg<PAIR>::STAGES, STAGE_BYTES = Cfg<PAIR>::STAGE_BYTES, B_ROWS = Cfg<PAIR>::B_ROWS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem_base;
    const uint32_t epi = smem_base + STAGES * STAGE_BYTES;
    const uint32_t ctrl = epi + EPI_BYTES;
    uint8_t* ctrl_p = smem_raw + (ctrl - smem_u32(smem_raw));
    const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * STAGES;
    const uint32_t bar_tfull = ctrl + 16 * STAGES, bar_tempty = bar_tfull + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl_p + 16 * STAGES + 32);
    volatile int* abort_sm = reinterpret_cast<volatile int*>(ctrl_p + 16 * STAGES + 40);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{g.status, abort_sm};
    const int crank = PAIR == 2 ? static_cast<int>(cluster_ctarank()) : 0;
    const int unit = blockIdx.x / PAIR, nunits = gridDim.x / PAIR;
    const int num_tiles = g.tiles_m * g.tiles_n;

    if (threadIdx.x == 0) {
        *abort_sm = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + 8 * a, 1);
            mbar_init(bar_tempty + 8 * a, 128 * PAIR);  // the leader hears both CTAs' epilogues
        }
        fence_mbar_init();
        tma_prefetch_desc(&maps.a);
        tma_prefetch_desc(&maps.b);
    }
    if (warp == 1) {
        tmem_alloc<PAIR>(smem_u32(const_cast<uint32_t*>(tmem_slot)), TMEM_COLS);
        tmem_relinquish<PAIR>();
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR == 2) {
        // both CTAs' barriers exist before either signals the other's
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += nunits) {
                int m, n;
                tile_coords(t, g, m, n);
                m = m * PAIR + crank;  // this CTA's 128-row tile
                for (int kb = 0; kb < g.num_kb; ++kb) {
                    if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, wc, SITE_EMPTY, t)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = ring + s * STAGE_BYTES, sb = sa + A_BYTES;
                    // a pair's loads complete on the leader's barrier, which expects the bytes of both CTAs
                    const uint32_t full = PAIR == 2 ? mapa_shared(bar_full + 8 * s, 0) : bar_full + 8 * s;
                    if (crank == 0) mbar_expect_tx(bar_full + 8 * s, PAIR * STAGE_BYTES);
                    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                        if (PAIR == 2) tma_load_2d_pair(dst, map, full, x, y);
                        else tma_load_2d(dst, map, full, x, y);
                    };
                    if (A_MN) {
                        for (int i = 0; i < BM / 64; ++i) load(sa + i * MN_BLOCK, &maps.a, m * BM + 64 * i, kb * BK);
                    } else {
                        load(sa, &maps.a, kb * BK, m * BM);
                    }
                    if (EPI == EPI_GATED) {
                        // gate rows that do not exist read up rows instead, up rows zeros: not stored
                        if (PAIR == 2) {
                            load(sb, &maps.b, kb * BK, crank * g.N + n * 128);
                        } else {
                            load(sb, &maps.b, kb * BK, n * 128);
                            load(sb + 128 * BK * 2, &maps.b, kb * BK, g.N + n * 128);
                        }
                    } else if (B_MN) {
                        for (int i = 0; i < B_ROWS / 64; ++i)
                            load(sb + i * MN_BLOCK, &maps.b, n * BN + crank * B_ROWS + 64 * i, kb * BK);
                    } else {
                        load(sb, &maps.b, kb * BK, n * BN + crank * B_ROWS);
                    }
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && crank == 0) {
            constexpr uint32_t idesc = umma_idesc(1, 1, BM * PAIR, BN) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
            // descriptor steps of 16 elements of K, in 16-byte units: 32 bytes along the swizzle row, or
            // 16 rows of 128 bytes
            constexpr uint64_t a_step = A_MN ? 16 * 128 / 16 : 2, b_step = B_MN ? 16 * 128 / 16 : 2;
            int s = 0, acc = 0;
            uint32_t ph = 0, acc_ph = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += nunits) {
                if (!mbar_wait(bar_tempty + 8 * acc, acc_ph ^ 1, wc, SITE_TMEM_EMPTY, t)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                for (int kb = 0; kb < g.num_kb; ++kb) {
                    if (!mbar_wait(bar_full + 8 * s, ph, wc, SITE_FULL, t)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = ring + s * STAGE_BYTES, sb = sa + A_BYTES;
                    const uint64_t da = A_MN ? desc_mn(sa) : umma_desc_sw128(sa);
                    const uint64_t db = B_MN ? desc_mn(sb) : umma_desc_sw128(sb);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        umma_f16<PAIR>(d_tmem, da + a_step * k, db + b_step * k, idesc, (kb | k) != 0);
                    // the stage is free in both CTAs once these MMAs have read it
                    if (PAIR == 2) umma_commit_pair(bar_empty + 8 * s, 3);
                    else umma_commit<1>(bar_empty + 8 * s);
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) break;
                if (PAIR == 2) umma_commit_pair(bar_tfull + 8 * acc, 3);
                else umma_commit<1>(bar_tfull + 8 * acc);
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1;
            }
        }
    } else {
        const int q = warp & 3;  // TMEM lane quarter this warp may read
        const uint32_t my_epi = epi + (warp - 2) * 2 * EPI_BUF;
        int acc = 0, nbuf = 0;
        uint32_t acc_ph = 0;
        // a buffer whose last store (two stores ago) has been read
        auto next_buf = [&]() {
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
            return my_epi + (nbuf++ & 1) * EPI_BUF;
        };
        // `words`: bf16 units an element takes up (the maps count in those)
        auto send = [&](uint32_t buf, const CUtensorMap* map, int col, int row, int words = 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (col < g.N && row < g.M) tma_store_2d(map, buf, col * words, row);
                tma_store_commit();
            }
        };
        for (int t = unit; t < num_tiles; t += nunits) {
            int m, n;
            tile_coords(t, g, m, n);
            const int row0 = (m * PAIR + crank) * BM + q * 32;
            if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, acc_ph, wc, SITE_TMEM_FULL, t))) break;
            tc_fence_after();
            const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
            if constexpr (EPI == EPI_STORE) {
#pragma unroll 1
                for (int c = 0; c < BN / 64; ++c) {
                    const uint32_t buf = next_buf();
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        float f[32];
                        uint32_t p[16];
                        ld_acc(t_acc + c * 64 + hi * 32, f);
                        pack32(f, p);
                        stage_half(buf, lane, hi, p);
                    }
                    send(buf, &maps.out[0], n * BN + c * 64, row0);
                }
            } else if constexpr (EPI == EPI_GATED) {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    const int col = n * 128 + c * 64;
                    if (g.save) {
#pragma unroll 1
                        for (int part = 0; part < 4; ++part) {  // gate, up of 32 columns, gate, up of the next 32
                            const int sub = (part & 1) * 128 + c * 64 + (part >> 1) * 32;
                            const uint32_t buf = next_buf();
                            uint32_t p[32];
                            tmem_ld_32x32b_x32(t_acc + sub, p);
                            tmem_ld_wait(p);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t addr = buf + lane * 128 + ((j ^ (lane & 7)) << 4);
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(p[4 * j]),
                                             "r"(p[4 * j + 1]), "r"(p[4 * j + 2]), "r"(p[4 * j + 3])
                                             : "memory");
                            }
                            send(buf, &maps.out[1 + (part & 1)], col + (part >> 1) * 32, row0, 2);
                        }
                    }
                    const uint32_t buf = next_buf();
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        float gate[32], up[32];
                        uint32_t p[16];
                        ld_acc(t_acc + c * 64 + hi * 32, gate);
                        ld_acc(t_acc + 128 + c * 64 + hi * 32, up);
#pragma unroll
                        for (int i = 0; i < 32; ++i) gate[i] = gate[i] * sigmoid_f(gate[i]) * up[i];
                        pack32(gate, p);
                        stage_half(buf, lane, hi, p);
                    }
                    send(buf, &maps.out[0], col, row0);
                }
            } else {
                const int row = row0 + lane;
                const bool row_ok = row < g.M;
                const float* gu = g.gu + static_cast<size_t>(row) * (2 * static_cast<size_t>(g.N));
#pragma unroll 1
                for (int c = 0; c < BN / 64; ++c) {
                    const int col0 = n * BN + c * 64;
                    const uint32_t bg = next_buf();
                    uint32_t pu[2][16];
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const int col = col0 + hi * 32;
                        float gate[32], up[32], dh[32];
                        ld_row32(gu + col, col, g.N, row_ok, gate);
                        ld_row32(gu + g.N + col, col, g.N, row_ok, up);
                        ld_acc(t_acc + c * 64 + hi * 32, dh);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float s = sigmoid_f(gate[i]);
                            const float d = dh[i];
                            dh[i] = d * gate[i] * s;                                          // du
                            gate[i] = d * up[i] * s * (1.0f + gate[i] * (1.0f - s));          // dg
                        }
                        uint32_t pg[16];
                        pack32(gate, pg);
                        stage_half(bg, lane, hi, pg);
                        pack32(dh, pu[hi]);
                    }
                    send(bg, &maps.out[0], col0, row0);
                    const uint32_t bu = next_buf();
                    stage_half(bu, lane, 0, pu[0]);
                    stage_half(bu, lane, 1, pu[1]);
                    send(bu, &maps.out[1], col0, row0);
                }
            }
            tc_fence_before();
            if (PAIR == 2 && crank != 0) mbar_arrive_cluster(mapa_shared(bar_tempty + 8 * acc, 0));
            else mbar_arrive(bar_tempty + 8 * acc);
            acc ^= 1;
            if (acc == 0) acc_ph ^= 1;
        }
        if (lane == 0) tma_store_wait_all<0>();
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR == 2) {
        // neither CTA leaves (or frees the pair's TMEM) while the other may still signal it
        cluster_arrive();
        cluster_wait();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (*abort_sm) {
            // give copies still in flight time to land before the shared memory goes away
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) {
            }
        }
        tmem_dealloc<PAIR>(tmem_base, TMEM_COLS);
    }
}

// --------------------------------------------------------------------------------------------
// Few rows (single tokens, batches of sequences being answered): bound by reading the weights once. The roles are
// swapped: 128 weight rows are the tensor core's M, the tokens its N (padded to 16..256), so a tile is 16 KB of
// weights per 64 of K whatever the number of tokens, and F / 64 or H / 128 tiles are cut along K over a cluster
// of S CTAs until there are enough CTAs to draw on all of HBM. Each CTA leaves its fp32 partial sums in its own
// shared memory; the cluster's CTAs then add up each other's through distributed shared memory, in rank order: no
// workspace, no second launch, the same bits on every run.
//   GATED: a tile is 64 gate rows and the 64 up rows of the same columns; silu(g) * u leaves.
// The second product (from h) may start while the first still runs: its weights do not depend on the first, so the
// ring is filled with them, and only then does it wait for the rows of h.
constexpr int ROWS_THREADS = 192;
template <int N>
struct RowsCfg {
    static constexpr int W_BYTES = 128 * BK * 2;
    static constexpr int STAGE = W_BYTES + N * BK * 2;
    // two CTAs per SM up to 128 tokens, one for 256
    static constexpr int STAGES = N <= 32 ? 5 : N == 64 ? 4 : N == 128 ? 3 : 4;
    static constexpr int CTAS_PER_SM = N <= 128 ? 2 : 1;
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE + 128;
    static constexpr int TMEM = N < 32 ? 32 : N;
    static_assert(N * 128 * 4 <= STAGES * STAGE, "the partial sums reuse the ring");
};
struct RowsMaps {
    CUtensorMap w, x;
};
struct RowsArgs {
    int T, cols, num_kb;  // cols: columns of the output (F or H)
    __nv_bfloat16* out;   // [T, cols]
    float* gu;            // GATED: [T, 2 cols], may be null
    unsigned* status;
};
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

template <bool GATED, int N>
__global__ void __launch_bounds__(ROWS_THREADS) ffn_rows_kernel(const __grid_constant__ RowsMaps maps, const RowsArgs g) {
    using C = RowsCfg<N>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ctrl = ring + C::STAGES * C::STAGE;
    uint8_t* ctrl_p = smem_raw + (ctrl - smem_u32(smem_raw));
    const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * C::STAGES, bar_done = ctrl + 16 * C::STAGES;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl_p + 16 * C::STAGES + 8);
    volatile int* abort_sm = reinterpret_cast<volatile int*>(ctrl_p + 16 * C::STAGES + 16);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{g.status, abort_sm};
    uint32_t split;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
    const int S = static_cast<int>(split), rank = static_cast<int>(cluster_ctarank());
    const int tile = blockIdx.x / S;
    const int tok0 = blockIdx.y * N;
    const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * g.num_kb / S);
    const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * g.num_kb / S);

    if (threadIdx.x == 0) {
        *abort_sm = 0;
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_done, 1);
        fence_mbar_init();
        tma_prefetch_desc(&maps.w);
        tma_prefetch_desc(&maps.x);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), C::TMEM);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // the next kernel's CTAs may take the places that this one's leave
    if (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            auto load_w = [&](int kb, int s) {
                const uint32_t sw = ring + s * C::STAGE, full = bar_full + 8 * s;
                mbar_expect_tx(full, C::STAGE);
                if (GATED) {
                    // gate rows that do not exist read up rows instead, up rows zeros: not stored
                    tma_load_2d(sw, &maps.w, full, kb * BK, tile * 64);
                    tma_load_2d(sw + C::W_BYTES / 2, &maps.w, full, kb * BK, g.cols + tile * 64);
                } else {
                    tma_load_2d(sw, &maps.w, full, kb * BK, tile * 128);
                }
            };
            auto load_x = [&](int kb, int s) {
                tma_load_2d(ring + s * C::STAGE + C::W_BYTES, &maps.x, bar_full + 8 * s, kb * BK, tok0);
            };
            const int ahead = min(kb1 - kb0, C::STAGES);
            for (int i = 0; i < ahead; ++i) load_w(kb0 + i, i);
            if (!GATED) {
                // h is complete and visible from here on, to the copy engine too
                asm volatile("griddepcontrol.wait;" ::: "memory");
                asm volatile("fence.proxy.async;" ::: "memory");
            }
            for (int i = 0; i < ahead; ++i) load_x(kb0 + i, i);
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0 + ahead; kb < kb1; ++kb) {
                if (!mbar_wait(bar_empty + 8 * s, ph, wc, SITE_EMPTY, tile)) break;
                load_w(kb, s);
                load_x(kb, s);
                if (++s == C::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc(1, 1, 128, N);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(bar_full + 8 * s, ph, wc, SITE_FULL, tile)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t da = umma_desc_sw128(ring + s * C::STAGE);
                const uint64_t db = umma_desc_sw128(ring + s * C::STAGE + C::W_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) umma_f16<1>(tmem, da + 2 * k, db + 2 * k, idesc, kb != kb0 || k != 0);
                umma_commit<1>(bar_empty + 8 * s);
                if (++s == C::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (ok) umma_commit<1>(bar_done);
        }
    } else {
        // partial sums as [token][weight row]; every load has been consumed, so the ring is free
        const int q = warp & 3;
        if (__all_sync(0xffffffffu, mbar_wait(bar_done, 0, wc, SITE_TMEM_FULL, tile))) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < N; c += 32) {
                if (tok0 + c >= g.T) break;
                uint32_t r[32];
                tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, r);
                tmem_ld_wait(r);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < N)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring + ((c + j) * 128 + q * 32 + lane) * 4), "r"(r[j])
                                     : "memory");
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    {
        constexpr int PAIRS = GATED ? 32 : 64;  // pairs of neighbouring output columns of a tile
        const int count = min(N, g.T - tok0) * PAIRS;
        for (int e = rank * ROWS_THREADS + threadIdx.x; e < count; e += S * ROWS_THREADS) {
            const int n = e / PAIRS, p = e % PAIRS;
            const int col = tile * (2 * PAIRS) + 2 * p;
            const uint32_t at = ring + (n * 128 + 2 * p) * 4;
            float2 a = make_float2(0.f, 0.f), b = make_float2(0.f, 0.f);
            for (int s = 0; s < S; ++s) {
                const uint32_t peer = mapa_shared(at, s);
                const float2 v = ld_cluster_f2(peer);
                a.x += v.x;
                a.y += v.y;
                if (GATED) {
                    const float2 u = ld_cluster_f2(peer + 64 * 4);
                    b.x += u.x;
                    b.y += u.y;
                }
            }
            if (col >= g.cols) continue;
            const size_t row = static_cast<size_t>(tok0 + n);
            if (GATED) {
                if (g.gu != nullptr) {
                    float* gu = g.gu + row * (2 * static_cast<size_t>(g.cols)) + col;
                    *reinterpret_cast<float2*>(gu) = a;
                    *reinterpret_cast<float2*>(gu + g.cols) = b;
                }
                a.x = a.x * sigmoid_f(a.x) * b.x;
                a.y = a.y * sigmoid_f(a.y) * b.y;
            }
            *reinterpret_cast<uint32_t*>(g.out + row * g.cols + col) = pack_bf16x2(a.x, a.y);
        }
    }
    // a CTA's partial sums stay until every peer has read them
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        if (*abort_sm) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) {
            }
        }
        tmem_dealloc<1>(tmem, C::TMEM);
    }
}

// --------------------------------------------------------------------------------------------
// host side

// K-major operand [rows, K] or MN-major operand [K, cols]; `box` rows of a K-major one
static int operand_map(CUtensorMap* map, const void* p, bool mn, int rows_or_cols, int K, int box) {
    if (mn) return make_tmap_2d(map, p, 2, rows_or_cols, K, static_cast<uint64_t>(rows_or_cols) * 2, 64, BK);
    return make_tmap_2d(map, p, 2, K, rows_or_cols, static_cast<uint64_t>(K) * 2, BK, box);
}

template <bool A_MN, bool B_MN, int EPI, int PAIR>
static int launch(const Maps& maps, const Args& g, cudaStream_t st) {
    const auto kernel = ffn_gemm_kernel<A_MN, B_MN, EPI, PAIR>;
    static bool attr_set[64] = {false};
    int dev = 0, sms = 0;
    DK_CUDA_OK(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        DK_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<PAIR>::SMEM_BYTES));
        attr_set[dev & 63] = true;
    }
    const int rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const int64_t tiles = static_cast<int64_t>(g.tiles_m) * g.tiles_n;
    const int units = sms / PAIR;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<int>(tiles < units ? tiles : units) * PAIR);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Cfg<PAIR>::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    DK_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, maps, g));
    return DK_OK;
}

// Two-CTA tiles unless more than one row tile in nine would be computed for nothing.
static bool use_pair(int M) {
    const int tiles = (M + BM - 1) / BM;
    return tiles % 2 == 0 || tiles >= 9;
}

// D[M,N] = A B. GATED: B = W13 [2N, K], D = h. DGATED: D = dgu [M, 2N].
template <bool A_MN, bool B_MN, int EPI>
static int product(const void* A, const void* B, void* D, int M, int N, int K, void* gu, cudaStream_t st) {
    Maps maps;
    Args g{};
    const int pair = use_pair(M) ? 2 : 1;
    int rc = operand_map(&maps.a, A, A_MN, M, K, BM);
    if (rc != DK_OK) return rc;
    rc = operand_map(&maps.b, B, B_MN, EPI == EPI_GATED ? 2 * N : N, K, EPI == EPI_GATED ? 128 : BN / pair);
    if (rc != DK_OK) return rc;
    // a map counts bf16 units: `words` of them to an element
    auto out = [&](int i, void* p, uint64_t stride, int words) {
        return make_tmap_2d(&maps.out[i], p, 2, static_cast<uint64_t>(N) * words, M, stride, 64, 32);
    };
    const uint64_t n = static_cast<uint64_t>(N);
    if (EPI == EPI_DGATED) {
        rc = out(0, D, 4 * n, 1);
        if (rc == DK_OK) rc = out(1, static_cast<__nv_bfloat16*>(D) + n, 4 * n, 1);
    } else {
        rc = out(0, D, 2 * n, 1);
        if (EPI == EPI_GATED && gu != nullptr) {
            if (rc == DK_OK) rc = out(1, gu, 8 * n, 2);
            if (rc == DK_OK) rc = out(2, static_cast<float*>(gu) + n, 8 * n, 2);
        }
    }
    if (rc != DK_OK) return rc;
    g.M = M;
    g.N = N;
    g.num_kb = (K + BK - 1) / BK;
    g.tiles_m = (M + BM * pair - 1) / (BM * pair);
    g.tiles_n = (N + (EPI == EPI_GATED ? 128 : BN) - 1) / (EPI == EPI_GATED ? 128 : BN);
    g.group_m = 16 / pair;
    g.save = EPI == EPI_GATED && gu != nullptr;
    g.gu = static_cast<const float*>(gu);
    rc = device_status_ptr(&g.status);
    if (rc != DK_OK) return rc;
    return pair == 2 ? launch<A_MN, B_MN, EPI, 2>(maps, g, st) : launch<A_MN, B_MN, EPI, 1>(maps, g, st);
}

template <bool GATED, int N>
static int launch_rows(const RowsMaps& maps, const RowsArgs& g, int tiles, int S, cudaStream_t st) {
    using C = RowsCfg<N>;
    const auto kernel = ffn_rows_kernel<GATED, N>;
    static bool attr_set[64] = {false};
    int dev = 0;
    DK_CUDA_OK(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        DK_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
        attr_set[dev & 63] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * S, (g.T + N - 1) / N);
    cfg.blockDim = dim3(ROWS_THREADS);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    // the second product overlaps the end of the first, which is the kernel before it on the stream
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = GATED ? 1 : 2;
    DK_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, maps, g));
    return DK_OK;
}

// out [T, cols] = x W^T for few rows; GATED: W = W13, out = h
template <bool GATED>
static int rows_product(const void* x, const void* W, void* out, int T, int cols, int K, void* gu, cudaStream_t st) {
    int sms = 0;
    int rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const int N = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
    RowsMaps maps;
    rc = make_tmap_2d(&maps.w, W, 2, K, GATED ? 2 * cols : cols, static_cast<uint64_t>(K) * 2, BK, GATED ? 64 : 128);
    if (rc == DK_OK) rc = make_tmap_2d(&maps.x, x, 2, K, T, static_cast<uint64_t>(K) * 2, BK, N);
    if (rc != DK_OK) return rc;
    RowsArgs g{};
    g.T = T;
    g.cols = cols;
    g.num_kb = (K + BK - 1) / BK;
    g.out = static_cast<__nv_bfloat16*>(out);
    g.gu = static_cast<float*>(gu);
    rc = device_status_ptr(&g.status);
    if (rc != DK_OK) return rc;
    const int tiles = (cols + (GATED ? 64 : 128) - 1) / (GATED ? 64 : 128);
    // cut K while the CTAs still run all at once and each keeps a few K blocks
    const int places = sms * (N <= 128 ? 2 : 1);
    int S = 1;
    while (S < 8 && tiles * S * 2 * ((T + N - 1) / N) <= places && g.num_kb / (S * 2) >= 4) S *= 2;
    switch (N) {
        case 16: return launch_rows<GATED, 16>(maps, g, tiles, S, st);
        case 32: return launch_rows<GATED, 32>(maps, g, tiles, S, st);
        case 64: return launch_rows<GATED, 64>(maps, g, tiles, S, st);
        case 128: return launch_rows<GATED, 128>(maps, g, tiles, S, st);
        default: return launch_rows<GATED, 256>(maps, g, tiles, S, st);
    }
}

// Few rows: see ffn_rows_kernel.
constexpr int ROWS_MAX_T = 256;

static int check_shape(int T, int H, int F) {
    DK_REQUIRE(T >= 0, "the number of rows must not be negative");
    DK_REQUIRE(H >= 8 && F >= 8 && H % 8 == 0 && F % 8 == 0, "H and F must be positive multiples of 8");
    DK_REQUIRE(T <= (1 << 24) && H <= (1 << 20) && F <= (1 << 20), "at most 2^24 rows and widths of 2^20");
    return DK_OK;
}

}  // namespace ffn
}  // namespace dk

extern "C" int dk_gated_ffn(const void* x, const void* w13, const void* w2, int T, int H, int F, void* gu, void* h, void* y,
                            void* stream) {
    using namespace dk;
    using namespace dk::ffn;
    int rc = check_shape(T, H, F);
    if (rc != DK_OK) return rc;
    DK_REQUIRE(w13 != nullptr && w2 != nullptr, "null operand");
    if (T == 0) return DK_OK;
    DK_REQUIRE(x != nullptr && h != nullptr && y != nullptr, "null operand");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DK_REQUIRE(((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(gu)) & 15) == 0,
               "h, y and gu must be 16-byte aligned");
    if (T <= ROWS_MAX_T) {
        rc = rows_product<true>(x, w13, h, T, F, H, gu, st);
        if (rc != DK_OK) return rc;
        return rows_product<false>(h, w2, y, T, H, F, nullptr, st);
    }
    rc = product<false, false, EPI_GATED>(x, w13, h, T, F, H, gu, st);
    if (rc != DK_OK) return rc;
    return product<false, false, EPI_STORE>(h, w2, y, T, H, F, nullptr, st);
}

extern "C" int dk_gated_ffn_bwd(const void* dy, const void* x, const void* w13, const void* w2, const void* gu, const void* h,
                                int T, int H, int F, void* dgu, void* dx, void* dw13, void* dw2, void* stream) {
    using namespace dk;
    using namespace dk::ffn;
    int rc = check_shape(T, H, F);
    if (rc != DK_OK) return rc;
    DK_REQUIRE(w13 != nullptr && w2 != nullptr && dw13 != nullptr && dw2 != nullptr, "null operand");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        DK_CUDA_OK(cudaMemsetAsync(dw13, 0, static_cast<size_t>(F) * H * 4, st));
        DK_CUDA_OK(cudaMemsetAsync(dw2, 0, static_cast<size_t>(F) * H * 2, st));
        return DK_OK;
    }
    DK_REQUIRE((reinterpret_cast<uintptr_t>(gu) & 15) == 0, "gu must be 16-byte aligned");
    DK_REQUIRE(dy != nullptr && x != nullptr && gu != nullptr && h != nullptr && dgu != nullptr && dx != nullptr, "null operand");
    // dh = dy W2 (K = H, W2 [H,F] is [K,N]), straight into dg and du
    rc = product<false, true, EPI_DGATED>(dy, w2, dgu, T, F, H, const_cast<void*>(gu), st);
    if (rc == DK_OK) rc = product<false, true, EPI_STORE>(dgu, w13, dx, T, H, 2 * F, nullptr, st);
    if (rc == DK_OK) rc = product<true, true, EPI_STORE>(dgu, x, dw13, 2 * F, H, T, nullptr, st);
    if (rc == DK_OK) rc = product<true, true, EPI_STORE>(dy, h, dw2, H, F, T, nullptr, st);
    return rc;
}
