// Gated feed-forward block and its backward pass, bf16, for sm_100a.
//
//   [g | u] = x W13^T        x [T,H], W13 [2F,H] (F gate rows, then F up rows, as in the MoE layer)
//   h = silu(g) * u          silu(g) = g * s, s = 1 / (1 + exp(-g))
//   y = h W2^T               W2 [H,F]
//
//   dh = dy W2,  dg = dh * u * s * (1 + g * (1 - s)),  du = dh * g * s
//   dx = [dg|du] W13,  dW13 = [dg|du]^T x,  dW2 = dy^T h
//
// One kernel serves all six products, D[M,N] = A B with fp32 accumulation in tensor memory. Its operands lie in
// memory K-major ([M,K] and [N,K], the weights of a forward pass) or MN-major ([K,M] and [K,N]: W2 and W13 seen from
// the other side, and the token axis as K in the weight gradients), which the tensor core reads through a
// descriptor of its own, so nothing is transposed in memory. What it does with a finished tile:
//   EPI_STORE   bf16 rows of D
//   EPI_GATED   the B tile is as many gate rows as up rows, so a thread holds g and u of the same
//               place: silu(g) * u leaves as h, and g, u too when a backward pass will follow
//   EPI_DGATED  D is dh: with the kept g, u of the same place, dg and du leave
// A launch takes up to three products of one kind, their tiles in one list: dx, dW13 and dW2 need no launch of their
// own, and the last wave of one is filled by the next.
// h, dg and du are rounded to bf16, the type in which the tensor core takes them up again. g and u are kept in
// 32 bits: dx and dW13 then carry two roundings, [dg|du] and their own (error against 64 bits 0.0024); kept in bf16
// their roundings entered too (0.0030). The price is 8 bytes a value of h instead of 4, written and read beside
// matrix products.
//
//   warp 0      TMA producer: 128-byte-swizzled boxes into a ring of stages
//   warp 1      an elected thread issues tcgen05.mma into one of two 256-column accumulators
//   warps 2-5   epilogue: tcgen05.ld, swizzled staging in shared memory, TMA stores (which clip the
//               ragged edges)
//
// PAIR = 2: a cluster of two CTAs per 256x256 tile (cta_group::2). Each stages its 128 rows of A and half of
// the B tile (gated: CTA 0 the gate rows, CTA 1 the up rows), so a stage is 32 KiB instead of 48, the ring six
// deep instead of four, and a flop needs two thirds of the shared-memory fill. Both CTAs' loads complete on the
// leader's barrier, the leader issues the MMAs. PAIR = 1: one CTA per tile of 128 rows, where pairs would leave
// rows or a last wave half empty (choose()).
//
// Few rows go by a kernel of their own with the weights as A, ffn_rows_kernel below; few_rows() says when.
#include "dk_host.h"
#include "dk_launch.cuh"
#include "dk_ptx.cuh"

#include <algorithm>
#include <initializer_list>

namespace dk {

namespace ffn {

constexpr int BM = 128;
constexpr int BN_MAX = 256;  // a tile is 256, 192 or 128 columns wide, see choose()
constexpr int BK = 64;  // 64 bf16 = 128 bytes = one swizzle row
constexpr int UMMA_K = 16;
constexpr int A_BYTES = BM * BK * 2;
constexpr int MN_BLOCK = 64 * BK * 2;  // an MN-major box: 64 elements of M or N (128 bytes) x 64 of K
constexpr int EPI_BUF = 32 * 128;      // 32 rows x 64 bf16
constexpr int EPI_BYTES = 4 * 2 * EPI_BUF;
constexpr int RING_BYTES = 192 * 1024;  // as many stages as fit: 6 of 256 columns a pair, 8 of 128
constexpr int MAX_STAGES = 8;
constexpr int SMEM_BYTES = 1024 + RING_BYTES + EPI_BYTES + 256;
constexpr int THREADS = 192;
constexpr int TMEM_COLS = 512;

enum : int { EPI_STORE = 0, EPI_GATED = 1, EPI_DGATED = 2 };
enum : unsigned { SITE_EMPTY = 101, SITE_FULL = 102, SITE_TMEM_EMPTY = 103, SITE_TMEM_FULL = 104 };

constexpr int MAX_PRODUCTS = 3;
struct Maps {
    CUtensorMap a[MAX_PRODUCTS], b[MAX_PRODUCTS];
    CUtensorMap out[MAX_PRODUCTS];  // STORE: D of each product; GATED: h, g, u
};

struct Product {
    int M, N, num_kb;               // N: columns of the output (GATED, DGATED: F)
    int tiles_m, tiles_n, group_m;  // tiles of 128 * PAIR rows
    int first;                      // the product's first tile in the launch's list
    int a_mn, b_mn;
};
struct Args {
    Product p[MAX_PRODUCTS];
    int products, num_tiles;
    int bn;           // width of the B tile (GATED: gate and up rows together)
    int save;         // GATED: g and u leave too
    const float* gu;     // DGATED: kept [g|u], [M, 2N]
    __nv_bfloat16* dgu;  // DGATED: [dg|du], [M, 2N]
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

// Tile t of the list -> its product and place. Column tiles run slowest inside a group of group_m row tiles, so
// that CTAs running together share operand tiles in L2.
__device__ __forceinline__ int tile_coords(int t, const Args& g, int& m, int& n) {
    int i = 0;
    while (i + 1 < g.products && t >= g.p[i + 1].first) ++i;
    const Product& p = g.p[i];
    t -= p.first;
    const int per_group = p.group_m * p.tiles_n;
    const int grp = t / per_group;
    const int first = grp * p.group_m;
    const int gsz = min(p.tiles_m - first, p.group_m);
    const int r = t - grp * per_group;
    m = first + r % gsz;
    n = r / gsz;
    return i;
}

__device__ __forceinline__ float sigmoid_f(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// dg, du of one value of h from dh and the kept g, u
__device__ __forceinline__ void d_gated(float dh, float gate, float up, float& dg, float& du) {
    const float s = sigmoid_f(gate);
    du = dh * gate * s;
    dg = dh * up * s * (1.0f + gate * (1.0f - s));
}

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
__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// The kept values of a warp's 32 rows x 32 columns: read from global memory whole lines at a time (eight lanes to a row of
// 128 bytes), then handed out through shared memory, a row to a lane. (A lane reading its own row touches 32 lines with
// every load; a step of 1357 rows of 2048 x 3592 then takes 230 us instead of 222.)
struct Kept {
    uint4 v[8];
    __device__ __forceinline__ void load(const float* p, size_t stride, int lane, int rows, int cols) {
        const int c = (lane & 7) * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + (lane >> 3);
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows && c < cols) v[i] = *reinterpret_cast<const uint4*>(p + row * stride + c);
        }
    }
    __device__ __forceinline__ void stage(uint32_t buf, int lane) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + (lane >> 3);
            st_shared16(buf + row * 128 + (((lane & 7) ^ (row & 7)) << 4), v[i]);
        }
    }
};
__device__ __forceinline__ void staged_row(uint32_t buf, int lane, float (&f)[32]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint4 v = ld_shared16(buf + lane * 128 + ((j ^ (lane & 7)) << 4));
        f[4 * j] = __uint_as_float(v.x);
        f[4 * j + 1] = __uint_as_float(v.y);
        f[4 * j + 2] = __uint_as_float(v.z);
        f[4 * j + 3] = __uint_as_float(v.w);
    }
}
// A lane's row of 32 bf16 into a 32 x 64-byte buffer, and from there to global memory, four lanes to a row.
__device__ __forceinline__ void stage_row(uint32_t buf, int lane, const float (&f)[32]) {
    uint32_t p[16];
    pack32(f, p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        st_shared16(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4),
                    make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]));
}
__device__ __forceinline__ void store_rows(uint32_t buf, __nv_bfloat16* p, size_t stride, int lane, int rows, int cols) {
    const int j = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2);
        const uint4 v = ld_shared16(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4));
        if (row < rows && 8 * j < cols) *reinterpret_cast<uint4*>(p + row * stride + 8 * j) = v;
    }
}

template <int EPI, int PAIR>
__global__ void __launch_bounds__(THREADS, 1) ffn_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    const int bn = g.bn;
    const int stage_bytes = A_BYTES + bn / PAIR * (BK * 2), stages = min(MAX_STAGES, RING_BYTES / stage_bytes);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem_base;
    const uint32_t epi = smem_base + RING_BYTES;
    const uint32_t ctrl = epi + EPI_BYTES;
    uint8_t* ctrl_p = smem_raw + (ctrl - smem_u32(smem_raw));
    const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * MAX_STAGES;
    const uint32_t bar_tfull = ctrl + 16 * MAX_STAGES, bar_tempty = bar_tfull + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl_p + 16 * MAX_STAGES + 32);
    volatile int* abort_sm = reinterpret_cast<volatile int*>(ctrl_p + 16 * MAX_STAGES + 40);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{g.status, abort_sm};
    const int crank = PAIR == 2 ? static_cast<int>(cluster_ctarank()) : 0;
    const int unit = blockIdx.x / PAIR, nunits = gridDim.x / PAIR;
    const int num_tiles = g.num_tiles;

    if (threadIdx.x == 0) {
        *abort_sm = 0;
        for (int s = 0; s < stages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + 8 * a, 1);
            mbar_init(bar_tempty + 8 * a, 128 * PAIR);  // the leader hears both CTAs' epilogues
        }
        fence_mbar_init();
        for (int i = 0; i < g.products; ++i) {
            tma_prefetch_desc(&maps.a[i]);
            tma_prefetch_desc(&maps.b[i]);
        }
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
    next_may_begin();
    previous_done();

    // Producer and issuer run their loops as whole warps and elect one thread for the instructions themselves: what
    // the instructions take (descriptors, coordinates, barriers) then stays in uniform registers. With one thread
    // in the loops a stage of 64 of K took 0.37 us to issue whatever its width; now 0.27 (128 columns).
    if (warp == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");  // what earlier kernels wrote, for the copy engine
        const int b_rows = bn / PAIR;
        const uint32_t tx = A_BYTES + b_rows * BK * 2;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += nunits) {
            int m, n;
            const int pi = tile_coords(t, g, m, n);
            const Product& p = g.p[pi];
            m = m * PAIR + crank;  // this CTA's 128-row tile
            for (int kb = 0; kb < p.num_kb; ++kb) {
                if (!__all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph ^ 1, wc, SITE_EMPTY, t))) {
                    ok = false;
                    break;
                }
                const uint32_t sa = ring + s * stage_bytes, sb = sa + A_BYTES;
                // a pair's loads complete on the leader's barrier, which expects the bytes of both CTAs
                const uint32_t full = PAIR == 2 ? mapa_shared(bar_full + 8 * s, 0) : bar_full + 8 * s;
                if (elect_one()) {
                    if (crank == 0) mbar_expect_tx(bar_full + 8 * s, PAIR * tx);
                    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                        if (PAIR == 2) tma_load_2d_pair(dst, map, full, x, y);
                        else tma_load_2d(dst, map, full, x, y);
                    };
                    if (p.a_mn) {
                        for (int i = 0; i < BM / 64; ++i) load(sa + i * MN_BLOCK, &maps.a[pi], m * BM + 64 * i, kb * BK);
                    } else {
                        load(sa, &maps.a[pi], kb * BK, m * BM);
                    }
                    if (EPI == EPI_GATED) {
                        // gate rows that do not exist read up rows instead, up rows zeros: not stored
                        const int half = bn / 2;
                        if (PAIR == 2) {
                            load(sb, &maps.b[0], kb * BK, crank * p.N + n * half);
                        } else {
                            load(sb, &maps.b[0], kb * BK, n * half);
                            load(sb + half * BK * 2, &maps.b[0], kb * BK, p.N + n * half);
                        }
                    } else if (p.b_mn) {
                        for (int i = 0; i < b_rows / 64; ++i)
                            load(sb + i * MN_BLOCK, &maps.b[pi], n * bn + crank * b_rows + 64 * i, kb * BK);
                    } else {
                        load(sb, &maps.b[pi], kb * BK, n * bn + crank * b_rows);
                    }
                }
                if (++s == stages) {
                    s = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (crank == 0) {
            const uint32_t idesc0 = umma_idesc(1, 1, BM * PAIR, bn);
            int s = 0, acc = 0;
            uint32_t ph = 0, acc_ph = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += nunits) {
                if (!__all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * acc, acc_ph ^ 1, wc, SITE_TMEM_EMPTY, t))) break;
                tc_fence_after();
                int m, n;
                const Product& p = g.p[tile_coords(t, g, m, n)];
                const bool a_mn = p.a_mn != 0, b_mn = p.b_mn != 0;
                const uint32_t idesc = idesc0 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
                // descriptor steps of 16 elements of K, in 16-byte units: 32 bytes along the swizzle row, or
                // 16 rows of 128 bytes
                const uint64_t a_step = a_mn ? 16 * 128 / 16 : 2, b_step = b_mn ? 16 * 128 / 16 : 2;
                const uint32_t d_tmem = tmem_base + acc * BN_MAX;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    if (!__all_sync(0xffffffffu, mbar_wait(bar_full + 8 * s, ph, wc, SITE_FULL, t))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = ring + s * stage_bytes, sb = sa + A_BYTES;
                    const uint64_t da = a_mn ? desc_mn(sa) : umma_desc_sw128(sa);
                    const uint64_t db = b_mn ? desc_mn(sb) : umma_desc_sw128(sb);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)
                            umma_f16<PAIR>(d_tmem, da + a_step * k, db + b_step * k, idesc, (kb | k) != 0);
                        // the stage is free in both CTAs once these MMAs have read it
                        if (PAIR == 2) umma_commit_pair(bar_empty + 8 * s, 3);
                        else umma_commit<1>(bar_empty + 8 * s);
                    }
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) break;
                if (elect_one()) {
                    if (PAIR == 2) umma_commit_pair(bar_tfull + 8 * acc, 3);
                    else umma_commit<1>(bar_tfull + 8 * acc);
                }
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
        int rows = 0, cols = 0;  // of the current tile's product
        auto send = [&](uint32_t buf, const CUtensorMap* map, int col, int row, int words = 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (col < cols && row < rows) tma_store_2d(map, buf, col * words, row);
                tma_store_commit();
            }
        };
        for (int t = unit; t < num_tiles; t += nunits) {
            int m, n;
            const int pi = tile_coords(t, g, m, n);
            rows = g.p[pi].M;
            cols = g.p[pi].N;
            const int row0 = (m * PAIR + crank) * BM + q * 32;
            Kept gate_in, up_in;  // DGATED: of the next 32 columns
            const size_t wide = 2 * static_cast<size_t>(cols);
            auto fetch_kept = [&](int col) {
                const float* from = g.gu + static_cast<size_t>(row0) * wide + col;
                gate_in.load(from, wide, lane, rows - row0, cols - col);
                up_in.load(from + cols, wide, lane, rows - row0, cols - col);
            };
            if constexpr (EPI == EPI_DGATED) fetch_kept(n * bn);
            if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, acc_ph, wc, SITE_TMEM_FULL, t))) break;
            tc_fence_after();
            const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN_MAX;
            if constexpr (EPI == EPI_STORE) {
#pragma unroll 1
                for (int c = 0; c < bn / 64; ++c) {
                    const uint32_t buf = next_buf();
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        float f[32];
                        uint32_t p[16];
                        ld_acc(t_acc + c * 64 + hi * 32, f);
                        pack32(f, p);
                        stage_half(buf, lane, hi, p);
                    }
                    send(buf, &maps.out[pi], n * bn + c * 64, row0);
                }
            } else if constexpr (EPI == EPI_GATED) {
#pragma unroll 1
                for (int c = 0; c < bn / 128; ++c) {
                    const int half = bn / 2, col = n * half + c * 64;
                    if (g.save) {
#pragma unroll 1
                        for (int part = 0; part < 4; ++part) {  // gate, up of 32 columns, gate, up of the next 32
                            const int sub = (part & 1) * half + c * 64 + (part >> 1) * 32;
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
                        ld_acc(t_acc + half + c * 64 + hi * 32, up);
#pragma unroll
                        for (int i = 0; i < 32; ++i) gate[i] = gate[i] * sigmoid_f(gate[i]) * up[i];
                        pack32(gate, p);
                        stage_half(buf, lane, hi, p);
                    }
                    send(buf, &maps.out[0], col, row0);
                }
            } else {
                const uint32_t buf_g = my_epi, buf_u = my_epi + EPI_BUF;
                const int units = bn / 32;
#pragma unroll 1
                for (int c = 0; c < units; ++c) {
                    const int col = n * bn + c * 32;
                    float gate[32], up[32], dh[32];
                    gate_in.stage(buf_g, lane);
                    up_in.stage(buf_u, lane);
                    if (c + 1 < units) fetch_kept(col + 32);
                    __syncwarp();
                    staged_row(buf_g, lane, gate);
                    staged_row(buf_u, lane, up);
                    ld_acc(t_acc + c * 32, dh);
#pragma unroll
                    for (int i = 0; i < 32; ++i) d_gated(dh[i], gate[i], up[i], gate[i], dh[i]);
                    __syncwarp();  // every lane has its kept values
                    stage_row(buf_g, lane, gate);
                    stage_row(buf_u, lane, dh);
                    __syncwarp();
                    __nv_bfloat16* to = g.dgu + static_cast<size_t>(row0) * wide + col;
                    store_rows(buf_g, to, wide, lane, rows - row0, cols - col);
                    store_rows(buf_u, to + cols, wide, lane, rows - row0, cols - col);
                    __syncwarp();
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
// swapped: 128 weight rows are the tensor core's M, the tokens its N (16 to 256, in steps of 16), so a tile is 16 KB of
// weights per 64 of K whatever the number of tokens, and F / 64 or H / 128 tiles are cut along K over a cluster
// of S CTAs until there are enough CTAs to draw on all of HBM. Each CTA leaves its fp32 partial sums in its own
// shared memory; the cluster's CTAs then add up each other's through distributed shared memory, in rank order: no
// workspace, no second launch, the same bits on every run.
//   EPI_GATED   a tile is 64 gate rows and the 64 up rows of the same columns; silu(g) * u leaves as h
//   EPI_STORE   y from h and W2, or dx from [dg|du] and W13 (MN-major: 128 columns of W13)
//   EPI_DGATED  dh from dy and W2 (MN-major: 128 columns of W2), with the kept g, u straight into dg, du
// A product that follows another of the same call fills its ring with weights while that one ends. (More of them sent
// to L2 ahead gained nothing: HBM is busy from the first CTA's start.)
constexpr int ROWS_THREADS = 192;
constexpr int ROWS_W_BYTES = 128 * BK * 2;
// Shared memory of the ring: two CTAs on an SM up to 128 tokens, one above. The partial sums reuse it: N * 512 bytes.
constexpr int ROWS_MAX_STAGES = 8;
__host__ __device__ constexpr int rows_ring(int N) { return N <= 128 ? 110 * 1024 : 208 * 1024; }
constexpr int rows_smem(int N) { return 1024 + rows_ring(N) + 256; }
static_assert(128 * 512 <= rows_ring(128) && 256 * 512 <= rows_ring(256), "the partial sums reuse the ring");
struct RowsMaps {
    CUtensorMap w, x;
};
struct RowsArgs {
    int N;                // tokens of a tile, a multiple of 16
    int weights_ready;    // the kernel before this one belongs to the same call
    int T, cols, num_kb;  // cols: columns of the output (GATED, DGATED: F)
    __nv_bfloat16* out;   // [T, cols]; DGATED: [T, 2 cols]
    float* gu;            // [T, 2 cols]; GATED: written, may be null; DGATED: read
    unsigned* status;
};
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

template <int EPI, bool W_MN>
__global__ void __launch_bounds__(ROWS_THREADS) ffn_rows_kernel(const __grid_constant__ RowsMaps maps, const RowsArgs g) {
    const int N = g.N, stage = ROWS_W_BYTES + N * BK * 2, stages = min(ROWS_MAX_STAGES, rows_ring(N) / stage);
    const int tmem_cols = N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;  // a power of two
    constexpr bool GATED = EPI == EPI_GATED;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ctrl = ring + rows_ring(N);
    uint8_t* ctrl_p = smem_raw + (ctrl - smem_u32(smem_raw));
    const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * ROWS_MAX_STAGES, bar_done = ctrl + 16 * ROWS_MAX_STAGES;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl_p + 16 * ROWS_MAX_STAGES + 8);
    volatile int* abort_sm = reinterpret_cast<volatile int*>(ctrl_p + 16 * ROWS_MAX_STAGES + 16);

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
        for (int s = 0; s < stages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_done, 1);
        fence_mbar_init();
        tma_prefetch_desc(&maps.w);
        tma_prefetch_desc(&maps.x);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto meet = [&]() {  // of the cluster's CTAs, every thread of them
        if (S == 1) {
            __syncthreads();
        } else {
            __syncwarp();
            cluster_arrive();
            cluster_wait();
        }
    };

    if (warp == 0) {  // whole warps, one elected thread: as in ffn_gemm_kernel
        auto load_w = [&](int kb, int s) {
            const uint32_t sw = ring + s * stage, full = bar_full + 8 * s;
            mbar_expect_tx(full, stage);
            if (GATED) {
                // gate rows that do not exist read up rows instead, up rows zeros: not stored
                tma_load_2d(sw, &maps.w, full, kb * BK, tile * 64);
                tma_load_2d(sw + ROWS_W_BYTES / 2, &maps.w, full, kb * BK, g.cols + tile * 64);
            } else if (W_MN) {
                tma_load_2d(sw, &maps.w, full, tile * 128, kb * BK);
                tma_load_2d(sw + MN_BLOCK, &maps.w, full, tile * 128 + 64, kb * BK);
            } else {
                tma_load_2d(sw, &maps.w, full, kb * BK, tile * 128);
            }
        };
        auto load_x = [&](int kb, int s) {
            tma_load_2d(ring + s * stage + ROWS_W_BYTES, &maps.x, bar_full + 8 * s, kb * BK, tok0);
        };
        const int ahead = min(kb1 - kb0, stages);
        if (elect_one()) {
            // A kernel of the same call writes no weights, and it let this one begin only when all before it was complete:
            // the ring takes its first stages of weights while that kernel ends.
            for (int i = 0; i < ahead && g.weights_ready; ++i) load_w(kb0 + i, i);
        }
        __syncwarp();
        previous_done();
        next_may_begin();  // not before: the next kernel may load weights at once
        asm volatile("fence.proxy.async;" ::: "memory");  // what earlier kernels wrote, for the copy engine
        if (elect_one()) {
            for (int i = 0; i < ahead; ++i) {
                if (!g.weights_ready) load_w(kb0 + i, i);
                load_x(kb0 + i, i);
            }
        }
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0 + ahead; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * s, ph, wc, SITE_EMPTY, tile))) break;
            if (elect_one()) {
                load_w(kb, s);
                load_x(kb, s);
            }
            if (++s == stages) {
                s = 0;
                ph ^= 1;
            }
        }
    } else if (warp == 1) {
        previous_done();  // before any bounded wait: its limit is not for the kernel before
        const uint32_t idesc = umma_idesc(1, 1, 128, N) | (W_MN ? 1u << 15 : 0u);
        constexpr uint64_t w_step = W_MN ? 16 * 128 / 16 : 2;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar_full + 8 * s, ph, wc, SITE_FULL, tile))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint64_t da = W_MN ? desc_mn(ring + s * stage) : umma_desc_sw128(ring + s * stage);
            const uint64_t db = umma_desc_sw128(ring + s * stage + ROWS_W_BYTES);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)
                    umma_f16<1>(tmem, da + w_step * k, db + 2 * k, idesc, kb != kb0 || k != 0);
                umma_commit<1>(bar_empty + 8 * s);
            }
            if (++s == stages) {
                s = 0;
                ph ^= 1;
            }
        }
        if (ok && elect_one()) umma_commit<1>(bar_done);
    } else {
        // partial sums as [token][weight row]; every load has been consumed, so the ring is free
        previous_done();
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
    meet();
    {
        constexpr int PAIRS = GATED ? 32 : 64;  // pairs of neighbouring output columns of a tile
        const int count = min(N, g.T - tok0) * PAIRS;
        // U elements a turn, so that their loads (a peer's shared memory, the kept g and u) are in flight together
        constexpr int U = 4;
        const int step = S * ROWS_THREADS;
        for (int e0 = rank * ROWS_THREADS + threadIdx.x; e0 < count; e0 += U * step) {
            float2 a[U], b[U], gate[U], up[U];
            uint32_t at[U];
            size_t place[U];  // of the output, and of g in [g|u]
            bool ok[U];
            const size_t wide = EPI == EPI_STORE ? g.cols : 2 * static_cast<size_t>(g.cols);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int e = e0 + i * step, n = e / PAIRS, p = e % PAIRS;
                const int col = tile * (2 * PAIRS) + 2 * p;
                ok[i] = e < count && col < g.cols;
                at[i] = ring + (n * 128 + 2 * p) * 4;
                place[i] = static_cast<size_t>(tok0 + n) * wide + col;
                a[i] = make_float2(0.f, 0.f);
                b[i] = make_float2(0.f, 0.f);
                if (EPI == EPI_DGATED && ok[i]) {
                    gate[i] = *reinterpret_cast<const float2*>(g.gu + place[i]);
                    up[i] = *reinterpret_cast<const float2*>(g.gu + place[i] + g.cols);
                }
            }
            for (int s = 0; s < S; ++s) {
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    if (!ok[i]) continue;
                    const uint32_t peer = mapa_shared(at[i], s);
                    const float2 v = ld_cluster_f2(peer);
                    a[i].x += v.x;
                    a[i].y += v.y;
                    if (GATED) {
                        const float2 u = ld_cluster_f2(peer + 64 * 4);
                        b[i].x += u.x;
                        b[i].y += u.y;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (!ok[i]) continue;
                if (EPI == EPI_DGATED) {
                    float2 dg, du;
                    d_gated(a[i].x, gate[i].x, up[i].x, dg.x, du.x);
                    d_gated(a[i].y, gate[i].y, up[i].y, dg.y, du.y);
                    *reinterpret_cast<uint32_t*>(g.out + place[i]) = pack_bf16x2(dg.x, dg.y);
                    *reinterpret_cast<uint32_t*>(g.out + place[i] + g.cols) = pack_bf16x2(du.x, du.y);
                    continue;
                }
                size_t to = place[i];
                if (GATED) {
                    if (g.gu != nullptr) {
                        *reinterpret_cast<float2*>(g.gu + place[i]) = a[i];
                        *reinterpret_cast<float2*>(g.gu + place[i] + g.cols) = b[i];
                    }
                    a[i].x = a[i].x * sigmoid_f(a[i].x) * b[i].x;
                    a[i].y = a[i].y * sigmoid_f(a[i].y) * b[i].y;
                    const int n = (e0 + i * step) / PAIRS;
                    to -= static_cast<size_t>(tok0 + n) * g.cols;  // h has rows of half that width
                }
                *reinterpret_cast<uint32_t*>(g.out + to) = pack_bf16x2(a[i].x, a[i].y);
            }
        }
    }
    // a CTA's partial sums stay until every peer has read them
    meet();
    if (warp == 1) {
        tc_fence_after();
        if (*abort_sm) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) {
            }
        }
        tmem_dealloc<1>(tmem, tmem_cols);
    }
}

// --------------------------------------------------------------------------------------------
// host side

// K-major operand [rows, K] or MN-major operand [K, cols]; `box` rows of a K-major one
static int operand_map(CUtensorMap* map, const void* p, bool mn, int rows_or_cols, int K, int box) {
    if (mn) return make_tmap_2d(map, p, 2, rows_or_cols, K, static_cast<uint64_t>(rows_or_cols) * 2, 64, BK);
    return make_tmap_2d(map, p, 2, K, rows_or_cols, static_cast<uint64_t>(K) * 2, BK, box);
}

template <typename K>
static int allow_smem(K kernel, int bytes, bool (&done)[64]) {
    int dev = 0;
    DK_CUDA_OK(cudaGetDevice(&dev));
    if (!done[dev & 63]) {
        DK_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done[dev & 63] = true;
    }
    return DK_OK;
}

template <int EPI, int PAIR>
static int launch(const Maps& maps, const Args& g, cudaStream_t st) {
    const auto kernel = ffn_gemm_kernel<EPI, PAIR>;
    static bool done[64] = {false};
    int sms = 0;
    int rc = allow_smem(kernel, SMEM_BYTES, done);
    if (rc == DK_OK) rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const int units = sms / PAIR;
    return launch_early(kernel, dim3((g.num_tiles < units ? g.num_tiles : units) * PAIR), THREADS, SMEM_BYTES, PAIR, st, maps, g);
}

// One product: D[M,N] = A B. GATED: B = W13 [2N, K], D = h; DGATED: D = dgu [M, 2N].
struct Spec {
    const void *A, *B;
    void* D;
    int M, N, K;
    bool a_mn, b_mn;
};

// How the products of a launch are tiled. A tile's time is its K blocks, each as long as measured with all SMs at work
// (in units of a pair's 256 columns, 0.335 us), and its epilogue, overlapped with the next tile's K blocks:
//   two CTAs    256 columns 1.0   192 columns 0.85   128 columns 0.8
//   one CTA     256 columns 1.1   192 columns 0.95   128 columns 0.75
// Wide pairs are fastest per flop (they load least per flop; 128 columns are bound by shared-memory bandwidth); narrow tiles and single CTAs cut
// the work finer where it would not go evenly into waves, or compute fewer rows for nothing. 192 columns only where
// nothing but a K-major B is loaded and stored.
struct Tiling {
    int pair, bn;
};
static Tiling choose(const Spec* s, int count, int epi, int sms) {
    static const double block[2][3] = {{0.75, 0.95, 1.1}, {0.8, 0.85, 1.0}};
    Tiling best{1, 256};
    double least = 1e300;
    for (int pair = 1; pair <= 2; ++pair)
        for (int bn = 256; bn >= 128; bn -= 64) {
            bool allowed = true;
            double work = 0, longest = 0;
            int64_t tiles = 0;
            const double epilogue = bn * (epi == EPI_STORE ? 0.02 : 0.04);
            for (int i = 0; i < count; ++i) {
                if (bn == 192 && (epi != EPI_STORE || s[i].b_mn)) allowed = false;
                const int rows = BM * pair, cols = epi == EPI_GATED ? bn / 2 : bn;
                const int64_t n = static_cast<int64_t>((s[i].M + rows - 1) / rows) * ((s[i].N + cols - 1) / cols);
                double one = ((s[i].K + BK - 1) / BK) * block[pair - 1][bn / 64 - 2];
                if (one < epilogue) one = epilogue;
                work += n * one;
                tiles += n;
                if (one > longest) longest = one;
            }
            if (!allowed) continue;
            const int units = sms / pair;
            // equal tiles go in whole waves, a mix of them evenly
            const double time = (count == 1 ? ((tiles + units - 1) / units) * longest
                                            : (tiles <= units ? longest : work / units + 0.5 * longest)) + epilogue;
            if (time < least) {
                least = time;
                best = Tiling{pair, bn};
            }
        }
    return best;
}

// gu: GATED: where g and u go (may be null); DGATED: where they come from
template <int EPI>
static int products(const Spec* s, int count, void* gu, cudaStream_t st) {
    int sms = 0;
    int rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const Tiling t = choose(s, count, EPI, sms);
    Maps maps;
    Args g{};
    for (int i = 0; i < count && rc == DK_OK; ++i) {
        Product& p = g.p[i];
        const int bn_out = EPI == EPI_GATED ? t.bn / 2 : t.bn;
        p.M = s[i].M;
        p.N = s[i].N;
        p.num_kb = (s[i].K + BK - 1) / BK;
        p.tiles_m = (p.M + BM * t.pair - 1) / (BM * t.pair);
        p.tiles_n = (p.N + bn_out - 1) / bn_out;
        p.group_m = 16 / t.pair;
        p.first = g.num_tiles;
        p.a_mn = s[i].a_mn;
        p.b_mn = s[i].b_mn;
        const int64_t all = g.num_tiles + static_cast<int64_t>(p.tiles_m) * p.tiles_n;
        DK_REQUIRE(all < (1 << 30), "too many tiles");
        g.num_tiles = static_cast<int>(all);
        rc = operand_map(&maps.a[i], s[i].A, s[i].a_mn, p.M, s[i].K, BM);
        if (rc == DK_OK)
            rc = operand_map(&maps.b[i], s[i].B, s[i].b_mn, EPI == EPI_GATED ? 2 * p.N : p.N, s[i].K,
                             EPI == EPI_GATED ? t.bn / 2 : t.bn / t.pair);
        // a map counts bf16 units: `words` of them to an element
        auto out = [&](int j, void* d, uint64_t stride, int words) {
            if (rc == DK_OK)
                rc = make_tmap_2d(&maps.out[j], d, 2, static_cast<uint64_t>(p.N) * words, p.M, stride, 64, 32);
        };
        const uint64_t n = static_cast<uint64_t>(p.N);
        if (EPI == EPI_DGATED) {
            g.dgu = static_cast<__nv_bfloat16*>(s[i].D);
        } else {
            out(i, s[i].D, 2 * n, 1);
            if (EPI == EPI_GATED && gu != nullptr) {
                out(1, gu, 8 * n, 2);
                out(2, static_cast<float*>(gu) + n, 8 * n, 2);
            }
        }
    }
    if (rc != DK_OK) return rc;
    g.products = count;
    g.bn = t.bn;
    g.save = EPI == EPI_GATED && gu != nullptr;
    g.gu = static_cast<const float*>(gu);
    rc = device_status_ptr(&g.status);
    if (rc != DK_OK) return rc;
    return t.pair == 2 ? launch<EPI, 2>(maps, g, st) : launch<EPI, 1>(maps, g, st);
}

// Tokens of a tile: all of them (up to 256), or near 64, above 256 rows near 96, where the weights come from L2 when they
// are read again, and the shorter epilogue and the larger number of CTAs are worth more (training steps: 140 rows of
// 2048 x 4096 71 us against 80, 256 rows 81 against 95; of 4096 x 4096, 64 MB, 119 against 103). Tiles are equally full.
constexpr size_t SMALL_WEIGHTS = 32u << 20;
static int rows_tokens(int T, size_t weights) {
    int most = 256;
    if (weights <= SMALL_WEIGHTS) most = T <= 256 || weights <= SMALL_WEIGHTS / 2 ? 64 : 96;
    const int tiles = (T + most - 1) / most;
    return ((T + tiles - 1) / tiles + 15) / 16 * 16;
}

// out [T, cols] = x W^T for few rows. GATED: W = W13, out = h; DGATED: x = dy, out = dgu. W_MN: W is [K, cols].
template <int EPI, bool W_MN>
static int rows_product(const void* x, const void* W, void* out, int T, int cols, int K, void* gu, bool follows,
                        cudaStream_t st) {
    const auto kernel = ffn_rows_kernel<EPI, W_MN>;
    static bool done[64] = {false};
    int sms = 0;
    int rc = allow_smem(kernel, rows_smem(256), done);
    if (rc == DK_OK) rc = sm_count(&sms);
    if (rc != DK_OK) return rc;
    const bool gated = EPI == EPI_GATED;
    const int N = rows_tokens(T, static_cast<size_t>(gated ? 2 : 1) * cols * K * 2);
    RowsMaps maps;
    rc = operand_map(&maps.w, W, W_MN, gated ? 2 * cols : cols, K, gated ? 64 : 128);
    if (rc == DK_OK) rc = operand_map(&maps.x, x, false, T, K, N);
    RowsArgs g{};
    if (rc == DK_OK) rc = device_status_ptr(&g.status);
    if (rc != DK_OK) return rc;
    g.N = N;
    g.T = T;
    g.cols = cols;
    g.num_kb = (K + BK - 1) / BK;
    g.out = static_cast<__nv_bfloat16*>(out);
    g.gu = static_cast<float*>(gu);
    const int tiles = (cols + (gated ? 64 : 128) - 1) / (gated ? 64 : 128), token_tiles = (T + N - 1) / N;
    // Cut K while the CTAs still run all at once and each keeps two K blocks. Powers of two only: the places they leave
    // go to the next product's CTAs, which start loading weights there (48 rows of 8192 x 3584: 41.4 us, with every place
    // taken 43.3).
    const int places = sms * (N <= 128 ? 2 : 1);
    int S = 1;
    while (S < 8 && tiles * token_tiles * S * 2 <= places && g.num_kb >= S * 4) S *= 2;
    g.weights_ready = follows;
    return launch_early(kernel, dim3(tiles * S, token_tiles), ROWS_THREADS, rows_smem(N), S, st, maps, g);
}

// Whether a call's products go by ffn_rows_kernel: up to 256 rows, and more where the weights are small. Measured, training
// steps, against ffn_gemm_kernel: 300 rows of 1536 x 2048 (12 MB) 53 us against 71, 513 62 against 77, 700 77 against 80 (forward
// alone 32 against 26); 300 rows of 2048 x 4096 (32 MB) 89 against 123, 384 99 against 121, 513 136 against 141 (forward 49
// against 45); 384 rows of 4096 x 4096 (64 MB) 178 against 174.
static bool few_rows(int T, int H, int F) {
    const size_t w13 = static_cast<size_t>(4) * F * H;
    return T <= (w13 <= SMALL_WEIGHTS / 2 ? 576 : w13 <= SMALL_WEIGHTS ? 400 : 256);
}

static int check_shape(int T, int H, int F) {
    DK_REQUIRE(T >= 0, "the number of rows must not be negative");
    DK_REQUIRE(H >= 8 && F >= 8 && H % 8 == 0 && F % 8 == 0, "H and F must be positive multiples of 8");
    DK_REQUIRE(T <= (1 << 24) && H <= (1 << 20) && F <= (1 << 20), "at most 2^24 rows and widths of 2^20");
    return DK_OK;
}

static int check_aligned(std::initializer_list<const void*> ps) {
    uintptr_t bits = 0;
    for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
    DK_REQUIRE((bits & 15) == 0, "every tensor must be 16-byte aligned");
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
    rc = check_aligned({x, w13, w2, gu, h, y});
    if (rc != DK_OK) return rc;
    if (few_rows(T, H, F)) {
        rc = rows_product<EPI_GATED, false>(x, w13, h, T, F, H, gu, false, st);
        if (rc != DK_OK) return rc;
        return rows_product<EPI_STORE, false>(h, w2, y, T, H, F, nullptr, true, st);
    }
    const Spec up{x, w13, h, T, F, H, false, false}, down{h, w2, y, T, H, F, false, false};
    rc = products<EPI_GATED>(&up, 1, gu, st);
    if (rc != DK_OK) return rc;
    return products<EPI_STORE>(&down, 1, nullptr, st);
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
    DK_REQUIRE(dy != nullptr && x != nullptr && gu != nullptr && h != nullptr && dgu != nullptr && dx != nullptr, "null operand");
    rc = check_aligned({dy, x, w13, w2, gu, h, dgu, dx, dw13, dw2});
    if (rc != DK_OK) return rc;
    // dW13 [2F,H] = dgu^T x and dW2 [H,F] = dy^T h, the tokens as K
    const Spec d_w13{dgu, x, dw13, 2 * F, H, T, true, true}, d_w2{dy, h, dw2, H, F, T, true, true};
    if (few_rows(T, H, F)) {
        // dh = dy W2 straight into dg and du, then dx = dgu W13
        rc = rows_product<EPI_DGATED, true>(dy, w2, dgu, T, F, H, const_cast<void*>(gu), false, st);
        if (rc == DK_OK) rc = rows_product<EPI_STORE, true>(dgu, w13, dx, T, H, 2 * F, nullptr, true, st);
        const Spec two[2] = {d_w13, d_w2};
        if (rc == DK_OK) rc = products<EPI_STORE>(two, 2, nullptr, st);
        return rc;
    }
    const Spec d_h{dy, w2, dgu, T, F, H, false, true}, d_x{dgu, w13, dx, T, H, 2 * F, false, true};
    rc = products<EPI_DGATED>(&d_h, 1, const_cast<void*>(gu), st);
    if (rc != DK_OK) return rc;
    // the longest tiles first
    Spec three[3] = {d_x, d_w13, d_w2};
    if (T > 2 * F) {
        three[0] = d_w13;
        three[1] = d_w2;
        three[2] = d_x;
    }
    rc = products<EPI_STORE>(three, 3, nullptr, st);
    return rc;
}
