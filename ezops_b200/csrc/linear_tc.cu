// Linear layers of prompts on the 5th-generation tensor cores:
//   out[m, n] = act( sum_k x[m, k] W[n, k] + bias[n] ) + residual[m, n],            fp32 until the one rounding,
//   SwiGLU: silu(gate + bias_g) * (up + bias_u) with W = [gate rows | up rows].
//
// Two CTAs of a cluster share a tile of 256 rows of A by BN rows of B, A = x and B = W or the
// other way round (tcgen05.mma.cta_group::2: each CTA holds half of both operands' rows, and 128 x BN of the result in its
// tensor memory), so each operand byte that enters an SM is used by two.  One elected thread per CTA fills a ring of 64-element
// K blocks by TMA (both CTAs' bytes are counted on the first CTA's barrier), one thread of the first CTA issues the MMAs,
// eight warps of each CTA drain one of two accumulators while the next tile is multiplied: bias, activation, residual and
// rounding happen there, in registers.  Grid: one CTA per SM, tiles in groups of kLtGroup tiles along A so that the x and W
// tiles in flight stay in L2.  BN = 256 reads least per product; narrower tiles, in steps of 16 or 32, are taken where the rounds of
// tiles come out even with them (linear_widths: 777 x 4096, K = 12288 in four rows of tiles of 208 instead of 256, 74 -> 63 us).
//   A = x: a lane of the epilogue has a row of the result and stores whole sectors of it.
//   A = W: a lane has a column, and a warp's stores run along a row: for rows that start anywhere (a vocabulary or a number of
// experts that is no multiple of 16, columns of a wider tensor), where a lane with a row would write parts of sectors, and for
// up to kLtSwapRows rows, where half of a tile of 256 rows of x would be empty.  SwiGLU then has gate and up rows as two A
// operands, two accumulators side by side.  Measured, A = x against A = W: 7404 x 17921, K = 96, gelu 422 and 184 us (with 17920
// columns: 154 and 163); 4530 x 3350, K = 720, fp32 62 and 32; 104 x 22304, K = 7360 86 and 67; 128 rows of 4096 through SwiGLU to
// 12288 61 to 67 and 50; 300 x 4096, K = 4096 15.2 to 16.6 and 16.0 to 16.9; 8192 x 4096, K = 4096 193 and 188 to 193.
// What bounds it: the tensor cores where tiles fill the clusters evenly (4096 rows of 4096 through SwiGLU to 12288: 516 us,
// 1600 TFLOP/s, tensor pipe active 98 % of the time; 587 to 640 at the 1.3 GHz of the power cap, by the card), with 64 to 74 of them busy to the end; the
// operands' way from L2 for narrow tiles; from a few hundred rows down the weights' bytes (104 x 22304, K = 7360: 5.1 TB/s).
// fp32 results of more than kLtSegment k blocks: the tensor cores cut their sums towards zero (gemm_tc.cu), so the sums leave them
// every kLtSegment blocks and are added up, rounded to nearest, in the registers of the lane whose column it is (A = W); the relative
// error is 4.7e-7 for K = 512 to 12800 (1.4e-5 at K = 12800 otherwise) and grows with the root of the number of segments, one rounding
// each, beside that (5.0e-7 at K = 204800); 8192 x 4096, K = 4096 takes 193 us instead of 191.  Rounded to bf16 that error does not show.
// Few rows or few results (linear_in_groups): the kernel of the batched decode projections (gemm_tc.cu) with this epilogue
// (17 x 6144, K = 4096: 10.4 us, 4.9 TB/s; 64 x 151936, K = 1024 to fp32: 57 us, 6.1 TB/s).
#include <atomic>

#include "prompt.h"
#include "tc.cuh"

namespace ezb {

static constexpr int kLtThreads = 320;  // TMA warp, MMA warp, eight epilogue warps
static constexpr int kLtBlockK = 64;
static constexpr int kLtMaxStages = 12;
static constexpr int kLtSegment = 8;  // k blocks of a sum that stays in the tensor cores, where the result is not rounded to bf16
static constexpr int kLtGroup = 8;  // row tiles per group of the tile order

struct LtParams {
    const bf16 *bias, *residual;
    void* out;
    long long ldres, ldout;
    int M, N, kblocks;
    int bn, tiles_a, tiles_b, act, out_f32;  // rows of B in a tile (SwiGLU with A = x: the template's); tiles along A's and B's rows
    int rows_aligned;  // rows of out start at 32-byte, of residual at 16-byte boundaries
    int vec_bias;      // so does bias
    unsigned int* status;
};
// ---- cta_group::2 wrappers ------------------------------------------------------
// The same barrier (or address) in the first CTA of the pair.
__device__ __forceinline__ uint32_t pair_leader(uint32_t shared_addr) { return shared_addr & 0xFEFFFFFFu; }
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(pair_leader(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_mma_bf16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on this barrier in both CTAs once the MMAs issued so far have finished.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void cluster_sync_full() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int BN, bool PAIR, bool SWAP>
struct LtSmem {
    static constexpr int kARows = 128 * kLtBlockK * 2;
    static constexpr int kA = (PAIR && SWAP ? 2 : 1) * kARows;  // this CTA's rows of A; SwiGLU, swapped: gate rows | up rows
    static constexpr int kB = BN / 2 * kLtBlockK * 2;           // and of B
    static constexpr int kStage = kA + kB;
    static constexpr int kTail = 1024;
    static constexpr int kTurn = SWAP ? 0 : 8 * 32 * 33 * 4;    // a 32 x 32 block of each epilogue warp
    static constexpr int kRoom = 232448 - 1024 - kTail - kTurn;
    static constexpr int kStages = kRoom / kStage < kLtMaxStages ? kRoom / kStage : kLtMaxStages;
    static constexpr int kBytes = 1024 + kStages * kStage + kTurn + kTail;
};

// W bf16 values, as they are; beyond `left` zeros.
template <int W>
__device__ __forceinline__ void load_packed(const bf16* src, int left, int vec, uint32_t (&w)[W / 2]) {
    if (vec && left >= W) {
#pragma unroll
        for (int e = 0; e < W / 2; e += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(src + 2 * e);
            w[e] = q.x, w[e + 1] = q.y, w[e + 2] = q.z, w[e + 3] = q.w;
        }
    } else {
        const unsigned short* raw = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
        for (int e = 0; e < W / 2; ++e)
            w[e] = (2 * e < left ? raw[2 * e] : 0u) | (2 * e + 1 < left ? (uint32_t)raw[2 * e + 1] << 16 : 0u);
    }
}

// BN: the most rows of B in a tile (p.bn).  SEG: the products of kLtSegment k blocks at a time, added up in registers (fp32 results, swapped form).
template <int BN, bool PAIR, bool SWAP, bool SEG>
__global__ void __launch_bounds__(kLtThreads, 1)
linear_tc_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW0,
                 const __grid_constant__ CUtensorMap mapW1, const __grid_constant__ LtParams p) {
    using L = LtSmem<BN, PAIR, SWAP>;
    const int bn = PAIR && !SWAP ? BN : p.bn, units = PAIR && !SWAP ? BN / 2 : bn;  // output columns of a tile; swapped: rows
    const uint32_t idesc = umma_idesc_bf16(256, bn);
    constexpr int ACC = PAIR && SWAP ? 2 * BN : BN;     // columns of tensor memory of a tile
    static_assert(2 * ACC <= 512);
    extern __shared__ unsigned char lt_raw[];
    const uint32_t raw = smem_u32(lt_raw);
    unsigned char* smem = lt_raw + (((raw + 1023u) & ~1023u) - raw);
    unsigned char* tail = smem + L::kStages * L::kStage + L::kTurn;
    uint64_t* full = reinterpret_cast<uint64_t*>(tail);
    uint64_t* empty = full + kLtMaxStages;
    uint64_t* acc_full = empty + kLtMaxStages;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = (int)cluster_rank();

    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) mbar_init(smem_u32(&full[s]), 1), mbar_init(smem_u32(&empty[s]), 1);
        for (int a = 0; a < 2; ++a) mbar_init(smem_u32(&acc_full[a]), 1), mbar_init(smem_u32(&acc_empty[a]), 16);  // warps of both CTAs
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 2 * ACC);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_full();  // the barriers of both CTAs exist
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_open(1);

    const int n_clusters = gridDim.x >> 1, cluster = blockIdx.x >> 1;
    const int n_tiles = p.tiles_a * p.tiles_b;
    auto tile_at = [&](int i, int& m, int& n) {  // groups of kLtGroup tiles along A, tile by tile along B
        const int per = kLtGroup * p.tiles_b, g = i / per, rows = min(kLtGroup, p.tiles_a - g * kLtGroup), r = i - g * per;
        m = g * kLtGroup + r % rows, n = r / rows;
    };
    if (warp == 0) {
        if (elect_one()) {
            int it = 0;
            for (int tile = cluster; tile < n_tiles && !*abort_flag; tile += n_clusters) {
                int tm, tn;
                tile_at(tile, tm, tn);
                const int y_a = tm * 256 + rank * 128;
                // SwiGLU: the second CTA brings the up rows
                const CUtensorMap *mapA = SWAP ? &mapW0 : &mapX, *mapB = SWAP ? &mapX : PAIR && rank ? &mapW1 : &mapW0;
                const int y_b = PAIR && !SWAP ? tn * units : tn * bn + rank * (bn / 2);
                for (int kb = 0; kb < p.kblocks; ++kb, ++it) {
                    const int s = it % L::kStages;
                    if (!mbar_wait_bounded(smem_u32(&empty[s]), (uint32_t)(((it / L::kStages) & 1) ^ 1), abort_flag, p.status, FAULT_GEMV_EMPTY_WAIT)) break;
                    const uint32_t bar = smem_u32(&full[s]), a = smem_u32(smem) + s * L::kStage;
                    if (rank == 0) mbar_arrive_expect_tx(bar, 2 * (L::kA + bn * kLtBlockK));  // both CTAs' halves of B
                    tma_load_2d_pair(a, mapA, kb * kLtBlockK, y_a, bar);
                    if constexpr (PAIR && SWAP) tma_load_2d_pair(a + L::kARows, &mapW1, kb * kLtBlockK, y_a, bar);
                    tma_load_2d_pair(a + L::kA, mapB, kb * kLtBlockK, y_b, bar);
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int it = 0;
            for (int tile = cluster, n = 0, k0 = 0; tile < n_tiles && !*abort_flag; ++n) {
                const int acc = n & 1;
                if (!mbar_wait_bounded_cluster(smem_u32(&acc_empty[acc]), (uint32_t)(((n >> 1) & 1) ^ 1), abort_flag, p.status, FAULT_TC_ACC_WAIT)) break;
                tc_fence_after();
                const int k1 = SEG ? min(k0 + kLtSegment, p.kblocks) : p.kblocks;
                for (int kb = k0; kb < k1; ++kb, ++it) {
                    const int s = it % L::kStages;
                    if (!mbar_wait_bounded_cluster(smem_u32(&full[s]), (uint32_t)((it / L::kStages) & 1), abort_flag, p.status, FAULT_GEMV_FULL_WAIT)) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem) + s * L::kStage;
                    const uint64_t ad = umma_desc_sw128(a), bd = umma_desc_sw128(a + L::kA);
#pragma unroll
                    for (int k = 0; k < kLtBlockK / 16; ++k) tc_mma_bf16_pair(tmem + acc * ACC, ad + 2 * k, bd + 2 * k, idesc, kb > k0 || k > 0);
                    if constexpr (PAIR && SWAP) {
                        const uint64_t ud = umma_desc_sw128(a + L::kARows);
#pragma unroll
                        for (int k = 0; k < kLtBlockK / 16; ++k)
                            tc_mma_bf16_pair(tmem + acc * ACC + BN, ud + 2 * k, bd + 2 * k, idesc, kb > k0 || k > 0);
                    }
                    tc_commit_pair(smem_u32(&empty[s]));
                }
                tc_commit_pair(smem_u32(&acc_full[acc]));
                k0 = k1;
                if (!SEG || k1 == p.kblocks) tile += n_clusters, k0 = 0;
            }
        }
    } else if constexpr (SWAP) {
        // A lane has an output column and walks rows of it, W at a time: a warp's loads and stores run along the rows of the
        // output, wherever those start.  The residual is requested a step ahead.
        constexpr int W = SEG ? 16 : 32;
        const int q = warp & 3, c0 = ((warp - 2) >> 2) * W;
        for (int tile = cluster, n = 0; tile < n_tiles; tile += n_clusters, ++n) {
            int ta, tb;
            tile_at(tile, ta, tb);
            const int n0 = ta * 256 + rank * 128 + q * 32, col = n0 + lane, m0 = tb * units;
            const int rows = n0 < p.N ? min(units, p.M - m0) : 0;
            const bool live = col < p.N;
            const bf16* res_col = p.residual && live ? p.residual + (long long)m0 * p.ldres + col : nullptr;
            const float bias = p.bias && live ? __bfloat162float(p.bias[col]) : 0.f;
            const float bias_up = PAIR && p.bias && live ? __bfloat162float(p.bias[p.N + col]) : 0.f;
            unsigned short res[W];
            auto request = [&](int c) {
                if (!res_col) return;
                const unsigned short* src = reinterpret_cast<const unsigned short*>(res_col + (long long)c * p.ldres);
#pragma unroll
                for (int e = 0; e < W; ++e) res[e] = c + e < rows ? src[e * p.ldres] : 0;
            };
            auto finish = [&](int c, float (&v)[W], float (&up)[PAIR ? W : 1], bool fine) {
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] += bias;
                if constexpr (PAIR) {
#pragma unroll
                    for (int e = 0; e < W; ++e) v[e] = silu_fast(v[e]) * (up[e] + bias_up);
                } else if (p.act != ACT_NONE) {
                    linear_act(v, p.act);
                }
                if (res_col) {
#pragma unroll
                    for (int e = 0; e < W; ++e) v[e] += __uint_as_float((uint32_t)res[e] << 16);
                    if (!SEG) request(c + 2 * W);
                }
                if (live && fine) {
                    const long long o = (long long)(m0 + c) * p.ldout + col;
                    auto store = [&](auto* dst, auto round) {
                        if (rows - c >= W) {
#pragma unroll
                            for (int e = 0; e < W; ++e) dst[e * p.ldout] = round(v[e]);
                        } else {
#pragma unroll
                            for (int e = 0; e < W; ++e)
                                if (c + e < rows) dst[e * p.ldout] = round(v[e]);
                        }
                    };
                    if (SEG || p.out_f32) store(static_cast<float*>(p.out) + o, [](float x) { return x; });
                    else store(static_cast<bf16*>(p.out) + o, [](float x) { return __float2bfloat16_rn(x); });
                }
                __syncwarp();
            };
            auto filled = [&]() {  // the accumulator's first column
                const int acc = n & 1;
                mbar_wait_bounded_cluster(smem_u32(&acc_full[acc]), (uint32_t)((n >> 1) & 1), abort_flag, p.status, FAULT_TC_ACC_WAIT);
                tc_fence_after();
                return tmem + ((uint32_t)(q * 32) << 16) + acc * ACC;
            };
            auto drained = [&]() {
                __syncwarp();
                tc_fence_before();
                if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[n & 1]), 0));
            };
            if constexpr (SEG) {
                constexpr int STEPS = BN / (2 * W);  // this warp's share: W columns of every 2 W
                float sum[STEPS][W], sum_up[PAIR ? STEPS : 1][PAIR ? W : 1];
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        sum[j][e] = 0.f;
                        if constexpr (PAIR) sum_up[j][e] = 0.f;
                    }
#pragma unroll 1
                for (int k = 0; k < p.kblocks; k += kLtSegment) {
                    const uint32_t t = filled();
#pragma unroll
                    for (int j = 0; j < STEPS; ++j) {
                        const int c = c0 + j * 2 * W;
                        if (c >= rows) break;
                        float v[W];
                        tmem_ld16(t + c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < W; ++e) sum[j][e] += v[e];
                        if constexpr (PAIR) {
                            tmem_ld16(t + BN + c, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < W; ++e) sum_up[j][e] += v[e];
                        }
                    }
                    drained();
                    if (k + kLtSegment < p.kblocks) ++n;
                }
                const bool fine = !__any_sync(0xffffffffu, *abort_flag);
#pragma unroll
                for (int j = 0; j < STEPS; ++j) {
                    const int c = c0 + j * 2 * W;
                    if (c >= rows) break;
                    request(c);
                    if constexpr (PAIR) finish(c, sum[j], sum_up[j], fine);
                    else finish(c, sum[j], sum_up[0], fine);
                }
            } else {
                request(c0);
                const uint32_t t = filled();
#pragma unroll 1
                for (int c = c0; c < rows; c += 2 * W) {
                    float v[W], up[PAIR ? W : 1];
                    tmem_ld32(t + c, v);
                    if constexpr (PAIR) tmem_ld32(t + BN + c, up);
                    tmem_ld_wait();
                    finish(c, v, up, !__any_sync(0xffffffffu, *abort_flag));
                }
                drained();
            }
        }
    } else {
        // A warp of the quarter of rows that it may read; W columns at a time.  What the residual stream holds there is requested
        // one step ahead (the first step: before the products are complete), or its latency would be paid once per step.
        constexpr int W = 32;
        const int q = warp & 3, row = q * 32 + lane;
        float* turn = reinterpret_cast<float*>(smem + L::kStages * L::kStage) + (warp - 2) * 32 * (W + 1);
        const int c0 = ((warp - 2) >> 2) * W;  // two warps share a quarter: every other step each
        for (int tile = cluster, n = 0; tile < n_tiles; tile += n_clusters, ++n) {
            int tm, tn;
            tile_at(tile, tm, tn);
            const int acc = n & 1;
            const int m = tm * 256 + rank * 128 + row;
            const bool live_row = m < p.M;
            const int n0 = tn * units;
            const int cols = min(units, p.N - n0);
            const bf16* res_row = p.residual && p.rows_aligned ? p.residual + (long long)m * p.ldres + n0 : nullptr;
            uint32_t ahead[W / 2];  // residual values of the next step, packed
            if (res_row && live_row && cols - c0 >= W) load_packed<W>(res_row + c0, W, 1, ahead);
            mbar_wait_bounded_cluster(smem_u32(&acc_full[acc]), (uint32_t)((n >> 1) & 1), abort_flag, p.status, FAULT_TC_ACC_WAIT);
            tc_fence_after();
            const uint32_t t = tmem + ((uint32_t)(q * 32) << 16) + acc * ACC;
            auto drained = [&]() {
                __syncwarp();
                tc_fence_before();
                if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[acc]), 0));
            };
#pragma unroll 1
            for (int c = c0; c < cols; c += 2 * W) {
                float v[W], up[PAIR ? W : 1];
                tmem_ld32(t + c, v);
                if constexpr (PAIR) tmem_ld32(t + units + c, up);
                const int left = cols - c, col = n0 + c;
                uint32_t res[W / 2];
                if (res_row) {
#pragma unroll
                    for (int e = 0; e < W / 2; ++e) res[e] = ahead[e];
                    if (live_row && left >= 3 * W) load_packed<W>(res_row + c + 2 * W, W, 1, ahead);
                }
                tmem_ld_wait();
                const bool fine = !__any_sync(0xffffffffu, *abort_flag);
                if (live_row && fine) {
                    if (p.bias) {
                        uint32_t b[W / 2];
                        load_packed<W>(p.bias + col, left, p.vec_bias, b);
#pragma unroll
                        for (int e = 0; e < W; ++e) v[e] += (e & 1) ? bf16_hi(b[e / 2]) : bf16_lo(b[e / 2]);
                        if constexpr (PAIR) {
                            load_packed<W>(p.bias + p.N + col, left, p.vec_bias, b);
#pragma unroll
                            for (int e = 0; e < W; ++e) up[e] += (e & 1) ? bf16_hi(b[e / 2]) : bf16_lo(b[e / 2]);
                        }
                    }
                    if constexpr (PAIR) {
#pragma unroll
                        for (int e = 0; e < W; ++e) v[e] = silu_fast(v[e]) * up[e];
                    } else if (p.act != ACT_NONE) {
                        linear_act(v, p.act);
                    }
                    if (p.rows_aligned && left >= W) {
                        if (res_row) {
#pragma unroll
                            for (int e = 0; e < W; ++e) v[e] += (e & 1) ? bf16_hi(res[e / 2]) : bf16_lo(res[e / 2]);
                        }
                        const long long o = (long long)m * p.ldout + col;
                        if (p.out_f32) {
#pragma unroll
                            for (int e = 0; e < W; e += 8) store32(static_cast<float*>(p.out) + o + e, reinterpret_cast<const uint32_t(&)[8]>(v[e]));
                        } else {
#pragma unroll
                            for (int e = 0; e < W; e += 16) {
                                uint32_t w[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) w[k] = pack_bf16(v[e + 2 * k], v[e + 2 * k + 1]);
                                store32(static_cast<bf16*>(p.out) + o + e, w);
                            }
                        }
                    }
                }
                if (!(p.rows_aligned && left >= W) && fine) {
                    // Rows that start anywhere, or the last columns: the 32 x 32 block turns in shared memory, and a lane has a column.
#pragma unroll
                    for (int e = 0; e < W; ++e) turn[lane * (W + 1) + e] = v[e];
                    __syncwarp();
                    const int rows = min(32, p.M - (m - lane));
                    if (lane < left) {
                        const bf16* res_col = p.residual ? p.residual + (long long)(m - lane) * p.ldres + col + lane : nullptr;
                        const long long o = (long long)(m - lane) * p.ldout + col + lane;
#pragma unroll 1
                        for (int r0 = 0; r0 < rows; r0 += 16) {
                            float x[16];  // 16 rows on their way at a time
                            if (res_col) {
#pragma unroll
                                for (int r = 0; r < 16; ++r) x[r] = r0 + r < rows ? __bfloat162float(__ldg(res_col + (r0 + r) * p.ldres)) : 0.f;
                            } else {
#pragma unroll
                                for (int r = 0; r < 16; ++r) x[r] = 0.f;
                            }
#pragma unroll
                            for (int r = 0; r < 16; ++r) x[r] += turn[(r0 + r) * (W + 1) + lane];
                            if (p.out_f32) {
                                float* dst = static_cast<float*>(p.out) + o + r0 * p.ldout;
#pragma unroll
                                for (int r = 0; r < 16; ++r)
                                    if (r0 + r < rows) dst[r * p.ldout] = x[r];
                            } else {
                                bf16* dst = static_cast<bf16*>(p.out) + o + r0 * p.ldout;
#pragma unroll
                                for (int r = 0; r < 16; ++r)
                                    if (r0 + r < rows) dst[r * p.ldout] = __float2bfloat16_rn(x[r]);
                            }
                        }
                    }
                }
                __syncwarp();
            }
            drained();
        }
    }
    __syncwarp();
    if (*abort_flag) __nanosleep(200000);  // copies and products that may still be in flight
    tc_fence_before();
    __syncthreads();
    cluster_sync_full();  // nothing is written to or signalled in a CTA that has left
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * ACC);
    }
}

// ---- host ---------------------------------------------------------------------
static bool encode_rows(CUtensorMap* map, const bf16* base, long long rows, long long cols, long long ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)kLtBlockK, (cuuint32_t)box_rows}, one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<bf16*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The form and the width of the tiles.  With all SMs busy a k block of a tile takes its cluster the longer of its products (368 ns
// for 256 x 256, at the clock that the power cap leaves) and of its operands' way from L2 (98 bytes per ns and SM; measured 368, 251
// and 209 ns for 256, 128 and 64 rows of B), and the last round of tiles takes as long as a full one: the width with the least sum is
// taken, the narrower of equal rounds, so that a last tile is not left nearly empty.
struct LtPlan {
    int bn, clusters;
    bool swap, seg;
    double cost;
};
static constexpr int kLtSwapRows = 128;  // rows of x up to which W's rows are A
static LtPlan linear_widths(int M, int N, bool pair, bool swap) {
    const long long most = sm_count() / 2, a_tiles = ((swap ? N : M) + 255ll) / 256;
    // what the epilogue takes at a time without a remainder; SwiGLU, swapped: two A operands, and two accumulators
    const int step = swap ? 16 : 32, widest = swap && pair ? 128 : 256, halves = swap && pair ? 2 : 1;
    LtPlan best = {0, 0, swap, false, 0.};
    for (int bn = widest; bn >= 64; bn = pair && !swap ? bn / 2 : bn - step) {
        const long long per = pair && !swap ? bn / 2 : bn, tiles = a_tiles * (((swap ? M : N) + per - 1) / per);
        const double products = 368. / 256. * bn * halves, operands = 1.306 * (128 * halves + bn / 2.);
        const double cost = (double)((tiles + most - 1) / most) * (products > operands ? products : operands);
        if (best.bn == 0 || cost < best.cost) best.bn = bn, best.cost = cost, best.clusters = (int)(tiles < most ? tiles : most);
    }
    return best;
}
static LtPlan linear_plan(int M, int N, int K, int act, bool aligned, bool f32) {
    const bool pair = act == ACT_SWIGLU, seg = f32 && (K + kLtBlockK - 1) / kLtBlockK > kLtSegment;
    LtPlan plan = linear_widths(M, N, pair, !aligned || M <= kLtSwapRows || seg);
    if (!plan.swap && !pair) {  // scattered rows cost a little: swapped only for a better fit
        const LtPlan other = linear_widths(M, N, pair, true);
        if (other.cost < 0.95 * plan.cost) plan = other;  // 776 x 5984, K = 3712 39 -> 28 us, 500 x 24576, K = 4096 101 -> 87
    }
    plan.seg = seg;
    return plan;
}

// Few rows, or few results behind a long K, for which pairs of CTAs would leave most SMs idle: groups of 64 rows, each with the
// weight cut along K over clusters that add their parts up in shared memory (us, pairs against groups: 128 x 64, K = 4096 10.3 and
// 5.8; 128 x 515, K = 4600 20.8 and 7.3; 300 x 512, K = 2048 8.7 and 7.3, but 555 rows 8.6 and 10.0; 2048 x 128, K = 4096 13.3 and 9.0;
// 400 x 128, K = 512 5.2 and 4.8, but 800 rows 5.2 and 5.7; 128 x 4096, K = 12288 32.6 and 28.4, K = 4096 14.3 and 15.0, K = 1024 6.8
// and 9.3).  The border is a fit to these: 128 x 4096, K = 4096 lies on it and takes the groups, the slower side by 5 %.  Above 64 rows
// each group brings the weight through L2 again, and the pairs do not cut K: neither is near the weight's bytes (5.4 us there).
static bool linear_in_groups(int M, int N, int K) {
    const long long tiles = ((long long)M + kLinearGroupRows - 1) / kLinearGroupRows * ((N + 127ll) / 128);
    if (((long long)M + kLinearGroupRows - 1) / kLinearGroupRows > sm_count()) return false;  // a cluster each at least
    return M <= kLinearGroupRows || (tiles <= 64 && 60 * tiles <= K);
}

template <int BN, bool PAIR, bool SWAP, bool SEG = false>
static cudaError_t launch_linear_tile(const LinearArgs& a, const LtPlan& plan, LtParams& p, cudaStream_t stream) {
    constexpr int kBytes = LtSmem<BN, PAIR, SWAP>::kBytes;
    alignas(64) CUtensorMap mx, w0, w1;
    const int box_x = SWAP ? plan.bn / 2 : 128, box_w = SWAP ? 128 : plan.bn / 2, units = PAIR && !SWAP ? plan.bn / 2 : plan.bn;
    if (!encode_rows(&mx, a.x, a.M, a.K, a.ldx, box_x) || !encode_rows(&w0, a.W, a.N, a.K, a.K, box_w)) return cudaErrorInvalidValue;
    if (!PAIR) w1 = w0;
    else if (!encode_rows(&w1, a.W + (long long)a.N * a.K, a.N, a.K, a.K, box_w)) return cudaErrorInvalidValue;
    static std::atomic<bool> configured[64];
    if (cudaError_t e = allow_smem_once(linear_tc_kernel<BN, PAIR, SWAP, SEG>, kBytes, configured)) return e;
    p.tiles_a = ((SWAP ? a.N : a.M) + 255) / 256, p.tiles_b = ((SWAP ? a.M : a.N) + units - 1) / units, p.bn = plan.bn;
    chain_begin();
    return launch_pdl_cluster(linear_tc_kernel<BN, PAIR, SWAP, SEG>, dim3(2u * plan.clusters), dim3(kLtThreads), 2, kBytes, stream, mx, w0, w1, p);
}
template <bool PAIR>
static cudaError_t launch_linear_form(const LinearArgs& a, const LtPlan& plan, LtParams& p, cudaStream_t stream) {
    if (plan.seg) {
        if constexpr (!PAIR)
            if (plan.bn > 128) return launch_linear_tile<256, PAIR, true, true>(a, plan, p, stream);
        return plan.bn > 64 ? launch_linear_tile<128, PAIR, true, true>(a, plan, p, stream) : launch_linear_tile<64, PAIR, true, true>(a, plan, p, stream);
    }
    if (plan.swap) {
        if constexpr (!PAIR)
            if (plan.bn > 128) return launch_linear_tile<256, PAIR, true>(a, plan, p, stream);
        return plan.bn > 64 ? launch_linear_tile<128, PAIR, true>(a, plan, p, stream) : launch_linear_tile<64, PAIR, true>(a, plan, p, stream);
    }
    if (plan.bn > 128) return launch_linear_tile<256, PAIR, false>(a, plan, p, stream);
    return plan.bn > 64 ? launch_linear_tile<128, PAIR, false>(a, plan, p, stream) : launch_linear_tile<64, PAIR, false>(a, plan, p, stream);
}

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t stream) {
    if (linear_in_groups(a.M, a.N, a.K)) return launch_linear_groups(a, stream);
    LtParams p;
    p.bias = a.bias, p.residual = a.residual, p.out = a.out, p.ldres = a.ldres, p.ldout = a.ldout;
    p.M = a.M, p.N = a.N, p.kblocks = (a.K + kLtBlockK - 1) / kLtBlockK;
    p.act = a.act, p.out_f32 = a.out_f32;
    p.rows_aligned = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0 && a.ldout % (a.out_f32 ? 8 : 16) == 0 &&
                     (!a.residual || (aligned16(a.residual) && a.ldres % 8 == 0));
    p.vec_bias = a.bias && aligned16(a.bias) && (a.act != ACT_SWIGLU || a.N % 8 == 0);
    p.status = status_ptr();
    if (!p.status) return cudaErrorUnknown;
    const LtPlan plan = linear_plan(a.M, a.N, a.K, a.act, p.rows_aligned, a.out_f32);
    return a.act == ACT_SWIGLU ? launch_linear_form<true>(a, plan, p, stream) : launch_linear_form<false>(a, plan, p, stream);
}

}  // namespace ezb
