// Causal attention of ragged rows over paged KV caches, on the 5th-generation tensor cores:
//   row b has n_b queries (tokens cu[b] .. cu[b+1]) behind c_b = len_b - n_b cached keys; query i of it sees the keys
//   0 .. c_b + i:   out = softmax(q K^T / sqrt(D)) V,   H query heads share NKV key/value heads (G = H / NKV).
//
// Tile: the G heads of a group are packed next to each other, so 128 rows of an MMA are floor(128/G) tokens x G heads and
// every key and value is read once per group.  A unit of work is 256 such rows (two tiles, two softmax warpgroups) of one
// (row, kv head); it walks the keys 128 at a time.  Scores S (fp32) live in tensor memory, one thread owns a whole row of
// them: running maximum and sum without a shuffle.  P is written back over S in bf16 (relative error 2^-8 of a weight, the
// sum keeps the unrounded one) and is the MMA's A operand from tensor memory, in two halves so that the products of the first
// start under the exponentials of the second; O (fp32) stays there too.  2 x (128 + D) columns of the 512.  The two warpgroups
// take turns: while one exponentiates, the other tile's products run.  The output is rescaled only when a row's maximum has
// grown by more than 2^8 since the last time (the result does not depend on which maximum is subtracted; sums and P stay far
// inside their ranges), so the first half of a block is exponentiated before its maximum is known.
// A unit with at most 128 rows (single tokens, the end of a prompt) uses the second warpgroup for every other block of keys;
// the halves meet in tensor memory.
//
// Work is dealt out on the device, since the lengths are there: all units form one line, weighted by their keys, and CTA c
// takes the c-th equal share; a unit that is cut leaves (max, sum, O) parts in the workspace, and the CTA that finishes its
// last part joins them in the order of the keys (equal calls give equal bits).  Units of up to kApWhole tiles stay whole: a part
// costs a trip through the workspace (short prompts of 14 heads of 64: 37.7 -> 17.6 us).
//
// What bounds it: for prompts the exponentials and the products, one behind the other - 128 x 128 scores take 512 cycles each for
// QK^T and PV (D = 128) and 1024 cycles of the MUFU, twice per step, so either alone needs 2048 cycles of a step that takes about 3700.
// The two were meant to overlap, and hardly do (4096 tokens: tensor pipe busy for 51.5 % of the time, MUFU 51.7 %); where a step waits has not
// been measured.  8192 tokens, 32/8 heads of 128: 439 us, 1250
// TFLOP/s of the products that the mask leaves (505 us at the 1.6 GHz of the power cap; the MMAs alone in this order 355 to 370
// us); 8 prompts of 65 to 600 tokens behind 300 to 7400: 232 us (277 capped); 8192 tokens of D = 64: 380 us, of which 240 are
// exponentials.  For single tokens the bytes
// of the caches: 32 of them over 1000 to 8100 keys 103 to 112 us, 5.5 to 5.9 TB/s.
// Measured and left out: a polynomial in place of part of the exponentials, 512 softmax threads, P handed over at 75 %, blocks of
// 64 keys (+12 % for QK^T), a third block of scores beside O of 64 columns (3 %): no gain that carries its code.
// Keys behind a row's last one, entries outside the pools and everything masked are never added: K there is masked after
// the product, V is zero (out-of-range TMA boxes, or cleared in shared memory where a box straddles the end).
#include <atomic>

#include "prompt.h"
#include "tc.cuh"

namespace ezb {

static constexpr int kApThreads = 384;  // warps 0-3 and 4-7: softmax of tile 0 / 1; 8: TMA; 9: MMA; 10: deals out the work; 11 fills up its warpgroup
static constexpr int kApStages = 5;     // ring of K and V tiles
static constexpr int kApKeys = 128;     // keys per tile
static constexpr int kApSegments = 4;   // ring of work descriptors
static constexpr int kApUnitCost = 256;  // a unit's fixed cost in keys; at least 127, so that its last tile lies inside its cost
// Eighths that a unit of at most 128 rows costs less: half of the products, all of the bytes (32 rows of 1 to 100 tokens behind
// 1000 to 8000 keys 222 -> 207 us, 2/8 212, 4/8 217; 8 of 65 to 600 238 -> 234).
static constexpr int kApDualLess = 3;
static constexpr int kApWhole = 4;      // units of at most so many tiles are never cut
static constexpr int kApMinShare = 256;  // keys below which a further CTA is not worth its merge

struct ApParams {
    bf16* Out;
    long long ldo;
    const int *table, *lens, *cu;
    float* parts;        // [2 * grid slots][2 tiles][D + 2][128] fp32
    unsigned int* count;  // [grid], zero between calls
    int B, T, H, NKV, G, tpt, max_pages, page_shift, num_pages;
    int out32;  // rows of Out start at 32-byte boundaries
    float scale_log2;  // log2(e) / sqrt(D)
    unsigned int* status;
};

// ---- wrappers -----------------------------------------------------------------
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void store_row16(bf16* dst, const uint32_t (&w)[8], bool whole_sector) {  // 16 elements
    if (whole_sector) {
        store32(dst, w);
    } else {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
// Operand descriptors as halves: the low word holds the address (and the column block stride), the high word is one constant
// for all 128-byte-swizzled tiles (see umma_desc_sw128), so that only 32 bits a tile have to be kept.
static constexpr uint32_t kApDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t ap_desc(uint32_t smem_addr) { return (smem_addr & 0x3FFFFu) >> 4; }
__device__ __forceinline__ void ap_mma_ss(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(kApDescHigh), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ap_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(kApDescHigh), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// ---- the line of work ----------------------------------------------------------
// A unit: 2 * tpt consecutive tokens of a row for one kv head.
struct ApRow {
    int q0, n, len, units;  // first token, tokens, valid keys
    long long per_unit;     // cost of unit j: per_unit + (j + 1) * 2 * tpt,
    long long less;         // less this for the last one, when it has one tile of queries
    long long head_cost;    // cost of all units of one head
};
__device__ __forceinline__ ApRow ap_row(const ApParams& p, int b) {
    ApRow r;
    r.q0 = min(max(__ldg(p.cu + b), 0), p.T);
    r.n = min(max(__ldg(p.cu + b + 1), r.q0), p.T) - r.q0;
    r.len = min(max(__ldg(p.lens + b), 0), p.max_pages << p.page_shift);
    const int u = 2 * p.tpt;
    r.units = (r.n + u - 1) / u;
    r.per_unit = max(r.len - r.n, 0) + kApUnitCost;
    r.less = r.units && r.n - (r.units - 1) * u <= p.tpt ? (r.per_unit + (long long)r.units * u) * kApDualLess / 8 : 0;
    r.head_cost = r.units * r.per_unit + (long long)u * r.units * (r.units + 1) / 2 - r.less;
    return r;
}
__device__ __forceinline__ long long ap_unit_start(const ApParams& p, const ApRow& r, int j) {  // inside its head
    return j * r.per_unit + (long long)p.tpt * j * (j + 1);
}

struct ApLine {
    long long total, share;
    int ctas;  // CTAs that take a share
};
__device__ __forceinline__ long long ap_share(const ApLine& l, int c) {  // where CTA c's share starts
    const long long x = l.share * c;
    return x < l.total ? x : l.total;
}

struct ApCursor {
    int b, h, j;
    long long x0;  // where the unit starts on the line
    ApRow row;
};
// What the warps of a CTA have to know about the part of a unit that is theirs.
struct ApSegment {
    int cnt;            // tiles of 128 keys of this CTA (0: a unit without keys), or -1: no more segments
    int tiles, ks;      // tiles of the unit, first one of this CTA
    int dual;           // the unit has at most 128 rows
    int extent;         // keys that any of its queries sees
    int token, tokens;  // first token (in Q and Out), tokens
    int sees;           // keys that the first token sees (below 1: none); every further token sees one more
    int row, head;      // batch row, kv head
    int clear;          // the last V tile straddles the end of the row's keys
    int slot;           // where a part of it goes
    int c0, c1;         // first and last CTA with tiles of it
    long long x0;       // its start on the line
};
// The tile of the unit that starts at x0 at which place x of the line cuts it: short units are not cut, and no piece is
// shorter than two tiles (a part costs a trip through the workspace).
__device__ __forceinline__ int ap_tile_at(long long x, long long x0, int tiles, int dual) {
    if (x <= x0) return 0;
    const long long at = (dual ? (x - x0) * 8 / (8 - kApDualLess) : x - x0) >> 7;
    const int k = at < tiles ? (int)at : tiles;
    if (tiles <= kApWhole) return 2 * k >= tiles ? tiles : 0;
    return k < 2 ? 0 : (k > tiles - 2 ? tiles : k);
}
// The unit under the cursor as CTA `cta` with share [lo, hi) sees it; false when none of its tiles belongs to the share.
__device__ __forceinline__ bool ap_segment(const ApParams& p, const ApLine& line, const ApCursor& c, int cta, long long lo, long long hi,
                                           ApSegment& s) {
    const int u = 2 * p.tpt, first = c.j * u;
    s.tokens = min(u, c.row.n - first);
    s.extent = max(0, c.row.len - (c.row.n - first - s.tokens));
    s.tiles = (s.extent + kApKeys - 1) / kApKeys;
    s.dual = s.tokens <= p.tpt;
    s.ks = ap_tile_at(lo, c.x0, s.tiles, s.dual);
    s.cnt = ap_tile_at(hi, c.x0, s.tiles, s.dual) - s.ks;
    if (s.tiles ? s.cnt == 0 : lo > c.x0) return false;  // a unit without keys belongs to the share in which it starts
    s.token = c.row.q0 + first;
    s.sees = c.row.len - c.row.n + first + 1;
    s.row = c.b, s.head = c.h;
    s.clear = ((s.extent + 63) & ~63) > c.row.len && (s.extent & 63);
    s.x0 = c.x0;
    s.slot = 2 * cta + (c.x0 >= lo ? 1 : 0);  // 2 * cta: a unit that an earlier CTA began
    s.c0 = s.c1 = cta;
    // (a unit may start in one share and have all its tiles in the next)
    if (c.x0 < lo)
        while (s.c0 > 0 && ap_share(line, s.c0) > c.x0) --s.c0;
    if (s.ks + s.cnt < s.tiles)
        while (s.c1 + 1 < line.ctas && ap_tile_at(ap_share(line, s.c1 + 1), c.x0, s.tiles, s.dual) < s.tiles) ++s.c1;
    return true;
}
// Next unit; false at the end of the batch.  Called by a whole warp: rows without tokens are passed over 32 at a time.
__device__ __forceinline__ bool ap_advance(const ApParams& p, ApCursor& c, int lane) {
    c.x0 += c.row.per_unit + (long long)(c.j + 1) * 2 * p.tpt;
    if (++c.j < c.row.units) return true;
    c.x0 -= c.row.less;
    c.j = 0;
    if (++c.h < p.NKV) return true;
    c.h = 0;
    for (int b = c.b + 1; b < p.B; b += 32) {
        const uint32_t some = __ballot_sync(0xffffffffu, b + lane < p.B && ap_row(p, min(b + lane, p.B - 1)).units > 0);
        if (some) {
            c.b = b + __ffs(some) - 1;
            c.row = ap_row(p, c.b);
            return true;
        }
    }
    return false;
}

template <int D>
struct ApSmem {
    static constexpr int kTile = kApKeys * D * 2;  // a K, V or Q tile
    static constexpr int kQ = 0;
    static constexpr int kRing = 2 * kTile;
    static constexpr int kTail = kRing + kApStages * kTile;
    static constexpr int kBytes = kTail + 2048 + 1024;  // tail, alignment
};

struct ApTail {
    uint64_t full[kApStages], empty[kApStages];
    uint64_t q_full, q_empty, fix;
    uint64_t s_full[2], p_full[2], o_full[2], o_empty[2], turn[2], h_full[2];
    uint64_t seg_full[kApSegments], seg_empty[kApSegments];
    ApSegment seg[kApSegments];
    uint32_t tmem;
    int abort_flag;
    int published;  // descriptors in all, once they are all there (before: -1)
    int last;       // this CTA joins the parts of the unit
    int parts;
    short list[160];  // parts of a unit in the order of its keys: twice their slot
    union {
        struct {
            ApCursor start;  // where the CTA's share starts
            long long warp_sum[kApThreads / 32];
        };
        float stat[2][128];  // later: maxima and sums of warpgroup 1 on their way to warpgroup 0
    };
};
static_assert(sizeof(ApTail) <= 2048, "tail of the shared memory");

// Joins the n parts of a unit: out = sum_k w_k O_k / sum_k w_k sum_k with w_k = exp2(scale (max_k - max)), by the softmax
// threads that wrote them.  A thread keeps one row of the unit (rows rounded up to a power of two) and D / (threads / rows)
// neighbouring columns of it, 4 W at a time; what it loads of U parts is on its way together.  Not inlined: its registers would
// be taken from the loop over the keys.
template <int D, int W, int U>
__device__ __noinline__ void ap_join(const ApParams& p, const ApSegment& seg, const short* list, int n, int tid, int threads) {
    constexpr long long kPart = (long long)(D + 2) * 128;
    const int rows = seg.tokens * p.G, per_tile = p.tpt * p.G;
    const int log_rows = rows > 1 ? 32 - __clz(rows - 1) : 0, row = tid & ((1 << log_rows) - 1), share = threads >> log_rows;
    if (row >= rows) return;
    const int q = row / per_tile, rr = row - q * per_tile;  // tile of the pair (one of keys: always 0) and row in it
    const float* base = p.parts + q * kPart;
    const float* stat = base + (long long)D * 128 + rr;
    float top = -INFINITY;
#pragma unroll 8
    for (int k = 0; k < n; ++k) top = fmaxf(top, __ldcg(stat + list[k] * kPart));
    const int token = row / p.G, head = row - token * p.G;
    const bool any = seg.sees + token > 0;  // else the query sees no key
    bf16* out = p.Out + (long long)(seg.token + token) * p.ldo + (long long)(seg.head * p.G + head) * D;
    const int per = max(W, D / 4 / share);  // groups of four columns of this thread
#pragma unroll 1
    for (int g0 = (tid >> log_rows) * per, g1 = min(g0 + per, D / 4); g0 < g1; g0 += W) {
        float4 acc[W];
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        float all = 0.f;
#pragma unroll 1
        for (int k = 0; k < n; k += U) {
            float4 o[U][W];
            float w[U], ps[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long at = list[min(k + u, n - 1)] * kPart;
                const float4* part = reinterpret_cast<const float4*>(base + at) + rr;
#pragma unroll
                for (int e = 0; e < W; ++e) o[u][e] = __ldcg(part + (g0 + e) * 128);
                w[u] = __ldcg(stat + at), ps[u] = __ldcg(stat + at + 128);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = w[u] == -INFINITY || k + u >= n ? 0.f : exp2_approx((w[u] - top) * p.scale_log2);
                all += f * ps[u];
#pragma unroll
                for (int e = 0; e < W; ++e) acc[e].x += f * o[u][e].x, acc[e].y += f * o[u][e].y, acc[e].z += f * o[u][e].z, acc[e].w += f * o[u][e].w;
            }
        }
        const float inv = 1.0f / all;
        uint32_t w[2 * W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
            w[2 * e] = any ? pack_bf16(acc[e].x * inv, acc[e].y * inv) : 0u;
            w[2 * e + 1] = any ? pack_bf16(acc[e].z * inv, acc[e].w * inv) : 0u;
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int e = 0; e < W / 4; ++e) store_row16(out + (g0 + 4 * e) * 4, reinterpret_cast<const uint32_t(&)[8]>(w[8 * e]), p.out32);
        } else {
            *reinterpret_cast<uint2*>(out + g0 * 4) = make_uint2(w[0], w[1]);
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kApThreads, 1)
attn_prompt_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                   const __grid_constant__ CUtensorMap mapV, const __grid_constant__ ApParams p) {
    using L = ApSmem<D>;
    constexpr int BLOCKS = D / 64;  // column blocks of 64 elements (128 bytes)
    constexpr uint32_t IDESC_QK = umma_idesc_bf16(128, kApKeys);
    constexpr uint32_t IDESC_PV = umma_idesc_bf16(128, D) | (1u << 16);  // B transposed: N is the contiguous dimension
    extern __shared__ unsigned char ap_raw[];
    const uint32_t raw = smem_u32(ap_raw);
    unsigned char* smem = ap_raw + (((raw + 1023u) & ~1023u) - raw);
    ApTail& t = *reinterpret_cast<ApTail*>(smem + L::kTail);
    volatile int* abort_flag = &t.abort_flag;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < kApStages; ++s) mbar_init(smem_u32(&t.full[s]), 1), mbar_init(smem_u32(&t.empty[s]), 1);
        mbar_init(smem_u32(&t.q_full), 1), mbar_init(smem_u32(&t.q_empty), 1), mbar_init(smem_u32(&t.fix), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&t.s_full[i]), 1), mbar_init(smem_u32(&t.o_full[i]), 1);
            mbar_init(smem_u32(&t.p_full[i]), 4), mbar_init(smem_u32(&t.o_empty[i]), 4);  // one arrival per warp
            mbar_init(smem_u32(&t.turn[i]), 4), mbar_init(smem_u32(&t.h_full[i]), 4);
        }
        for (int i = 0; i < kApSegments; ++i)
            mbar_init(smem_u32(&t.seg_full[i]), 1), mbar_init(smem_u32(&t.seg_empty[i]), 10);  // warps that read it
        t.abort_flag = 0, t.published = -1;
        mbar_fence_init();
    }
    if (tid == 32) {
        prefetch_map(&mapQ), prefetch_map(&mapK), prefetch_map(&mapV);
    }
    // The tensor memory is taken before the next kernel may start: one that came to this SM first would hold some of it while it
    // waits for this kernel.
    if (warp == 9) {
        tmem_alloc(smem_u32(&t.tmem), 512);
        tmem_relinquish();
    }
    __syncthreads();
    pdl_open(1);

    // ---- where this CTA's share starts: running sums of the rows' costs, rows spread over the threads
    const int cta = blockIdx.x;
    auto row_cost = [&](int b) { return b < p.B ? ap_row(p, b).head_cost * p.NKV : 0; };
    auto chunk_scan = [&](long long v, long long& total) {  // exclusive prefix over the block
        long long s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += up;
        }
        __syncthreads();
        if (lane == 31) t.warp_sum[warp] = s;
        __syncthreads();
        long long before = 0, all = 0;
        for (int w = 0; w < kApThreads / 32; ++w) {
            if (w == warp) before = all;
            all += t.warp_sum[w];
        }
        total = all;
        return before + s - v;
    };
    long long total = 0, first_cost = 0, first_prefix = 0;
    ApRow first_row = {};  // of the first rows, one per thread: all there are, mostly
    if (tid < p.B) first_row = ap_row(p, tid);
    for (int b0 = 0; b0 < p.B; b0 += kApThreads) {
        const long long v = b0 == 0 ? first_row.head_cost * p.NKV : row_cost(b0 + tid);
        long long sum;
        const long long pre = chunk_scan(v, sum);
        if (b0 == 0) first_cost = v, first_prefix = pre;
        total += sum;
    }
    ApLine line;
    line.total = total;
    line.share = (total + gridDim.x - 1) / gridDim.x;
    if (line.share < kApMinShare) line.share = kApMinShare;
    line.ctas = (int)min((long long)gridDim.x, (total + line.share - 1) / line.share);
    const bool idle = total == 0 || cta >= line.ctas;
    const long long lo = idle ? 0 : ap_share(line, cta), hi = idle ? 0 : ap_share(line, cta + 1);
    if (!idle) {
        long long base = 0;
        for (int b0 = 0; b0 < p.B; b0 += kApThreads) {
            long long v = first_cost, pre = first_prefix, sum = 0;
            if (p.B > kApThreads) {
                v = row_cost(b0 + tid);
                pre = chunk_scan(v, sum);
            }
            const long long x = base + pre;
            if (v > 0 && x <= lo && lo < x + v) {
                ApCursor c;
                c.b = b0 + tid;
                c.row = b0 == 0 ? first_row : ap_row(p, c.b);
                c.h = (int)((float)(lo - x) / (float)c.row.head_cost);  // at most one off, below
                if (c.h >= p.NKV || c.h * c.row.head_cost > lo - x) --c.h;
                else if ((c.h + 1) * c.row.head_cost <= lo - x) ++c.h;
                const long long rem = (lo - x) - c.h * c.row.head_cost;
                int a = 0, z = c.row.units;  // last unit that starts at or before rem
                while (z - a > 1) {
                    const int mid = (a + z) >> 1;
                    if (ap_unit_start(p, c.row, mid) <= rem) a = mid;
                    else z = mid;
                }
                c.j = a;
                c.x0 = x + c.h * c.row.head_cost + ap_unit_start(p, c.row, a);
                t.start = c;
            }
            base += sum;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = t.tmem;
    const uint32_t sm_q = smem_u32(smem), sm_ring = sm_q + L::kRing;

    // The next work descriptor (all lanes of a warp); it is read in place and given back with `release`.
    int n_seg = 0;
    auto next_segment = [&]() -> const ApSegment* {
        const int i = n_seg % kApSegments;
        if (!mbar_wait_bounded(smem_u32(&t.seg_full[i]), (uint32_t)((n_seg / kApSegments) & 1), abort_flag, p.status, FAULT_PROMPT_WAIT)) {
            // Some wait has run out.  Warps that meet at barriers have to leave behind the same descriptor: the last one there is.
            const long long t0 = clock64();
            while (*(volatile int*)&t.published < 0)
                if (clock64() - t0 > kWaitLimitCycles) return nullptr;
            if (n_seg >= *(volatile int*)&t.published) return nullptr;
        }
        return t.seg[i].cnt < 0 ? nullptr : &t.seg[i];
    };
    auto release = [&]() {
        mbar_arrive(smem_u32(&t.seg_empty[n_seg % kApSegments]));
        ++n_seg;
    };

    // A softmax thread holds a row of scores: 384 threads x 168 registers at launch = 2 x 128 x 216 + 128 x 72.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (idle) {
        } else if (warp == 10) {
            // ------------------------------------------------------------ work descriptors
            ApCursor cur = t.start;
            for (bool more = true;; more = more && ap_advance(p, cur, lane)) {
                const bool end = !more || cur.x0 >= hi;
                ApSegment s;
                s.cnt = -1;
                if (!end && !ap_segment(p, line, cur, cta, lo, hi, s)) continue;
                const int i = n_seg % kApSegments;
                if (!mbar_wait_bounded(smem_u32(&t.seg_empty[i]), (uint32_t)(((n_seg / kApSegments) & 1) ^ 1), abort_flag, p.status, FAULT_PROMPT_WAIT)) break;
                if (lane == 0) {
                    t.seg[i] = s;
                    mbar_arrive(smem_u32(&t.seg_full[i]));
                }
                __syncwarp();
                ++n_seg;
                if (end) break;
            }
            __threadfence_block();
            if (lane == 0) *(volatile int*)&t.published = n_seg;
        } else if (warp == 8) {
            // ------------------------------------------------------------ TMA producer
            int it = 0, n_q = 0, n_fix = 0;  // ring tiles, query loads, repaired tiles so far
            while (const ApSegment* sp = next_segment()) {
                const ApSegment seg = *sp;
                __syncwarp();
                if (lane == 0) release();
                else ++n_seg;
                if (seg.cnt == 0) continue;
                const int* table = p.table + (long long)seg.row * p.max_pages;
                if (!mbar_wait_bounded(smem_u32(&t.q_empty), (uint32_t)((n_q & 1) ^ 1), abort_flag, p.status, FAULT_PROMPT_WAIT)) break;
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&t.q_full);
                    const int tiles_q = seg.dual ? 1 : 2;
                    mbar_arrive_expect_tx(bar, (uint32_t)(p.tpt * p.G * 128 * BLOCKS * tiles_q));
                    for (int m = 0; m < tiles_q; ++m)
#pragma unroll
                        for (int k = 0; k < BLOCKS; ++k)
                            tma_load_3d(sm_q + m * L::kTile + k * 16384, &mapQ, k * 64, seg.head * p.G, seg.token + m * p.tpt, bar);
                }
                __syncwarp();
                ++n_q;
                int ids = 0, ids_from = -16;  // lane i: pool page of key block (ids_from * 2 + i), 64 keys each
                // K and V tiles in the order of their use: K(0) V(0) K(1) V(1) ..., or K(0) K(1) V(0) K(2) V(1) ... (dual)
                const int ahead = seg.dual ? 2 : 1, lead = min(ahead, seg.cnt);
#pragma unroll 1
                for (int i = 0; i < 2 * seg.cnt && !*abort_flag; ++i) {
                    int v = 0, k = i;
                    if (i >= lead) {
                        const int o = i - lead;  // V(0) K(ahead) V(1) K(ahead + 1) ... then the last V
                        const int pairs = seg.cnt - lead;
                        if (o < 2 * pairs) v = !(o & 1), k = (o >> 1) + (v ? 0 : ahead);
                        else v = 1, k = pairs + (o - 2 * pairs);
                    }
                    k += seg.ks;
                    if (k < ids_from || k >= ids_from + 16) {
                        ids_from = k;
                        const long long key = ((long long)k * 2 + lane) * 64;
                        ids = p.num_pages;  // out of range: zeros
                        if (key < seg.extent) {
                            const int id = __ldg(table + (key >> p.page_shift));
                            if (id >= 0 && id < p.num_pages) ids = id;
                            else report_fault(p.status, FAULT_PAGE_RANGE);
                        }
                    }
                    const int stage = it % kApStages;
                    if (!mbar_wait_bounded(smem_u32(&t.empty[stage]), (uint32_t)(((it / kApStages) & 1) ^ 1), abort_flag, p.status, FAULT_PROMPT_WAIT)) break;
                    const int id0 = __shfl_sync(0xffffffffu, ids, (k - ids_from) * 2), id1 = __shfl_sync(0xffffffffu, ids, (k - ids_from) * 2 + 1);
                    const bool repair = v && seg.clear && k == seg.tiles - 1;
                    const uint32_t dst = sm_ring + stage * L::kTile, bar = smem_u32(repair ? &t.fix : &t.full[stage]);
                    if (elect_one()) {
                        const CUtensorMap* map = v ? &mapV : &mapK;
                        const int mask = (1 << p.page_shift) - 1, y0 = (k * kApKeys) & mask, y1 = (k * kApKeys + 64) & mask;
                        mbar_arrive_expect_tx(bar, L::kTile);
#pragma unroll
                        for (int c = 0; c < BLOCKS; ++c) {
                            tma_load_3d(dst + c * 16384, map, c * 64, y0, id0 * p.NKV + seg.head, bar);
                            tma_load_3d(dst + c * 16384 + 8192, map, c * 64, y1, id1 * p.NKV + seg.head, bar);
                        }
                    }
                    __syncwarp();
                    ++it;
                    if (repair) {
                        // rows behind the last key of the block that straddles it: P is zero there, and V has to be
                        mbar_wait_bounded(bar, (uint32_t)(n_fix & 1), abort_flag, p.status, FAULT_PROMPT_WAIT);
                        ++n_fix;
                        const int r0 = seg.extent - k * kApKeys, bytes = (((r0 + 63) & ~63) - r0) * 128;  // extent is no multiple of 64 here
                        for (int c = 0; c < BLOCKS; ++c)
                            for (int o = lane * 16; o < bytes; o += 512)
                                *reinterpret_cast<uint4*>(smem + L::kRing + stage * L::kTile + c * 16384 + r0 * 128 + o) = make_uint4(0u, 0u, 0u, 0u);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&t.full[stage]));
                    }
                }
            }
            if (*abort_flag) {  // nothing may still be landing in this CTA's shared memory when it exits
                const long long t0 = clock64();
                while (clock64() - t0 < kWaitLimitCycles / 100) {}
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------ MMA issuer
            if (elect_one()) {
                int it = 0, n_q = 0;
                uint32_t tiles_seen = 0, units_seen = 0;  // bit m: parity of the tiles / units of warpgroup m so far
                auto wait = [&](uint64_t* bar, uint32_t parity) {
                    const bool ok = mbar_wait_bounded(smem_u32(bar), parity, abort_flag, p.status, FAULT_PROMPT_WAIT);
                    tc_fence_after();
                    return ok;
                };
                auto wait_stage = [&](int i) { return wait(&t.full[i % kApStages], (uint32_t)((i / kApStages) & 1)); };
                const uint32_t q_low = ap_desc(sm_q), ring_low = ap_desc(sm_ring);
                auto scores = [&](int m, int q_tile, int i) {  // S[m] = Q K^T
                    const uint32_t a = q_low + q_tile * (L::kTile >> 4), b = ring_low + (i % kApStages) * (L::kTile >> 4);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const int off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
                        ap_mma_ss(tmem + m * 128, a + off, b + off, IDESC_QK, k > 0);
                    }
                    tc_commit(smem_u32(&t.s_full[m]));
                };
                // O[m] (+)= P V for one half of the keys.  V is stored [key][64 elements], so the MMA's N runs along the contiguous
                // dimension; 64-element column blocks lie 16 KB apart (the stride in the descriptor), groups of eight keys 1 KB.
                auto values = [&](int m, int i, bool fresh, int half) {
                    const uint32_t b = (ring_low + (i % kApStages) * (L::kTile >> 4) + half * (8192 >> 4)) | (D > 64 ? (16384u >> 4) << 16 : 0u);
#pragma unroll
                    for (int k = 0; k < kApKeys / 32; ++k)
                        ap_mma_ts(tmem + 256 + m * D, tmem + m * 128 + half * 32 + k * 8, b + k * (2048 >> 4), IDESC_PV, !(fresh && k == 0));
                };
                auto free_stage = [&](int i) { tc_commit(smem_u32(&t.empty[i % kApStages])); };
                // O[m] (+)= P[m] V as the halves of P come; for the first tile of a unit O[m] has to be drained first
                auto add_values = [&](int m, int i, bool fresh, bool wait_v) {
                    if (!wait(&t.h_full[m], (tiles_seen >> m) & 1u)) return false;
                    if (fresh) {
                        if (!wait(&t.o_empty[m], ((units_seen >> m) & 1u) ^ 1u)) return false;
                        units_seen ^= 1u << m;
                    }
                    if (wait_v && !wait_stage(i)) return false;
                    values(m, i, fresh, 0);
                    if (!wait(&t.p_full[m], (tiles_seen >> m) & 1u)) return false;
                    tiles_seen ^= 1u << m;
                    values(m, i, false, 1);
                    return true;
                };
                while (const ApSegment* sp = next_segment()) {
                    const int cnt = sp->cnt, dual = sp->dual;
                    release();
                    if (cnt == 0) continue;
                    if (!wait(&t.q_full, (uint32_t)(n_q & 1))) break;
                    ++n_q;
                    if (!dual) {
                        // every K and V tile serves both tiles of queries
                        if (!wait_stage(it)) break;
                        scores(0, 0, it);
                        scores(1, 1, it);
                        free_stage(it);
                        ++it;
                        if (cnt == 1) tc_commit(smem_u32(&t.q_empty));
#pragma unroll 1
                        for (int i = 0; i < cnt && !*abort_flag; ++i) {
                            const bool next = i + 1 < cnt;
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                if (!add_values(m, it, i == 0, m == 0)) break;
                                if (m == 1) free_stage(it);
                                if (next) {
                                    if (m == 0 && !wait_stage(it + 1)) break;
                                    scores(m, m, it + 1);
                                    if (m == 1) free_stage(it + 1);
                                } else {
                                    tc_commit(smem_u32(&t.o_full[m]));
                                }
                            }
                            if (i + 2 == cnt) tc_commit(smem_u32(&t.q_empty));
                            it += next ? 2 : 1;
                        }
                    } else {
                        // tile i of the keys belongs to warpgroup i & 1
#pragma unroll 1
                        for (int i = 0; i < 2 && i < cnt; ++i) {
                            if (!wait_stage(it)) break;
                            scores(i, 0, it);
                            free_stage(it);
                            ++it;
                        }
                        if (cnt <= 2) tc_commit(smem_u32(&t.q_empty));
#pragma unroll 1
                        for (int i = 0; i < cnt && !*abort_flag; ++i) {
                            const int m = i & 1;
                            if (!add_values(m, it, i < 2, true)) break;
                            free_stage(it);
                            ++it;
                            if (i + 2 < cnt) {
                                if (!wait_stage(it)) break;
                                scores(m, 0, it);
                                free_stage(it);
                                ++it;
                                if (i + 3 == cnt) tc_commit(smem_u32(&t.q_empty));
                            } else {
                                tc_commit(smem_u32(&t.o_full[m]));
                            }
                        }
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        if (!idle) {
            // ------------------------------------------------------------ softmax, one row per thread
            const int m = warp >> 2;                                    // tile
            const int r = (warp & 3) * 32 + lane;                       // row of the tile
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t t_s = tmem + lanes + m * 128, t_o = tmem + lanes + 256 + m * D;
            const int r_tok = r / p.G, r_head = r - r_tok * p.G;
            uint32_t n_tile = 0, n_unit = 0, n_turn = 0, n_other = 0;  // n_other: units of warpgroup 1, as warpgroup 0 counts them
            while (const ApSegment* sp = next_segment()) {
                const ApSegment& seg = *sp;  // stays in shared memory until the end of the segment
                const int cnt = seg.cnt, dual = seg.dual;
                const int first = dual ? 0 : m * p.tpt, tok = first + r_tok;  // within the unit
                const bool live = r_tok < p.tpt && tok < seg.tokens;
                // keys that this query sees, and that all queries of the tile see, counted from the CTA's first key
                const int from = seg.ks * kApKeys;
                const int limit = live ? seg.sees + tok - from : 0, all_see = seg.sees + first - from;
                const int my0 = dual ? m : 0, step = dual ? 2 : 1;
                float mx = -INFINITY, sum = 0.f;
                auto row_max = [](const float (&s)[kApKeys]) {
                    float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int c = 4; c < kApKeys; c += 8) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) top[e] = c + 4 + e < kApKeys ? max3(top[e], s[c + e], s[c + 4 + e]) : fmaxf(top[e], s[c + e]);
                    }
                    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                };
#pragma unroll 1
                for (int i = my0; i < cnt; i += step) {
                    const int key0 = i * kApKeys;
                    mbar_wait_bounded(smem_u32(&t.s_full[m]), n_tile & 1u, abort_flag, p.status, FAULT_PROMPT_WAIT);
                    ++n_tile;
                    tc_fence_after();
                    float s[kApKeys];
#pragma unroll
                    for (int c = 0; c < kApKeys; c += 32) tmem_ld32(t_s + c, s + c);
                    tmem_ld_wait();
                    if (key0 + kApKeys > all_see) {
#pragma unroll
                        for (int c = 0; c < kApKeys; ++c)
                            if (key0 + c >= limit) s[c] = -INFINITY;
                    }
                    if (i == my0) mx = row_max(s);
                    // The tiles take turns: side by side they would both exponentiate at half speed and then both wait for
                    // the tensor cores.
                    if (!dual) {
                        mbar_wait_bounded(smem_u32(&t.turn[m]), (n_turn & 1u) ^ (m == 0 ? 1u : 0u), abort_flag, p.status, FAULT_PROMPT_WAIT);
                        ++n_turn;
                    }
                    // The first half is exponentiated against the maximum of the blocks before, while this block's is being found: it
                    // hardly ever matters (the comment at the top), and the search costs nothing next to the MUFU.
                    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
                    float2 add[2];
                    uint32_t w[32];
                    auto first_half = [&]() {
                        const float shift = mx == -INFINITY ? 0.f : mx * p.scale_log2;
                        const float2 shift2 = make_float2(-shift, -shift);
                        add[0] = add[1] = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float2 x = fma2(make_float2(s[2 * e], s[2 * e + 1]), scale2, shift2);
                            x.x = exp2_approx(x.x), x.y = exp2_approx(x.y);
                            add[e & 1] = add2(add[e & 1], x);
                            w[e] = pack_bf16(x.x, x.y);
                        }
                    };
                    first_half();
                    const float higher = fmaxf(mx, row_max(s));
                    // all keys so far masked: nothing has been summed, and the factor is exp2(-inf) = 0
                    const bool grow = (higher - mx) * p.scale_log2 > 8.f;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? exp2_approx((mx - higher) * p.scale_log2) : 1.f;
                        if (grow) mx = higher;
                        sum *= f;
                        if (i != my0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                float o[16];
                                uint32_t u[16];
                                tmem_ld16(t_o + c, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * f);
                                tmem_st16(t_o + c, u);
                            }
                        }
                        first_half();
                    }
                    tmem_st16(t_s, w), tmem_st16(t_s + 16, w + 16);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&t.h_full[m]));  // half of P is there: its products may start
                    const float shift = mx == -INFINITY ? 0.f : mx * p.scale_log2;
                    const float2 shift2 = make_float2(-shift, -shift);
#pragma unroll
                    for (int c = kApKeys / 2; c < kApKeys; c += 32) {
                        uint32_t v[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 x = fma2(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), scale2, shift2);
                            x.x = exp2_approx(x.x), x.y = exp2_approx(x.y);
                            add[e & 1] = add2(add[e & 1], x);
                            v[e] = pack_bf16(x.x, x.y);
                        }
                        tmem_st16(t_s + c / 2, v);
                        if (c == 64 && !dual) {  // the rest of this tile and the start of the other one fill each other's gaps
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(&t.turn[1 - m]));
                        }
                    }
                    sum += (add[0].x + add[1].x) + (add[0].y + add[1].y);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&t.p_full[m]));
                }
                // ---- end of the segment
                const bool mine = my0 < cnt, whole = cnt == seg.tiles, two = dual && cnt > 1;
                if (mine) {
                    mbar_wait_bounded(smem_u32(&t.o_full[m]), n_unit & 1u, abort_flag, p.status, FAULT_PROMPT_WAIT);
                    ++n_unit;
                    tc_fence_after();
                }
                // Two sums over the same rows meet here: warpgroup 0 reads the other one's O from tensor memory (the same lanes).
                float w0 = 1.f, w1 = 0.f;
                bool writes = true;
                if (dual) {
                    if (two && m == 1) t.stat[0][r] = mx, t.stat[1][r] = sum;
                    named_bar_sync(1, 256);
                    writes = m == 0;
                    if (two && m == 0) {
                        mbar_wait_bounded(smem_u32(&t.o_full[1]), n_other & 1u, abort_flag, p.status, FAULT_PROMPT_WAIT);
                        tc_fence_after();
                        const float mx1 = t.stat[0][r], top = fmaxf(mx, mx1);
                        w0 = mx == -INFINITY ? 0.f : exp2_approx((mx - top) * p.scale_log2);
                        w1 = mx1 == -INFINITY ? 0.f : exp2_approx((mx1 - top) * p.scale_log2);
                        sum = w0 * sum + w1 * t.stat[1][r];
                        mx = top;
                    }
                }
                if (two || (!dual && cnt > 0)) ++n_other;
                if (writes) {
                    // 16 columns of the row's O; the other warpgroup's lie D columns behind
                    auto columns = [&](int c, float (&o)[16]) {
                        tmem_ld16(t_o + c, o);
                        if (two) {
                            float o1[16];
                            tmem_ld16(t_o + D + c, o1);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = w0 * o[e] + w1 * o1[e];
                        } else {
                            tmem_ld_wait();
                        }
                    };
                    auto drained = [&]() {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(smem_u32(&t.o_empty[m]));
                            if (two) mbar_arrive(smem_u32(&t.o_empty[1]));
                        }
                    };
                    if (whole) {
                        const bool store = live && !*abort_flag;
                        const float inv = 1.0f / sum;
                        bf16* out = p.Out + (long long)(seg.token + tok) * p.ldo + (long long)(seg.head * p.G + r_head) * D;
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            if (mine) columns(c, o);
                            uint32_t w[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q)  // a query that sees no key gives zero
                                w[q] = limit > 0 ? pack_bf16(o[2 * q] * inv, o[2 * q + 1] * inv) : 0u;
                            if (store) store_row16(out + c, w, p.out32);
                            __syncwarp();
                        }
                        if (mine) drained();
                    } else {
                        constexpr long long kPart = (long long)(D + 2) * 128;
                        float* part = p.parts + (seg.slot * 2 + m) * kPart;
                        if (live) __stcg(part + (long long)D * 128 + r, mx), __stcg(part + (long long)(D + 1) * 128 + r, sum);
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            columns(c, o);
                            if (live) {
#pragma unroll
                                for (int e = 0; e < 16; e += 4)
                                    __stcg(reinterpret_cast<float4*>(part) + (c + e) / 4 * 128 + r, make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                            }
                            __syncwarp();
                        }
                        drained();
                        const int writers = dual ? 128 : 256;
                        named_bar_sync(dual ? 2 : 1, writers);  // behind it thread 0 speaks for all
                        if (tid == 0) {
                            // One counter per share: of the units that start in it only the last can be cut.
                            __threadfence();
                            t.last = atomicAdd(p.count + seg.c0, (unsigned)cnt) + (unsigned)cnt == (unsigned)seg.tiles;
                            if (t.last) p.count[seg.c0] = 0u;
                            __threadfence();
                        }
                        if (warp == 1) {
                            // meanwhile the parts that there are, in the order of the keys
                            int n = 0;
                            for (int c0 = seg.c0; c0 <= seg.c1; c0 += 32) {
                                const int c = c0 + lane;
                                const bool has = c <= seg.c1 && ap_tile_at(ap_share(line, c + 1), seg.x0, seg.tiles, seg.dual) >
                                                                    ap_tile_at(ap_share(line, c), seg.x0, seg.tiles, seg.dual);
                                const uint32_t all = __ballot_sync(0xffffffffu, has);
                                if (has) t.list[n + __popc(all & ((1u << lane) - 1u))] = (short)(2 * (2 * c + (c == seg.c0 ? 1 : 0)));
                                n += __popc(all);
                            }
                            if (lane == 0) t.parts = n;
                        }
                        named_bar_sync(dual ? 2 : 1, writers);
                        if (t.last && !*abort_flag) {
                            if (seg.tokens * p.G > 32) ap_join<D, 8, 2>(p, seg, t.list, t.parts, tid, writers);
                            else if (seg.tokens * p.G > 8) ap_join<D, 4, 4>(p, seg, t.list, t.parts, tid, writers);
                            else ap_join<D, 1, 8>(p, seg, t.list, t.parts, tid, writers);
                        }
                        named_bar_sync(dual ? 2 : 1, writers);  // the list and the flag are free again
                    }
                }
                __syncwarp();
                if (lane == 0) release();
                else ++n_seg;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- host ---------------------------------------------------------------------
static constexpr int kApMaxGrid = 160;

static int attn_prompt_grid() { return sm_count() < kApMaxGrid ? sm_count() : kApMaxGrid; }

size_t attn_prompt_workspace_bytes(int D) {
    return (size_t)kApMaxGrid * 4 + (size_t)attn_prompt_grid() * 4 * (D + 2) * 128 * sizeof(float);
}

// bf16 [d2][d1][d0] with element strides; box [b2][b1][64], 128-byte swizzle, zeros out of range
static bool encode_3d(CUtensorMap* map, const bf16* base, long long d0, long long d1, long long d2, long long s1, long long s2, int b1, int b2) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
    cuuint64_t strides[2] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)b1, (cuuint32_t)b2}, one[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
static cudaError_t launch_attn_prompt_d(const AttnPromptArgs& a, const ApParams& p, cudaStream_t stream) {
    alignas(64) CUtensorMap mq, mk, mv;
    const long long P = 1ll << a.page_shift, z = (long long)a.num_pages * a.NKV;
    if (!encode_3d(&mq, a.Q, D, a.H, a.T, D, a.ldq, p.G, p.tpt) || !encode_3d(&mk, a.K, D, P, z, D, P * D, 64, 1) ||
        !encode_3d(&mv, a.V, D, P, z, D, P * D, 64, 1))
        return cudaErrorInvalidValue;
    static std::atomic<bool> configured[64];
    if (cudaError_t e = allow_smem_once(attn_prompt_kernel<D>, ApSmem<D>::kBytes, configured)) return e;
    chain_begin();
    return launch_pdl(attn_prompt_kernel<D>, dim3((unsigned)attn_prompt_grid()), dim3(kApThreads), ApSmem<D>::kBytes, stream, mq, mk, mv, p);
}

cudaError_t launch_attn_prompt(const AttnPromptArgs& a, cudaStream_t stream) {
    ApParams p;
    p.Out = a.Out, p.ldo = a.ldo;
    p.table = a.page_table, p.lens = a.seq_lens, p.cu = a.cu_tokens;
    p.count = static_cast<unsigned int*>(a.workspace);
    p.parts = reinterpret_cast<float*>(static_cast<unsigned char*>(a.workspace) + kApMaxGrid * 4);
    p.B = a.B, p.T = a.T, p.H = a.H, p.NKV = a.NKV, p.G = a.H / a.NKV, p.tpt = 128 / p.G;
    p.max_pages = a.max_pages, p.page_shift = a.page_shift, p.num_pages = a.num_pages;
    p.out32 = (reinterpret_cast<uintptr_t>(a.Out) & 31u) == 0 && a.ldo % 16 == 0;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a.D));
    p.status = status_ptr();
    if (!p.status) return cudaErrorUnknown;
    return a.D == 64 ? launch_attn_prompt_d<64>(a, p, stream) : launch_attn_prompt_d<128>(a, p, stream);
}

}  // namespace ezb
