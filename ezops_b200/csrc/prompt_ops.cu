// The small kernels of a step over paged KV caches that carries prompts as well as single tokens: the plan of the
// step (page tables, slots and positions from request lengths) and the head norm + rotary embedding + cache write of
// its tokens.
#include "launchers.h"
#include "prompt.h"

namespace ezb {

// ------------------------------------------------------------------- plan ---
// With h(x) = ceil(x / page_size), c_b cached and n_b new tokens of row b (offsets cu = running sum of n, cut at
// max_tokens):
//   table[b, j] = free[count - 1 - (sum of rows before b of (h(c+n) - h(c))) - (j - h(c_b))],   h(c_b) <= j < h(c_b + n_b)
//   token t of row b: position c_b + t - cu[b], slot = table[b, position / page_size] * page_size + position % page_size.
// What bounds it: latency - three dependent reads (lengths, then table or free list) and two block-wide running sums.
// Every CTA therefore forms the sums over all rows by itself (8 KB of lengths for 1024 rows, from L2) instead of
// waiting for another CTA, keeps them in shared memory and finds the row of a token there by bisection.  A token in a page
// that this call maps reads the free list itself, so no CTA reads a table entry that another one writes.
// Measured: 32 rows and tokens 3.5 us, 512 rows and 16384 tokens 7.2 us on the GPU; a call among others 8.1 to 8.8 us, the host's.
static constexpr int kPlanThreads = 256;
static constexpr int kPlanTokens = 1024;  // tokens per CTA

struct PlanParams {
    const int *ctx, *fresh, *free_pages, *free_count;
    int *table, *lens, *cu, *positions, *slots, *free_left;
    int B, T, max_pages, page_shift, num_pages, free_size;
};

// a + b, cut at cap.  All three lie between 0 and 2^30, so that the sum may reach 2^31: one more than an int holds.
__device__ __forceinline__ int cut_add(int a, int b, int cap) { return (int)min((unsigned)a + (unsigned)b, (unsigned)cap); }
// Exclusive running sum over the block's threads; the total in `total`.  Sums are cut at `cap`, and every value is at most that.
__device__ __forceinline__ int block_prefix(int v, int cap, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s = cut_add(s, up, cap);
    }
    __syncthreads();  // warp_sums may still be read from the sum before
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w == warp) before = all;
        all = cut_add(all, warp_sums[w], cap);
    }
    total = all;
    int up = __shfl_up_sync(0xffffffffu, s, 1);
    if (lane == 0) up = 0;
    return cut_add(before, up, cap);
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
    pdl_open(1);
    extern __shared__ int plan_smem[];
    int* cu = plan_smem;             // [B + 1] first token of a row
    int* base = plan_smem + p.B + 1;  // [B] new pages of the rows in front
    __shared__ int warp_sums[kPlanThreads / 32];
    const int tid = threadIdx.x;
    const int page = 1 << p.page_shift, cap = p.max_pages << p.page_shift;
    const int rows = (p.B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(tid * rows, p.B), b1 = min(b0 + rows, p.B);
    const int count = min(__ldg(p.free_count), p.free_size);
    auto cached = [&](int b) { return min(max(__ldg(p.ctx + b), 0), cap); };
    auto held = [&](int c) { return (int)(((long long)c + page - 1) >> p.page_shift); };
    auto fresh = [&](int b) { return min(max(__ldg(p.fresh + b), 0), p.T); };

    int sum = 0, total = 0;
    for (int b = b0; b < b1; ++b) sum = cut_add(sum, fresh(b), p.T);
    int at = block_prefix(sum, p.T, warp_sums, total);
    if (tid == 0) cu[p.B] = total;
    sum = 0;
    for (int b = b0; b < b1; ++b) {
        cu[b] = at;
        const int next = cut_add(at, fresh(b), p.T), c = cached(b);
        base[b] = sum;  // completed below
        sum += held(cut_add(c, next - at, cap)) - held(c);
        at = next;
    }
    int pages = 0;
    const int first = block_prefix(sum, 1 << 30, warp_sums, pages);
    for (int b = b0; b < b1; ++b) base[b] += first;
    __syncthreads();

    auto valid = [&](int id) { return id >= 0 && id < p.num_pages ? id : -1; };
    auto new_page = [&](int k) {  // k-th page that this step takes
        const int i = count - 1 - k;
        return i >= 0 ? valid(__ldg(p.free_pages + i)) : -1;
    };
    if (blockIdx.x == 0) {
        for (int b = tid; b <= p.B; b += kPlanThreads) {
            p.cu[b] = cu[b];
            if (b < p.B) p.lens[b] = cut_add(cached(b), cu[b + 1] - cu[b], cap);
        }
        if (tid == 0) *p.free_left = count - pages;
    }
    // table entries: a warp per row
    for (int b = blockIdx.x * (kPlanThreads / 32) + (tid >> 5); b < p.B; b += gridDim.x * (kPlanThreads / 32)) {
        const int n = cu[b + 1] - cu[b];
        if (n == 0) continue;
        const int c = cached(b), h = held(c), need = held(cut_add(c, n, cap));
        for (int j = h + (tid & 31); j < need; j += 32) p.table[(long long)b * p.max_pages + j] = new_page(base[b] + j - h);
    }
    for (int t = blockIdx.x * kPlanTokens + tid; t < min((blockIdx.x + 1) * kPlanTokens, p.T); t += kPlanThreads) {
        int pos = -1, slot = -1;
        if (t < total) {
            int lo = 0, hi = p.B;  // the last row whose first token is at most t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int c = cached(lo), h = held(c);
            pos = c + t - cu[lo];
            if (pos < cap) {
                const int j = pos >> p.page_shift;
                const int id = j < h ? valid(p.table[(long long)lo * p.max_pages + j]) : new_page(base[lo] + j - h);
                if (id >= 0) slot = (id << p.page_shift) + (pos & (page - 1));
            }
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
}

cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t stream) {
    PlanParams p;
    p.ctx = a.ctx_lens, p.fresh = a.new_lens, p.free_pages = a.free_pages, p.free_count = a.free_count;
    p.table = a.page_table, p.lens = a.seq_lens, p.cu = a.cu_tokens, p.positions = a.positions, p.slots = a.slots;
    p.free_left = a.free_left;
    p.B = a.B, p.T = a.T, p.max_pages = a.max_pages, p.page_shift = a.page_shift, p.num_pages = a.num_pages;
    p.free_size = a.free_size;
    int grid = (a.T + kPlanTokens - 1) / kPlanTokens;
    const int row_ctas = (a.B + 31) / 32;  // four rows per warp
    if (grid < row_ctas) grid = row_ctas;
    const size_t smem = (size_t)(2 * a.B + 1) * sizeof(int);
    if (smem > 47 * 1024) {  // 48 KB without opting in
        cudaError_t e = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    chain_begin();
    return launch_pdl(paged_plan_kernel, dim3((unsigned)grid), dim3(kPlanThreads), smem, stream, p);
}

// ---------------------------------------- head norm + rotary + paged write ---
// For token t, head vector x and frequency i < D/2 with axis a(i), position p = positions[a(i), t]:
//   n = x / sqrt(mean(x^2) + eps) * w
//   y_i = n_i cos[p, i] - n_{i+D/2} sin[p, i],   y_{i+D/2} = n_{i+D/2} cos[p, i+D/2] + n_i sin[p, i+D/2]
// in fp32 with one rounding, as the stand-alone operator of a decode step and the decode attention do.
// What bounds it: HBM for prompts (every head is read and written once: 8189 tokens of 32 heads with three axes 27 us, 137 MB,
// 5.1 TB/s), latency for a handful of tokens (32 tokens of 48 heads 2.2 us).  A head is D/8 lanes, each with four elements of
// its first half and their partners in the second, so that a rotation stays inside a lane, and two elements share an
// instruction.  A warp keeps the cos and sin values of ONE token in registers for all the heads it walks; how many that are
// (`steps`) follows from the number of tokens: one group of heads per warp while there are fewer warps than the chip holds,
// more when the table rows would otherwise be fetched again for every group (36.8 -> 27.9 us, and 27.0 with the next heads
// requested before these are worked off).
struct PagedRopeParams {
    const bf16* qkv;
    long long ld;
    const bf16 *qw, *kw, *cos, *sin;
    const int *positions, *slots;
    bf16 *K, *V, *q_out;
    int T, H, NKV, S, axes, page_shift, steps, chunks;
    long long n_slots;
    float eps;
    unsigned int* status;
    alignas(4) unsigned char axis[64];  // axis of frequency i
};

static constexpr int kRopeBatch = 2;  // heads that a lane works off while as many are on their way (more take too many registers)
__device__ __forceinline__ uint2 ld_stream8(const bf16* p) {  // read once
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

template <int D>
__global__ void __launch_bounds__(128, 7) paged_qk_norm_rope_kernel(const __grid_constant__ PagedRopeParams p) {
    constexpr int LPH = D / 8, HPW = 32 / LPH;  // lanes per head, heads per warp
    pdl_open(1);
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(unit / p.chunks), chunk = (int)(unit - (long long)t * p.chunks);
    if (t >= p.T) return;
    const int f0 = (lane & (LPH - 1)) * 4;  // first frequency of this lane: it holds the elements f0.. and D/2 + f0..
    const int heads = p.H + 2 * p.NKV;

    // Everything that does not depend on the position is requested together with it: the heads, the weights, the slot.
    const int h0 = chunk * p.steps * HPW + lane / LPH;
    const bf16* src = p.qkv + (long long)t * p.ld + (long long)h0 * D + f0;
    uint2 lo[2][kRopeBatch], hi[2][kRopeBatch];
    auto load = [&](int i, int z) {
#pragma unroll
        for (int u = 0; u < kRopeBatch; ++u)
            if (i + u < p.steps && h0 + (i + u) * HPW < heads)
                lo[z][u] = ld_stream8(src + (long long)(i + u) * HPW * D), hi[z][u] = ld_stream8(src + (long long)(i + u) * HPW * D + D / 2);
    };
    load(0, 0);
    int pos[3];
    bool real = true, inside = true;
#pragma unroll
    for (int a = 0; a < 3; ++a) {
        pos[a] = a < p.axes ? __ldg(p.positions + (long long)a * p.T + t) : 0;
        real = real && pos[a] >= 0;
        inside = inside && pos[a] < p.S;
    }
    const int slot = __ldg(p.slots + t);
    const uint2 one = make_uint2(0x3f803f80u, 0x3f803f80u);
    auto weights = [&](const bf16* w, int at) { return w ? __ldg(reinterpret_cast<const uint2*>(w + at)) : one; };
    const uint2 qw1 = weights(p.qw, f0), qw2 = weights(p.qw, D / 2 + f0), kw1 = weights(p.kw, f0), kw2 = weights(p.kw, D / 2 + f0);
    if (!real) return;  // a padded token: nothing is written
    if (!inside) {
        if (lane == 0) report_fault(p.status, FAULT_ROPE_POSITION);
        return;
    }
    const bool cached = slot >= 0 && slot < p.n_slots;
    if (slot >= p.n_slots && lane == 0) report_fault(p.status, FAULT_SLOT_RANGE);

    // Table rows: the lane's columns of every axis; the axis of each frequency picks, 16 bits at a time.
    auto unpack = [](const uint2& v, float2 (&x)[2]) {
        x[0] = make_float2(bf16_lo(v.x), bf16_hi(v.x)), x[1] = make_float2(bf16_lo(v.y), bf16_hi(v.y));
    };
    float2 c1[2], c2[2], s1[2], s2[2];
    if (chunk * p.steps * HPW < p.H + p.NKV) {  // a warp with v heads only copies
        const uint32_t axes4 = *reinterpret_cast<const uint32_t*>(p.axis + f0);
        uint2 row[4];  // cos of the first and second half, sin of the first and second half
#pragma unroll
        for (int a = 0; a < 3; ++a) {
            if (a < p.axes) {
                const bf16 *cr = p.cos + (long long)pos[a] * D + f0, *sr = p.sin + (long long)pos[a] * D + f0;
                const uint2 x[4] = {__ldg(reinterpret_cast<const uint2*>(cr)), __ldg(reinterpret_cast<const uint2*>(cr + D / 2)),
                                    __ldg(reinterpret_cast<const uint2*>(sr)), __ldg(reinterpret_cast<const uint2*>(sr + D / 2))};
                auto half = [&](int i) { return ((axes4 >> (8 * i)) & 255u) == (uint32_t)a ? 0xffffu : 0u; };
                const uint32_t m0 = a ? half(0) | half(1) << 16 : ~0u, m1 = a ? half(2) | half(3) << 16 : ~0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    row[i].x = a ? (row[i].x & ~m0) | (x[i].x & m0) : x[i].x;
                    row[i].y = a ? (row[i].y & ~m1) | (x[i].y & m1) : x[i].y;
                }
            }
        }
        row[2].x ^= 0x80008000u, row[2].y ^= 0x80008000u;
        unpack(row[0], c1), unpack(row[1], c2), unpack(row[2], s1), unpack(row[3], s2);
    }
    const long long page = slot >> p.page_shift, off = slot & ((1 << p.page_shift) - 1);
    bf16* q_row = p.q_out + (long long)t * p.H * D + f0;
    const long long kv_row = ((page * p.NKV) << p.page_shift) + off;  // + kv head * page size
#pragma unroll 1
    for (int i2 = 0; i2 < p.steps; i2 += 2 * kRopeBatch) {
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int i = i2 + z * kRopeBatch;
            if (i >= p.steps) break;
            load(i + kRopeBatch, 1 - z);
#pragma unroll
            for (int u = 0; u < kRopeBatch; ++u) {
                if (i + u >= p.steps) break;
                const int h = h0 + (i + u) * HPW;
                const bool live = h < heads, is_v = h >= p.H + p.NKV, is_q = h < p.H;
                uint2 out1 = lo[z][u], out2 = hi[z][u];
                if ((chunk * p.steps + i + u) * HPW < p.H + p.NKV) {  // the same for the whole warp
                    float2 a[2], b[2], w1[2], w2[2];
                    unpack(lo[z][u], a), unpack(hi[z][u], b);
                    unpack(is_q ? qw1 : kw1, w1), unpack(is_q ? qw2 : kw2, w2);
                    float2 sq = mul2(a[0], a[0]);
                    sq = fma2(a[1], a[1], sq), sq = fma2(b[0], b[0], sq), sq = fma2(b[1], b[1], sq);
                    float ssq = sq.x + sq.y;
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ssq += __shfl_xor_sync(0xffffffffu, ssq, o);
                    const float r = rsqrtf(ssq * (1.0f / D) + p.eps);
                    const float2 r2 = make_float2(r, r);
                    float2 y1[2], y2[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 n1 = mul2(mul2(a[e], r2), w1[e]), n2 = mul2(mul2(b[e], r2), w2[e]);
                        y1[e] = add2(mul2(n1, c1[e]), mul2(n2, s1[e]));
                        y2[e] = add2(mul2(n2, c2[e]), mul2(n1, s2[e]));
                    }
                    if (!is_v) {
                        out1 = make_uint2(pack_bf16(y1[0].x, y1[0].y), pack_bf16(y1[1].x, y1[1].y));
                        out2 = make_uint2(pack_bf16(y2[0].x, y2[0].y), pack_bf16(y2[1].x, y2[1].y));
                    }
                }
                bf16* dst = q_row + (long long)h * D;
                if (!is_q) {
                    const long long row = kv_row + ((long long)(h - p.H - (is_v ? p.NKV : 0)) << p.page_shift);
                    dst = (is_v ? p.V : p.K) + row * D + f0;
                }
                if (live && (is_q || cached)) {
                    *reinterpret_cast<uint2*>(dst) = out1;
                    *reinterpret_cast<uint2*>(dst + D / 2) = out2;
                }
            }
        }
    }
}

cudaError_t launch_paged_qk_norm_rope(const PagedRopeArgs& a, cudaStream_t stream) {
    PagedRopeParams p;
    p.qkv = a.qkv, p.ld = a.ld, p.qw = a.qw, p.kw = a.kw, p.cos = a.cos, p.sin = a.sin;
    p.positions = a.positions, p.slots = a.slots, p.K = a.K, p.V = a.V, p.q_out = a.q_out;
    p.T = a.T, p.H = a.H, p.NKV = a.NKV, p.S = a.S, p.axes = a.axes, p.page_shift = a.page_shift;
    p.n_slots = (long long)a.num_pages << a.page_shift;
    p.eps = a.eps;
    p.status = status_ptr();
    if (!p.status) return cudaErrorUnknown;
    for (int i = 0; i < 64; ++i) p.axis[i] = i < a.D / 2 ? a.axis_of_frequency[i] : 0;
    const int per_warp = 32 / (a.D / 8), groups = (a.H + 2 * a.NKV + per_warp - 1) / per_warp;
    const long long fill = (long long)sm_count() * 32;
    p.steps = 1;
    while (p.steps < groups && (long long)a.T * ((groups + 2 * p.steps - 1) / (2 * p.steps)) >= fill) p.steps *= 2;
    p.chunks = (groups + p.steps - 1) / p.steps;
    const long long warps = (long long)a.T * p.chunks;
    chain_begin();
    if (a.D == 64) return launch_pdl(paged_qk_norm_rope_kernel<64>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, p);
    return launch_pdl(paged_qk_norm_rope_kernel<128>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, p);
}

}  // namespace ezb
