// C entries of the prompt operators (declared in include/ezb200.h): argument checks, then one launch each.
#include <cstring>
#include <type_traits>
#include <utility>

#include "prompt.h"

using namespace ezb;

namespace {

int shift_of(int page_size) {  // log2 of a power of two >= 64, else -1
    if (page_size < 64 || (page_size & (page_size - 1))) return -1;
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

// Whether two row-major arrays of `rows` rows share a byte: `width` bytes of every `ld` bytes.
struct Rect {
    const void* base;
    long long rows, ld, width;
};
bool overlap(const Rect& a, const Rect& b) {
    const long long pa = (long long)reinterpret_cast<uintptr_t>(a.base), pb = (long long)reinterpret_cast<uintptr_t>(b.base);
    const long long ea = pa + (a.rows - 1) * a.ld + a.width, eb = pb + (b.rows - 1) * b.ld + b.width;
    if (ea <= pb || eb <= pa) return false;
    if (a.ld != b.ld) return true;
    // columns of one wider array: disjoint unless their columns meet
    const long long off = ((pb - pa) % a.ld + a.ld) % a.ld;
    return off < a.width || off + b.width > a.ld;
}
Rect span(const void* base, long long bytes) { return {base, 1, bytes, bytes}; }
// Whether any of the arrays that a call writes meets another of them, or one that it only reads (null: not there).
template <size_t W, size_t R>
bool any_overlap(const Rect (&writes)[W], const Rect (&reads)[R]) {
    for (size_t i = 0; i < W; ++i) {
        for (size_t j = 0; j < i; ++j)
            if (overlap(writes[i], writes[j])) return true;
        for (const Rect& r : reads)
            if (r.base && overlap(writes[i], r)) return true;
    }
    return false;
}

constexpr int kMost = 1 << 30;  // sizes, positions and slots are 32-bit on the device

// A call whose arguments are 64-bit words: pointers, sizes, and a float as its bits.
template <class T>
T from_word(long long w) {
    if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>(static_cast<uintptr_t>(w));
    else if constexpr (std::is_same_v<T, float>) {
        const int bits = static_cast<int>(w);
        float f;
        memcpy(&f, &bits, sizeof(f));
        return f;
    } else return static_cast<T>(w);
}
template <class T>
bool holds(long long w) {  // whether an argument of this type keeps the whole word (a float is its low 32 bits)
    if constexpr (std::is_same_v<T, int>) return w == static_cast<int>(w);
    else return true;
}
template <class... A, size_t... I>
int call_words(int (*f)(A...), const long long* w, std::index_sequence<I...>) {
    EZB_REQUIRE_SHAPE((holds<A>(w[I]) && ...), "a size does not fit in 32 bits");
    return f(from_word<A>(w[I])...);
}
template <class... A>
int call_packed(int (*f)(A...), const long long* w) {
    EZB_REQUIRE(w, "null pointer");
    return call_words(f, w, std::index_sequence_for<A...>{});
}

}  // namespace

extern "C" {

int ezb_paged_plan(const int* ctx_lens, const int* new_lens, int* page_table, const int* free_pages, const int* free_count,
                   int* seq_lens, int* cu_tokens, int* positions, int* slots, int* free_left, int B, int max_tokens, int max_pages,
                   int page_size, int num_pages, int free_size, ezb_stream_t stream) {
    EZB_REQUIRE(ctx_lens && new_lens && page_table && free_pages && free_count && seq_lens && cu_tokens && positions && slots && free_left,
                "null pointer");
    EZB_REQUIRE(B >= 1 && max_tokens >= 1 && max_pages >= 1 && num_pages >= 1 && free_size >= 1, "sizes must be positive");
    EZB_REQUIRE_SHAPE(shift_of(page_size) >= 0, "page_size must be a power of two >= 64");
    EZB_REQUIRE_SHAPE(B <= kPlanMaxRows, "at most 8192 rows");
    EZB_REQUIRE_SHAPE(max_tokens <= kMost && (long long)max_pages * page_size <= kMost && (long long)num_pages * page_size <= kMost,
                      "max_tokens, max_pages * page_size and num_pages * page_size are limited to 2^30");
    const Rect writes[] = {span(page_table, 4ll * B * max_pages), span(seq_lens, 4ll * B), span(cu_tokens, 4ll * (B + 1)),
                           span(positions, 4ll * max_tokens), span(slots, 4ll * max_tokens), span(free_left, 4)};
    const Rect reads[] = {span(ctx_lens, 4ll * B), span(new_lens, 4ll * B), span(free_pages, 4ll * free_size), span(free_count, 4)};
    EZB_REQUIRE(!any_overlap(writes, reads), "an output overlaps an input or another output (results go to tensors of their own)");
    PlanArgs p;
    p.ctx_lens = ctx_lens, p.new_lens = new_lens, p.free_pages = free_pages, p.free_count = free_count, p.page_table = page_table;
    p.seq_lens = seq_lens, p.cu_tokens = cu_tokens, p.positions = positions, p.slots = slots, p.free_left = free_left;
    p.B = B, p.T = max_tokens, p.max_pages = max_pages, p.page_shift = shift_of(page_size), p.num_pages = num_pages;
    p.free_size = free_size;
    EZB_CUDA_TRY(launch_paged_plan(p, stream));
    return EZB_OK;
}

int ezb_paged_qk_norm_rope(const void* qkv, long long ldqkv, const void* qw_or_null, const void* kw_or_null, const void* cos,
                           const void* sin, const int* positions, const int* slots, void* K_pool, void* V_pool, void* q_out, int T,
                           int H, int NKV, int D, int table_rows, int axes, const int* sections_host, int interleaved, int page_size,
                           int num_pages, float eps, ezb_stream_t stream) {
    EZB_REQUIRE(qkv && cos && sin && positions && slots && K_pool && V_pool && q_out && sections_host, "null pointer");
    EZB_REQUIRE(T >= 1 && H >= 1 && NKV >= 1 && table_rows >= 1 && num_pages >= 1, "sizes must be positive");
    EZB_REQUIRE_SHAPE(D == 64 || D == 128, "head_dim must be 64 or 128");
    EZB_REQUIRE_SHAPE(H % NKV == 0, "num_heads must be divisible by num_kv_heads");
    EZB_REQUIRE_SHAPE(shift_of(page_size) >= 0, "page_size must be a power of two >= 64");
    EZB_REQUIRE_SHAPE((long long)num_pages * page_size <= kMost, "num_pages * page_size is limited to 2^30");
    EZB_REQUIRE_SHAPE((long long)T * ((H + 2 * NKV + 1) / 2) < (1ll << 33), "too many tokens times heads");
    const long long width = ((long long)H + 2ll * NKV) * D;
    EZB_REQUIRE(ldqkv >= width && ldqkv % 8 == 0, "rows of qkv must be at least (H + 2 NKV) * D elements apart, a multiple of 8");
    EZB_REQUIRE(aligned16(qkv) && aligned16(qw_or_null) && aligned16(kw_or_null) && aligned16(cos) && aligned16(sin) && aligned16(K_pool) &&
                    aligned16(V_pool) && aligned16(q_out),
                "pointers must be 16-byte aligned");
    EZB_REQUIRE_SHAPE(axes >= 1 && axes <= 3, "one to three position axes");
    const int half = D / 2;
    long long sum = 0;
    for (int a = 0; a < axes; ++a) {
        EZB_REQUIRE_SHAPE(sections_host[a] >= 0 && sections_host[a] <= half, "a section must lie between 0 and head_dim / 2");
        sum += sections_host[a];
        if (interleaved && a > 0)
            EZB_REQUIRE_SHAPE(sections_host[a] == 0 || a + axes * (sections_host[a] - 1) < half,
                              "interleaved sections do not fit: axis a takes the frequencies a, a + axes, ...");
    }
    EZB_REQUIRE_SHAPE(sum == half, "the sections must add up to head_dim / 2");
    const long long pool = (long long)num_pages * NKV * page_size * D * 2, table = (long long)table_rows * D * 2;
    const Rect writes[] = {{q_out, T, (long long)H * D * 2, (long long)H * D * 2}, span(K_pool, pool), span(V_pool, pool)};
    const Rect reads[] = {{qkv, T, ldqkv * 2, width * 2}, span(qw_or_null, D * 2), span(kw_or_null, D * 2), span(cos, table), span(sin, table),
                          span(positions, 4ll * axes * T), span(slots, 4ll * T)};
    EZB_REQUIRE(!any_overlap(writes, reads), "q_out, K_pool and V_pool must not overlap each other or an input");
    unsigned char axis[64];
    for (int i = 0, a = 0, left = sections_host[0]; i < half; ++i) {
        if (interleaved) {
            const int c = i % axes;
            axis[i] = (unsigned char)(c > 0 && i / axes < sections_host[c] ? c : 0);
        } else {
            while (left == 0) left = sections_host[++a];
            axis[i] = (unsigned char)a, --left;
        }
    }
    PagedRopeArgs p;
    p.qkv = static_cast<const bf16*>(qkv), p.ld = ldqkv;
    p.qw = static_cast<const bf16*>(qw_or_null), p.kw = static_cast<const bf16*>(kw_or_null);
    p.cos = static_cast<const bf16*>(cos), p.sin = static_cast<const bf16*>(sin);
    p.positions = positions, p.slots = slots;
    p.K = static_cast<bf16*>(K_pool), p.V = static_cast<bf16*>(V_pool), p.q_out = static_cast<bf16*>(q_out);
    p.T = T, p.H = H, p.NKV = NKV, p.D = D, p.S = table_rows, p.axes = axes, p.page_shift = shift_of(page_size), p.num_pages = num_pages;
    p.axis_of_frequency = axis;
    p.eps = eps;
    EZB_CUDA_TRY(launch_paged_qk_norm_rope(p, stream));
    return EZB_OK;
}

int ezb_linear_bf16(const void* X, long long ldx, const void* W, const void* bias_or_null, const void* residual_or_null,
                    long long ldres, void* out, long long ldout, int M, int N, int K, int activation, int out_f32, ezb_stream_t stream) {
    EZB_REQUIRE(X && W && out, "null pointer");
    EZB_REQUIRE(M >= 1 && N >= 1 && K >= 1, "M, N and K must be positive");
    EZB_REQUIRE(activation >= EZB_ACT_NONE && activation <= EZB_ACT_SWIGLU, "unknown activation");
    EZB_REQUIRE_SHAPE(K % 8 == 0, "K must be divisible by 8");
    EZB_REQUIRE_SHAPE(M <= kMost && N <= kMost && K <= kMost && ((long long)M + 255) / 256 * (((long long)N + 31) / 32) < kMost,
                      "sizes are limited to 2^30, and so are the tiles of the result");
    EZB_REQUIRE(ldx >= K && ldx % 8 == 0, "rows of X must be at least K elements apart, a multiple of 8");
    EZB_REQUIRE(ldout >= N, "rows of out must be at least N elements apart");
    EZB_REQUIRE(!residual_or_null || ldres >= N, "rows of residual must be at least N elements apart");
    EZB_REQUIRE(aligned16(X) && aligned16(W), "X and W must be 16-byte aligned");
    const int size = out_f32 ? 4 : 2;
    EZB_REQUIRE(reinterpret_cast<uintptr_t>(out) % size == 0 && reinterpret_cast<uintptr_t>(residual_or_null) % 2 == 0 &&
                    reinterpret_cast<uintptr_t>(bias_or_null) % 2 == 0,
                "out, residual and bias must be aligned to their elements");
    const long long w_rows = activation == EZB_ACT_SWIGLU ? 2ll * N : N;
    const Rect o = {out, M, ldout * size, (long long)N * size};
    EZB_REQUIRE(!overlap(o, {X, M, ldx * 2, (long long)K * 2}), "out overlaps X");
    EZB_REQUIRE(!overlap(o, {W, w_rows, (long long)K * 2, (long long)K * 2}), "out overlaps W");
    EZB_REQUIRE(!bias_or_null || !overlap(o, {bias_or_null, 1, w_rows * 2, w_rows * 2}), "out overlaps bias");
    const bool in_place = residual_or_null == out && ldres == ldout && !out_f32;  // every element is read by the thread that writes it
    EZB_REQUIRE(!residual_or_null || in_place || !overlap(o, {residual_or_null, M, ldres * 2, (long long)N * 2}),
                "out overlaps residual (it may be the same bf16 tensor, not another view of it)");
    LinearArgs a;
    a.x = static_cast<const bf16*>(X), a.W = static_cast<const bf16*>(W), a.bias = static_cast<const bf16*>(bias_or_null);
    a.residual = static_cast<const bf16*>(residual_or_null), a.out = out;
    a.ldx = ldx, a.ldres = ldres, a.ldout = ldout;
    a.M = M, a.N = N, a.K = K, a.act = activation, a.out_f32 = out_f32 ? 1 : 0;
    EZB_CUDA_TRY(launch_linear(a, stream));
    return EZB_OK;
}

size_t ezb_attn_prompt_workspace_bytes(int D) { return D == 64 || D == 128 ? attn_prompt_workspace_bytes(D) : 0; }

int ezb_attn_prompt(const void* Q, long long ldq, const void* K_pool, const void* V_pool, const int* page_table, const int* seq_lens,
                    const int* cu_tokens, void* Out, long long ldo, void* workspace, size_t workspace_bytes, int B, int T, int H, int NKV,
                    int D, int max_pages, int page_size, int num_pages, ezb_stream_t stream) {
    EZB_REQUIRE(Q && K_pool && V_pool && page_table && seq_lens && cu_tokens && Out, "null pointer");
    EZB_REQUIRE(B >= 1 && T >= 1 && H >= 1 && NKV >= 1 && max_pages >= 1 && num_pages >= 1, "sizes must be positive");
    EZB_REQUIRE_SHAPE(D == 64 || D == 128, "head_dim must be 64 or 128");
    EZB_REQUIRE_SHAPE(H % NKV == 0, "num_heads must be divisible by num_kv_heads");
    EZB_REQUIRE_SHAPE(H / NKV <= 128, "at most 128 query heads per kv head");
    EZB_REQUIRE_SHAPE(shift_of(page_size) >= 0, "page_size must be a power of two >= 64");
    EZB_REQUIRE_SHAPE(T <= kMost && (long long)max_pages * page_size <= kMost && (long long)num_pages * NKV <= kMost,
                      "tokens, max_pages * page_size and num_pages * num_kv_heads are limited to 2^30");
    const long long width = (long long)H * D;
    EZB_REQUIRE(ldq >= width && ldq % 8 == 0 && ldo >= width && ldo % 8 == 0, "rows of Q and Out must be at least H * D elements apart, a multiple of 8");
    EZB_REQUIRE(aligned16(Q) && aligned16(K_pool) && aligned16(V_pool) && aligned16(Out), "Q, Out and the page pools must be 16-byte aligned");
    if (!workspace || !aligned16(workspace) || workspace_bytes < attn_prompt_workspace_bytes(D)) {
        set_last_message("workspace missing, misaligned or smaller than ezb_attn_prompt_workspace_bytes()");
        return EZB_ERR_WORKSPACE;
    }
    const long long pool = (long long)num_pages * NKV * page_size * D * 2;
    const Rect writes[] = {{Out, T, ldo * 2, width * 2}, span(workspace, (long long)attn_prompt_workspace_bytes(D))};
    const Rect reads[] = {{Q, T, ldq * 2, width * 2}, span(K_pool, pool), span(V_pool, pool), span(page_table, 4ll * B * max_pages),
                          span(seq_lens, 4ll * B), span(cu_tokens, 4ll * (B + 1))};
    EZB_REQUIRE(!any_overlap(writes, reads), "Out or the workspace overlaps an input, or each other");
    AttnPromptArgs a;
    a.Q = static_cast<const bf16*>(Q), a.K = static_cast<const bf16*>(K_pool), a.V = static_cast<const bf16*>(V_pool);
    a.Out = static_cast<bf16*>(Out), a.ldq = ldq, a.ldo = ldo;
    a.page_table = page_table, a.seq_lens = seq_lens, a.cu_tokens = cu_tokens;
    a.workspace = workspace;
    a.B = B, a.T = T, a.H = H, a.NKV = NKV, a.D = D, a.max_pages = max_pages, a.page_shift = shift_of(page_size), a.num_pages = num_pages;
    EZB_CUDA_TRY(launch_attn_prompt(a, stream));
    return EZB_OK;
}

unsigned long long ezb_stream_capture_id(ezb_stream_t stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    return status == cudaStreamCaptureStatusActive ? id : 0;
}

int ezb_paged_plan_packed(const long long* words) { return call_packed(ezb_paged_plan, words); }
int ezb_paged_qk_norm_rope_packed(const long long* words) { return call_packed(ezb_paged_qk_norm_rope, words); }
int ezb_linear_bf16_packed(const long long* words) { return call_packed(ezb_linear_bf16, words); }
int ezb_attn_prompt_packed(const long long* words) { return call_packed(ezb_attn_prompt, words); }

}  // extern "C"
