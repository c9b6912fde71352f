// Launch interfaces of the kernels behind the prompt operators.  Sizes and alignments are checked by the C entries.
#pragma once
#include "launchers.h"

namespace ezb {

// Two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

struct PlanArgs {
    const int *ctx_lens, *new_lens, *free_pages, *free_count;
    int *page_table, *seq_lens, *cu_tokens, *positions, *slots, *free_left;
    int B, T, max_pages, page_shift, num_pages, free_size;
};
cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t stream);
static constexpr int kPlanMaxRows = 8192;  // running sums of all rows live in shared memory

struct PagedRopeArgs {
    const bf16* qkv;  // [T, ld]: q heads | k heads | v heads
    long long ld;
    const bf16 *qw, *kw, *cos, *sin;  // norm weights null = unit
    const int *positions, *slots;     // [axes, T], [T]
    bf16 *K, *V, *q_out;
    int T, H, NKV, D, S, axes, page_shift, num_pages;
    const unsigned char* axis_of_frequency;  // [D / 2], host
    float eps;
};
cudaError_t launch_paged_qk_norm_rope(const PagedRopeArgs& a, cudaStream_t stream);

// out[M, N] = act(x[M, K] W^T + bias) + residual; SwiGLU: W [2N, K], bias [2N], gate rows first
enum LinearAct { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_RELU = 3, ACT_SWIGLU = 4 };
__device__ __forceinline__ float linear_act(float x, int act) {  // all but SwiGLU
    if (act == ACT_SILU) return silu_f32(x);
    if (act == ACT_GELU) return 0.5f * x * erfcf(x * -0.70710678118654752f);  // 1 + erf(y) = erfc(-y), without cancellation
    if (act == ACT_RELU) return x < 0.f ? 0.f : x;  // NaN stays
    return x;
}
struct LinearArgs {
    const bf16 *x, *W, *bias, *residual;
    void* out;
    long long ldx, ldres, ldout;
    int M, N, K, act, out_f32;
};
cudaError_t launch_linear(const LinearArgs& a, cudaStream_t stream);
static constexpr int kLinearFewRows = 64;
cudaError_t launch_linear_few(const LinearArgs& a, cudaStream_t stream);  // at most kLinearFewRows rows (gemm_tc.cu)

struct AttnPromptArgs {
    const bf16 *Q, *K, *V;
    bf16* Out;
    long long ldq, ldo;
    const int *page_table, *seq_lens, *cu_tokens;
    void* workspace;
    int B, T, H, NKV, D, max_pages, page_shift, num_pages;
};
size_t attn_prompt_workspace_bytes(int D);
cudaError_t launch_attn_prompt(const AttnPromptArgs& a, cudaStream_t stream);

}  // namespace ezb
