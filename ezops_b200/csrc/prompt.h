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
// x / (1 + e^-x) and x (1 - erfc(x / sqrt 2) / 2) from two MUFU results each.  Relative error, in units of 2^-23: at most |x| + 4
// and 3/4 x^2 + 17, the first terms from the rounding of the exponent (an exponent e has an error of up to |e| 2^-23, and the result
// that times ln 2).  So they are exact to a few units near zero and above it, and lose bits where a negative x makes them vanish (below -87 and
// -13 they are 0).  A result is rounded to bf16, or is as uncertain from its own sum, whose absolute error does not vanish there.  (With the division and erfcf a product of 5772 x 14592 results took
// 512 and 429 us instead of 201 without an activation.)
__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float silu_fast(float x) { return x * rcp_ftz(1.0f + ex2_ftz(x * -1.4426950408889634f)); }
__device__ __forceinline__ float gelu_fast(float x) {
    // erfc(y) = e^(-y^2) t P(t), t = 1 / (1 + 0.45 y), y >= 0: P of degree 7 with least maximum relative error (3.9e-7), found by
    // reweighted least squares
    const float t = rcp_ftz(fmaf(fabsf(x), 0.45f * 0.70710678118654752f, 1.0f));
    float s = 0.06947775930166245f;
    s = fmaf(s, t, -0.251302570104599f);
    s = fmaf(s, t, 0.22809070348739624f);
    s = fmaf(s, t, 0.0223945751786232f);
    s = fmaf(s, t, 0.19817346334457397f);
    s = fmaf(s, t, 0.225192591547966f);
    s = fmaf(s, t, 0.25409403443336487f);
    s = fmaf(s, t, 0.2538797855377197f);
    const float half = 0.5f * t * s * ex2_ftz(x * x * -0.72134752044448170f);  // erfc(|x| / sqrt 2) / 2
    return x * (x < 0.f ? half : 1.0f - half);
}
template <int W>
__device__ __forceinline__ void linear_act(float (&v)[W], int act) {  // all but SwiGLU
    if (act == ACT_SILU) {
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = silu_fast(v[e]);
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = gelu_fast(v[e]);
    } else if (act == ACT_RELU) {
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];  // NaN stays
    }
}
struct LinearArgs {
    const bf16 *x, *W, *bias, *residual;
    void* out;
    long long ldx, ldres, ldout;
    int M, N, K, act, out_f32;
};
cudaError_t launch_linear(const LinearArgs& a, cudaStream_t stream);
static constexpr int kLinearGroupRows = 64;
cudaError_t launch_linear_groups(const LinearArgs& a, cudaStream_t stream);  // groups of at most so many rows (gemm_tc.cu)

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
