// paged_attention.cuh - shared by the two kernels of PAGED_ATTENTION: the one
// for few query rows (paged_attention.cu) and the tensor-memory one for many
// (paged_prefill.cu).
#pragma once

#include "paged_common.cuh"

namespace vnpu_b200 {

// The kernel for many rows: takes a shape or answers cudaErrorNotSupported.
cudaError_t paged_attention_many_rows(const LaunchCtx &ctx, const PagedAttention &a);

namespace {

// What the attention kernels share: scaled weights (paged_attention.cu has the
// mathematics) and the parameters.
constexpr float kSlack = 6.0f;       // growth of the maximum before a rescale (log2)
constexpr float kLift = 8.0f;        // weights are scaled by 2^8: small ones stay normal numbers
// A page of zeros (V scale 0, or below kLeastScale: values below 2^-89) counts in the sum l alone,
// with the weight 2^(s - m + 8) of its score.  For the maximum m it stands in with a scale of
// 2^kZeroLog: m is then the others' wherever they are seen in the output (2^-8 below, a weight still
// has its 22 bits), and l stays below 2^102 a key.
constexpr float kLeastScale = 0x1p-96f;
constexpr float kZeroLog = -88.0f;

// 1 / l of a row: 0 where it saw nothing, NaN where it is NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

struct AttnParams {
    PagedCache c;
    PagedBatch pb;
    const void *Q;
    void *O;
    uint32_t ldq, ldo, group;
    uint32_t group_inverse;   // floor(2^32 / group); 0 for a group of one
    uint32_t causal, window;
    float scale_log2;
    uint32_t vec;          // bit 0: Q 16-byte accesses, bit 1: O 4-element, bit 2: O 16-byte accesses
    float *ws_o;           // [2 * grid][tile rows][DP] partial sums
    float2 *ws_ml;         // [2 * grid][tile rows] their m and l
    uint4 *ws_meta;        // [2 * grid]: who joins what
    float *ws_run;         // many f32 rows: [grid][DP][tile rows] sums of a run's earlier key tiles
    uint32_t *err;
    uint64_t limit_ns;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / x within a unit in the last place.
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A part's factor where the maximum of all is `all`: one that saw no key holds zeros (or the NaN of its
// query), taken as they are.
__device__ __forceinline__ float row_factor(float m, float all) { return m == -INFINITY ? 1.0f : ex2(m - all); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// The power of two that brings a row's largest element to [2^13, 2^14), as an
// exponent; rows of zeros, and of infinities, stay as they are.
__device__ __forceinline__ int row_exponent(float most) {
    const int ex = static_cast<int>((__float_as_uint(most) >> 23) & 255u) - 127;
    return most > 0.0f && most <= 3.402823466e38f ? max(-114, min(100, 13 - ex)) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }

// Row of a sequence's (token, head of the group) rows to its token: the product
// with the rounded-down inverse is the quotient or one less.
__device__ __forceinline__ uint32_t token_of(const AttnParams &p, uint32_t r) {
    if (p.group == 1) return r;
    const uint32_t q = __umulhi(r, p.group_inverse);
    return r - q * p.group >= p.group ? q + 1 : q;
}
inline uint32_t inverse_of(uint32_t group) {
    return group == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / group);
}

// Positions that row r (clamped to the sequence's last) of a sequence sees.
__device__ __forceinline__ void row_limits(const AttnParams &p, const PagedSeq &s, uint32_t r,
                                           int32_t &kmin, int32_t &kmax) {
    const uint32_t rows = static_cast<uint32_t>(s.n) * p.group;
    const int32_t pos = s.start + static_cast<int32_t>(token_of(p, min(r, rows - 1)));
    kmax = p.causal ? pos : s.len - 1;
    kmin = p.window && static_cast<uint32_t>(pos) + 1u > p.window ? pos + 1 - static_cast<int32_t>(p.window) : 0;
}

}  // namespace
}  // namespace vnpu_b200
