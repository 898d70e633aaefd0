// paged_common.cuh - what the kernels of the paged 8-bit key/value cache
// share: the rows of a batch, page addresses with their bounds, and 8- and
// 16-element row accesses in f32, f16 or bf16.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace vnpu_b200 {
namespace {

template <RowType T>
struct RowOf;
template <>
struct RowOf<RowType::kF32> {
    using type = float;
};
template <>
struct RowOf<RowType::kF16> {
    using type = __half;
};
template <>
struct RowOf<RowType::kBF16> {
    using type = __nv_bfloat16;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float x, float &y) { y = x; }
__device__ __forceinline__ void from_f32(float x, __half &y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }

// 8 consecutive elements; vec: their address is 16-byte aligned.
template <typename E>
__device__ __forceinline__ void load8(const E *p, bool vec, float (&v)[8]) {
    if (vec) {
        alignas(16) E e[8];
#pragma unroll
        for (uint32_t i = 0; i < sizeof(e) / 16; ++i)
            reinterpret_cast<uint4 *>(e)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = to_f32(p[i]);
    }
}
// 8 words to a 32-byte place, a whole sector in one store: sectors that are
// written in halves by two stores cost their way to L2 twice (read-back of 512
// tokens of 32 heads of 128 in f32: 14.0 us in 16-byte stores, 8.4 in these; of
// 19 000 tokens of 8 heads of 64 in f16: 14.9 and 11.7; append of f32 rows 4 to
// 6 % less).
__device__ __forceinline__ void store_sector(void *p, const uint32_t *r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// N consecutive elements to a place that `align` bytes divide: 32, 16, or less.
template <uint32_t N, typename E>
__device__ __forceinline__ void store_n(E *p, uint32_t align, const float (&v)[N]) {
    alignas(32) E e[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) from_f32(v[i], e[i]);
    if (sizeof(e) % 32 == 0 && align == 32) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(e) / 32; ++i)
            store_sector(reinterpret_cast<char *>(p) + 32 * i, reinterpret_cast<const uint32_t *>(e) + 8 * i);
    } else if (align >= 16) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(e) / 16; ++i)
            reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(e)[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) p[i] = e[i];
    }
}
// The largest power of two up to 32 that divides all of these.
inline uint32_t common_align(uint64_t places) {
    return places % 32u == 0 ? 32u : places % 16u == 0 ? 16u : 1u;
}

// One sequence's rows: rows row0 .. row0+n-1 at positions start .. len-1.
struct PagedSeq {
    int32_t row0 = 0, n = 0, start = 0, len = 0;
};

// Sequence b of the batch.  False, with nothing to do, when its numbers do not
// describe rows of the batch at positions the table reaches (the caller
// records kErrBadIndex).
__device__ __forceinline__ bool load_seq(const PagedBatch &pb, uint32_t page_shift, uint32_t b,
                                         PagedSeq &s) {
    const int32_t c0 = __ldg(pb.cu + b), c1 = __ldg(pb.cu + b + 1);
    s.len = __ldg(pb.lens + b);
    s.row0 = c0;
    s.n = c1 - c0;
    s.start = s.len - s.n;
    // c1 >= c0 >= 0 comes first: the differences above are then exact
    return c0 >= 0 && c1 >= c0 && static_cast<uint32_t>(c1) <= pb.tokens &&
           static_cast<uint32_t>(s.n) <= pb.max_tokens && s.len >= s.n &&
           s.len <= 0x7fffff00 &&   // key tiles' ends stay in 32 bits
           static_cast<uint64_t>(s.len) <= (static_cast<uint64_t>(pb.table_stride) << page_shift);
}

// The b for which the rising `base` first passes w, i.e. the number of
// sequences with base(b + 1) <= w (batch when w is past the last).  One pass
// over cu by the whole block, all threads get it; cu need not be monotone for
// the result to be in [0, batch].
template <uint32_t NT, typename F>
__device__ __forceinline__ uint32_t find_seq(uint32_t batch, const F &base_after, uint64_t w) {
    uint32_t found = 0;
    for (uint32_t b0 = 0; b0 < batch; b0 += NT) {
        const uint32_t b = b0 + threadIdx.x;
        found += __syncthreads_count(b < batch && base_after(b) <= w);
    }
    return found;
}

// 16-bit floats of 4 int8 codes (one 32-bit word): 0x6400 | (code + 128) is
// the half 1024 + 128 + code, and 1152 is taken off exactly.
__device__ __forceinline__ void codes_to_half4(uint32_t w, uint32_t &h01, uint32_t &h23) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    h01 = *reinterpret_cast<uint32_t *>(&x);
    h23 = *reinterpret_cast<uint32_t *>(&y);
}

}  // namespace
}  // namespace vnpu_b200
