// paged_kv.cu - the paged 8-bit key/value cache: append with rotation
// (VNPU_B200_OP_PAGED_KV_APPEND) and read-back (VNPU_B200_OP_PAGED_KV_READ).
//
// Both are bound by memory: each row element is read once and each code
// written once.  Work is split by segments: the part of one sequence's rows
// that falls into one page.  A CTA owns one (segment, head, K or V), so it
// alone sees all values that enter the page's scale: no atomics, and one
// result whatever the order.  Segments of ragged sequences need no prefix sum:
// a run of n rows touches at most floor(n / page_size) + 2 pages, so sequence
// b's segments can start at floor(cu[b] / page_size) + 2 b, which any CTA can
// search for; the numbers left over are CTAs that leave at once.
//
// Measured, bf16, 32/8 heads of 128 where not said: append of 6300 tokens in 16
// prompts 50 us (142 MB, 2.8 TB/s; issue slots and latency, not memory), of 64
// single tokens 5.5 us (three dependent loads); read-back, pass after pass, of
// 19 000 tokens of 8 heads of 64 in f16 11.7 us of one cache and 14.3 of three in
// turn (58 MB, 5.0 and 4.1 TB/s), of 512 tokens of 32 heads in f32 8.4 and 9.6 us
// (21 MB; one wave of CTAs and its latency).
#include <algorithm>

#include "paged_common.cuh"

namespace vnpu_b200 {
namespace {

// Tables are read 8 entries a lane, from places 8 apart: one entry of room after
// each 8 keeps lanes off each other's banks.
__host__ __device__ constexpr uint32_t pad8(uint32_t j) { return j + j / 8u; }

struct PagedTurns {
    uint64_t t[128];
};

// A page's part of a sequence's rows.
struct Segment {
    int32_t row0, n;    // rows
    int32_t slot0;      // slot of row0
    int32_t pos0;       // position of row0
    int64_t page;
};

// The sequence of a rising numbering: the first b with base_after(b) > w, by the
// whole block, with its numbers.  While batch <= NT the lookup and the numbers
// are one trip to memory.  False: none, or one with bad numbers (reported).
template <uint32_t NT, typename F>
__device__ __forceinline__ bool find_numbers(const PagedCache &c, const PagedBatch &pb, const F &base_after,
                                             uint64_t w, uint32_t *err, uint32_t &b, PagedSeq &s) {
    __shared__ PagedSeq sh_seq;
    __shared__ bool sh_good;
    bool good = false;
    if (pb.batch <= NT) {
        const uint32_t t = threadIdx.x;
        uint64_t base = ~0ull;
        if (t < pb.batch) {
            good = load_seq(pb, c.page_shift, t, s);
            base = base_after(t);
        }
        b = __syncthreads_count(base <= w);
        if (t == b) {
            sh_seq = s;
            sh_good = good;
        }
        __syncthreads();
        if (b >= pb.batch) return false;
        s = sh_seq;
        good = sh_good;
    } else {
        b = find_seq<NT>(pb.batch, base_after, w);
        if (b >= pb.batch) return false;
        good = load_seq(pb, c.page_shift, b, s);
    }
    if (!good && (threadIdx.x & 31u) == 0) record_error(err, kErrBadIndex);
    return good;
}

// Segment number `item` of the batch; false: no such segment, or a bad one.
// Its page is as the table gives it: page_there() looks at it.
template <uint32_t NT>
__device__ __forceinline__ bool find_segment(const PagedCache &c, const PagedBatch &pb,
                                             uint32_t item, uint32_t *err, Segment &g) {
    uint32_t b, seg = 0;
    PagedSeq s;
    if (pb.max_tokens == 1) {
        b = item;  // one segment a sequence: item b is sequence b's
        if (!load_seq(pb, c.page_shift, b, s)) {
            if ((threadIdx.x & 31u) == 0) record_error(err, kErrBadIndex);
            return false;
        }
    } else {
        const auto after = [&](uint32_t i) -> uint64_t {
            const int32_t cu = __ldg(pb.cu + i + 1);
            return (static_cast<uint64_t>(cu < 0 ? 0 : cu) >> c.page_shift) + 2ull * (i + 1);
        };
        if (!find_numbers<NT>(c, pb, after, item, err, b, s)) return false;
        const uint64_t base = (static_cast<uint64_t>(s.row0) >> c.page_shift) + 2ull * b;
        if (item < base) return false;  // only where cu falls
        seg = static_cast<uint32_t>(item - base);
    }
    if (s.n == 0) return false;
    const uint64_t index = (static_cast<uint32_t>(s.start) >> c.page_shift) + static_cast<uint64_t>(seg);
    const int64_t p0 = static_cast<int64_t>(index << c.page_shift);
    if (p0 >= s.len) return false;
    const int64_t lo = max(static_cast<int64_t>(s.start), p0);
    const int64_t hi = min(static_cast<int64_t>(s.len), p0 + (static_cast<int64_t>(1) << c.page_shift));
    g.page = __ldg(pb.table + static_cast<uint64_t>(b) * pb.table_stride + index);
    g.row0 = s.row0 + static_cast<int32_t>(lo - s.start);
    g.n = static_cast<int32_t>(hi - lo);
    g.slot0 = static_cast<int32_t>(lo - p0);
    g.pos0 = static_cast<int32_t>(lo);
    return true;
}
__device__ __forceinline__ bool page_there(const PagedCache &c, const Segment &g, uint32_t *err) {
    const bool there = g.page >= 0 && g.page < c.num_pages;
    if (!there && (threadIdx.x & 31u) == 0) record_error(err, kErrBadIndex);
    return there;
}

inline uint64_t segment_items(const PagedCache &c, const PagedBatch &b) {
    return b.max_tokens == 1 ? b.batch : (static_cast<uint64_t>(b.tokens) >> c.page_shift) + 2ull * b.batch;
}

// `pos` times t 2^-64 turns, in 2^-32 turns.  The product is taken modulo one
// turn (the 64-bit wrap): off by 2^-32 of a turn at every position, where a
// 32-bit position * frequency is off by 2^-24 of the whole angle, 1e-2 at
// position 1e5.
__device__ __forceinline__ uint32_t turn_fraction(int32_t pos, uint64_t t) {
    const uint32_t p = static_cast<uint32_t>(pos);
    return p * static_cast<uint32_t>(t >> 32) + __umulhi(p, static_cast<uint32_t>(t));
}
// Queries' angles, shared by their heads: the library's sine and cosine.
__device__ __forceinline__ void turn_sincos(int32_t pos, uint64_t t, float *sn, float *cs) {
    sincospif(static_cast<float>(static_cast<int32_t>(turn_fraction(pos, t))) * 0x1p-31f, sn, cs);
}
// Keys' angles, one for each pair and head: the nearest quarter turn is taken off
// in whole numbers, what is left is x in [-pi/4, pi/4], off by 2^-24 of itself,
// and the Taylor series of sine and cosine to x^9 and x^10 are within 2e-9 there.
// Sine and cosine are off by 2^-23.3 at most.  (The library's sincospif for each pair
// and head cost 60 % more time; its fast sine and cosine, 2^-21 off, flipped codes and
// took 58.0 us where these take 60.5: 16 prompts, 8600 tokens of 32/8 heads of 128.)
__device__ __forceinline__ void turn_sincos_series(int32_t pos, uint64_t t, float *sn, float *cs) {
    const uint32_t turn = turn_fraction(pos, t), quarter = (turn + (1u << 29)) >> 30;
    const float x = static_cast<float>(static_cast<int32_t>(turn - (quarter << 30))) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float y = x * x;
    const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float u = quarter & 1u ? c : s, v = quarter & 1u ? s : c;
    *sn = __uint_as_float(__float_as_uint(u) ^ (quarter & 2u) << 30);
    *cs = __uint_as_float(__float_as_uint(v) ^ ((quarter + 1u) & 2u) << 30);
}

// A head's 16 elements of unit u as two groups of 8 and their pairs' first
// index: for the half-split rotation the groups are 8u.. and rotary/2 + 8u..,
// else 16u.. and 16u + 8...  pair < 0: not rotated.
struct Unit {
    uint32_t o0, o1;
    int32_t pair;
};
__device__ __forceinline__ Unit unit_of(uint32_t u, uint32_t rotary, bool interleaved) {
    Unit x;
    const bool turned = u * 16u < rotary;
    x.o0 = turned && !interleaved ? 8u * u : 16u * u;
    x.o1 = turned && !interleaved ? rotary / 2u + 8u * u : 16u * u + 8u;
    x.pair = turned ? static_cast<int32_t>(8u * u) : -1;
    return x;
}

// Rotates a unit; cs(i, sn, cs) gives the sine and cosine of pair x.pair + i.
template <typename F>
__device__ __forceinline__ void rotate_unit(float (&a)[8], float (&b)[8], bool interleaved,
                                            const F &angle) {
    if (!interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float sn, cs;
            angle(i, &sn, &cs);
            const float x = a[i], y = b[i];
            a[i] = x * cs - y * sn;
            b[i] = x * sn + y * cs;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float sn, cs;
            angle(i, &sn, &cs);
            float x = a[2 * i], y = a[2 * i + 1];
            a[2 * i] = x * cs - y * sn;
            a[2 * i + 1] = x * sn + y * cs;
            angle(i + 4, &sn, &cs);
            x = b[2 * i];
            y = b[2 * i + 1];
            b[2 * i] = x * cs - y * sn;
            b[2 * i + 1] = x * sn + y * cs;
        }
    }
}

// What codes are made with: 1 / scale, the scale, half of it (infinite for a page
// of zeros), and 2^-24 of it.
struct Rounding {
    float inv, scale, half, unit;
};
// The code of x is the nearest whole number, ties to even, of the 32-bit quotient
// x / scale.  That is the nearest of x * inv, in the low bits of x * inv + 1.5 *
// 2^23, unless *rest, what x has more than that many scales, exactly, is within
// 2^-15 scales of half a scale: the product is off by 2^-24 of at most 127 and the
// quotient by half as much.
__device__ __forceinline__ uint32_t rounded(float x, const Rounding &by, float *rest) {
    const float z = __fmaf_rn(x, by.inv, 12582912.0f);
    *rest = __fmaf_rn(12582912.0f - z, by.scale, x);
    return __float_as_uint(z);
}
// There the quotient is a tie where it is half a unit in the last place from one
// at most (2^-24 of its power of two), and else on the side that the rest says.
// Ties are common: 16-bit x are one in a thousand times.
__device__ __forceinline__ uint32_t settled(float x, uint32_t z, float rest, const Rounding &by) {
    const float over = fabsf(rest) - by.half;
    const uint32_t power = max(__float_as_uint(fabsf(x * by.inv)) & 0x7f800000u, 0x3f000000u);   // of quotients from 1/2
    const bool tie = fabsf(over) <= __uint_as_float(power) * by.unit;
    return (tie ? (z & 1u) != 0 : over > 0.0f) ? z + (rest > 0.0f ? 1u : ~0u) : z;
}
// Codes of 8 values.
__device__ __forceinline__ uint2 codes8_finite(const float (&v)[8], const Rounding &by) {
    uint32_t q[8];
    float rest[8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = rounded(v[i], by, &rest[i]);
        most = fmaxf(most, fabsf(rest[i]));
    }
    if (most >= by.half * (1.0f - 0x1p-14f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = settled(v[i], q[i], rest[i], by);
    }
    const auto pack = [&](int i) {
        return __byte_perm(__byte_perm(q[i], q[i + 1], 0x0040), __byte_perm(q[i + 2], q[i + 3], 0x0040), 0x5410);
    };
    return make_uint2(pack(0), pack(4));
}
// The same with NaN 0 and infinities the largest code.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], const Rounding &by) {
    uint2 r = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float rest;
        const uint32_t z = rounded(v[i], by, &rest);
        uint32_t q = settled(v[i], z, rest, by);
        if (!(fabsf(v[i]) <= 3.402823466e38f)) q = v[i] > 0.0f ? 127u : v[i] < 0.0f ? 129u : 0u;
        (i < 4 ? r.x : r.y) |= (q & 0xffu) << (8 * (i & 3));
    }
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Older codes on a larger scale, whose part `ratio` theirs is.
__device__ __forceinline__ uint32_t rescaled4(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= (static_cast<uint32_t>(__float2int_rn(static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * ratio)) & 0xffu)
             << (8 * i);
    return r;
}

constexpr uint32_t kQueryRows(uint32_t nt) { return nt == 128 ? 1 : 4; }  // query rows of a CTA

// Grid: segments x heads x {K, V}, then the query rows.  A segment of one head
// is a CTA's work, or, where every sequence has one token, a warp's (kWarp).  A
// thread holds up to U units (16 elements each) of its segment in registers
// between the maximum and the rounding; a segment with more is read again,
// from L2.
template <RowType T, uint32_t NT, uint32_t U, bool kWarp>
__global__ void __launch_bounds__(NT, kWarp ? 6 : U == 2 ? 3 : 2) paged_append_kernel(
    const PagedCache c, const PagedBatch pb, const void *Qv, const void *Kv, const void *Vv,
    void *Qov, uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldqo, uint32_t q_heads,
    uint32_t rotary, bool interleaved, uint32_t vec, uint32_t q_align, uint32_t kv_ctas, uint32_t kv_items,
    const PagedTurns turns, uint32_t *err) {
    using E = typename RowOf<T>::type;
    constexpr uint32_t GT = kWarp ? 32 : NT;         // threads of a segment
    __shared__ float2 sh_turn[kQueryRows(NT)][pad8(128)];
    __shared__ uint64_t sh_rate[pad8(128)];          // turns: lanes read different ones
    __shared__ uint32_t sh_max[NT / 32];
    const uint32_t tid = threadIdx.x, D = c.head_dim, lane = kWarp ? tid & 31u : tid;
    if (tid < rotary / 2u) sh_rate[pad8(tid)] = turns.t[tid];
    pdl_enter();

    if (blockIdx.x >= kv_ctas) {
        // ---- queries: rotate rows r0 .. r0 + kQueryRows - 1, angles shared by the heads
        const uint32_t r0 = (blockIdx.x - kv_ctas) * kQueryRows(NT);
        int32_t pos[kQueryRows(NT)];
        PagedSeq s;                 // of the row before, mostly this one's too
        s.n = 0;
#pragma unroll
        for (uint32_t i = 0; i < kQueryRows(NT); ++i) {   // block-uniform
            const int32_t r = static_cast<int32_t>(r0 + i);
            pos[i] = -1;
            if (r0 + i >= pb.tokens) continue;
            bool good = s.n != 0 && r < s.row0 + s.n;
            if (!good && kWarp) {   // row b is sequence b's when every sequence has one
                good = r0 + i < pb.batch && load_seq(pb, c.page_shift, r0 + i, s) && s.row0 == r && s.n == 1;
            }
            if (!good) {
                uint32_t b;
                const auto after = [&](uint32_t j) -> uint64_t {
                    const int32_t cu = __ldg(pb.cu + j + 1);
                    return cu < 0 ? 0u : static_cast<uint64_t>(cu);
                };
                good = find_numbers<NT>(c, pb, after, r0 + i, err, b, s);
                if (!good || r < s.row0 || r >= s.row0 + s.n) {   // a row of no sequence, or of a bad one
                    s.n = 0;
                    continue;
                }
            }
            pos[i] = s.start + r - s.row0;
        }
        __syncthreads();
        const uint32_t pairs = rotary / 2u;
#pragma unroll
        for (uint32_t i = 0; i < kQueryRows(NT); ++i)
            for (uint32_t j = tid; j < pairs; j += NT)
                turn_sincos(pos[i], sh_rate[pad8(j)], &sh_turn[i][pad8(j)].y, &sh_turn[i][pad8(j)].x);
        __syncthreads();
        const uint32_t per_row = q_heads * (D / 16u);
        const bool vin = vec & 1u;
        for (uint32_t k = tid; k < per_row; k += NT) {
            const uint32_t h = k / (D / 16u);
            const Unit x = unit_of(k - h * (D / 16u), rotary, interleaved);
            constexpr uint32_t F = kQueryRows(NT) < 2 ? 1 : 2;    // rows in flight
#pragma unroll
            for (uint32_t i0 = 0; i0 < kQueryRows(NT); i0 += F) {
                float a[F][8], b[F][8];
#pragma unroll
                for (uint32_t i = 0; i < F; ++i) {
                    if (pos[i0 + i] < 0) continue;
                    const E *in = static_cast<const E *>(Qv) + static_cast<uint64_t>(r0 + i0 + i) * ldq + h * D;
                    load8(in + x.o0, vin, a[i]);
                    load8(in + x.o1, vin, b[i]);
                }
#pragma unroll
                for (uint32_t i = 0; i < F; ++i) {
                    if (pos[i0 + i] < 0) continue;
                    E *out = static_cast<E *>(Qov) + static_cast<uint64_t>(r0 + i0 + i) * ldqo + h * D;
                    if (x.pair >= 0)
                        rotate_unit(a[i], b[i], interleaved, [&](int e, float *sn, float *cs) {
                            const float2 t = sh_turn[i0 + i][pad8(x.pair) + e];
                            *cs = t.x;
                            *sn = t.y;
                        });
                    store_n(out + x.o0, q_align, a[i]);
                    store_n(out + x.o1, q_align, b[i]);
                }
            }
        }
        return;
    }

    if constexpr (kWarp) __syncthreads();
    const uint32_t index = kWarp ? blockIdx.x * (NT / 32u) + (tid >> 5) : blockIdx.x;
    if (index >= kv_items) return;
    const uint32_t item = index / (2u * c.heads);
    const uint32_t which = index - item * 2u * c.heads;
    const bool value = which >= c.heads;
    const uint32_t h = value ? which - c.heads : which;
    Segment g;
    if (!find_segment<NT>(c, pb, item, err, g)) return;
    if constexpr (!kWarp) __syncthreads();           // sh_rate
    const uint32_t ld = value ? ldv : ldk;
    const bool vin = vec & (value ? 4u : 2u);
    const E *in = static_cast<const E *>(value ? Vv : Kv) + static_cast<uint64_t>(g.row0) * ld + h * D;
    const uint32_t rot = value ? 0u : rotary;
    // This thread's units: row and place in the row, GT units on from one to the next.
    const uint32_t per_row = D / 16u, rows = static_cast<uint32_t>(g.n);
    struct Place {
        uint32_t r, u;
    };
    Place p0;
    p0.r = lane / per_row;
    p0.u = lane - p0.r * per_row;
    const uint32_t dr = GT / per_row, du = GT - dr * per_row;
    const auto next = [&](Place x) {
        x.r += dr;
        x.u += du;
        if (x.u >= per_row) {
            x.u -= per_row;
            ++x.r;
        }
        return x;
    };
    const auto fetch = [&](const Place &at, float (&a)[8], float (&b)[8]) {
        const Unit x = unit_of(at.u, rot, interleaved);
        const E *row = in + static_cast<uint64_t>(at.r) * ld;
        load8(row + x.o0, vin, a);
        load8(row + x.o1, vin, b);
    };
    const auto turn = [&](const Place &at, float (&a)[8], float (&b)[8]) {
        const Unit x = unit_of(at.u, rot, interleaved);
        if (x.pair >= 0)
            rotate_unit(a, b, interleaved, [&](int e, float *sn, float *cs) {
                turn_sincos_series(g.pos0 + static_cast<int32_t>(at.r), sh_rate[pad8(x.pair) + e], sn, cs);
            });
    };
    float most = 0.0f;
    const auto widen = [&](const float (&a)[8], const float (&b)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max_nan(most, max_nan(fabsf(a[i]), fabsf(b[i])));
    };
    Place at[U];
    float a[U][8], b[U][8];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {  // all loads in flight before the first is used
        at[u] = u ? next(at[u - 1]) : p0;
        if (at[u].r < rows) fetch(at[u], a[u], b[u]);
    }
    if (!page_there(c, g, err)) return;
    const uint64_t head = static_cast<uint64_t>(g.page) * c.heads + h;
    int8_t *page = (value ? c.V : c.K) + ((head << c.page_shift) * D);
    float *scale = (value ? c.V_scale : c.K_scale) + head;
    const float held = g.slot0 ? *scale : 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
        if (at[u].r < rows) {
            turn(at[u], a[u], b[u]);
            widen(a[u], b[u]);
        }
    const Place rest = next(at[U - 1]);
    for (Place k = rest; k.r < rows; k = next(k)) {
        float x[8], y[8];
        fetch(k, x, y);
        turn(k, x, y);
        widen(x, y);
    }
    // the bits of |x| rise with it, infinity and NaN last
    uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
    if constexpr (!kWarp) {
        if ((tid & 31u) == 0) sh_max[tid >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < NT / 32u; ++i) bits = max(bits, sh_max[i]);
    }
    const bool finite = bits < 0x7f800000u;
    if (!finite) {   // once more, without what is not finite
        if constexpr (!kWarp) __syncthreads();
        most = 0.0f;
        for (Place k = p0; k.r < rows; k = next(k)) {
            float x[8], y[8];
            fetch(k, x, y);
            turn(k, x, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (fabsf(x[i]) <= 3.402823466e38f) most = fmaxf(most, fabsf(x[i]));
                if (fabsf(y[i]) <= 3.402823466e38f) most = fmaxf(most, fabsf(y[i]));
            }
        }
        bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if constexpr (!kWarp) {
            if ((tid & 31u) == 0) sh_max[tid >> 5] = bits;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < NT / 32u; ++i) bits = max(bits, sh_max[i]);
        }
    }

    // A scale below the smallest normal number has no finite reciprocal: such a page is zero.
    const float larger = fmaxf(held, __fdiv_rn(__uint_as_float(bits), 127.0f));
    const float now = larger < 1.17549435e-38f ? 0.0f : larger;
    const Rounding by = {now > 0.0f ? __fdiv_rn(1.0f, now) : 0.0f, now, now > 0.0f ? 0.5f * now : INFINITY,
                         now * 0x1p-24f};
    if (lane == 0) *scale = now;
    const auto put = [&](const Place &k, const float (&a)[8], const float (&b)[8]) {
        const Unit x = unit_of(k.u, rot, interleaved);
        int8_t *row = page + static_cast<uint32_t>(g.slot0 + k.r) * D;
        *reinterpret_cast<uint2 *>(row + x.o0) = finite ? codes8_finite(a, by) : codes8(a, by);
        *reinterpret_cast<uint2 *>(row + x.o1) = finite ? codes8_finite(b, by) : codes8(b, by);
    };
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
        if (at[u].r < rows) put(at[u], a[u], b[u]);
    for (Place k = rest; k.r < rows; k = next(k)) {
        float x[8], y[8];
        fetch(k, x, y);
        turn(k, x, y);
        put(k, x, y);
    }
    if (g.slot0 && now > held) {  // the scale grew: round the page's older codes to it
        const float ratio = __fdiv_rn(held, now);
        uint4 *old = reinterpret_cast<uint4 *>(page);
        for (uint32_t k = lane; k < static_cast<uint32_t>(g.slot0) * per_row; k += GT) {
            uint4 w = old[k];
            w.x = rescaled4(w.x, ratio);
            w.y = rescaled4(w.y, ratio);
            w.z = rescaled4(w.z, ratio);
            w.w = rescaled4(w.w, ratio);
            old[k] = w;
        }
    }
}

// A CTA reads one segment of `span` heads, of K or of V; a thread has 4 units
// in flight.
template <RowType T, uint32_t NT>
__global__ void __launch_bounds__(NT, 10) paged_read_kernel(
    const PagedCache c, const PagedBatch pb, void *first, void *second, uint64_t ld_row,
    uint64_t ld_head, uint32_t span, uint32_t spans, uint32_t align, bool swap, uint32_t *err) {
    using E = typename RowOf<T>::type;
    pdl_enter();
    const uint32_t item = blockIdx.x / spans, h0 = (blockIdx.x - item * spans) * span;
    Segment g;
    if (!find_segment<NT>(c, pb, item, err, g) || !page_there(c, g, err)) return;
    const bool value = (blockIdx.y != 0) != swap;
    E *const out0 = static_cast<E *>(blockIdx.y ? second : first);
    const int8_t *const pool = value ? c.V : c.K;
    const float *const scales = value ? c.V_scale : c.K_scale;
    const uint32_t D = c.head_dim, per_row = D / 16u, per_head = g.n * per_row;
    const uint32_t units = min(span, c.heads - h0) * per_head;
    const uint64_t at0 = static_cast<uint64_t>(g.page) * c.heads + h0;
    const auto put = [&](const uint4 &w, float s, E *out) {
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
        float v[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t x, y;          // by way of exact 16-bit floats
            codes_to_half4(word[i], x, y);
            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&x));
            const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&y));
            v[4 * i] = lo.x * s;
            v[4 * i + 1] = lo.y * s;
            v[4 * i + 2] = hi.x * s;
            v[4 * i + 3] = hi.y * s;
        }
        store_n(out, align, v);
    };
    constexpr uint32_t B = 4;
    for (uint32_t k0 = threadIdx.x; k0 < units; k0 += B * NT) {
        uint4 w[B];
        float sc[B];
        E *out[B];
#pragma unroll
        for (uint32_t i = 0; i < B; ++i) {
            const uint32_t k = k0 + i * NT;
            if (k >= units) continue;
            const uint32_t h = k / per_head, in_head = k - h * per_head, r = in_head / per_row;
            const uint64_t at = at0 + h;
            w[i] = __ldg(reinterpret_cast<const uint4 *>(
                pool + ((at << c.page_shift) + static_cast<uint32_t>(g.slot0)) * D + in_head * 16u));
            sc[i] = __ldg(scales + at);
            out[i] = out0 + (g.row0 + static_cast<uint64_t>(r)) * ld_row + (h0 + h) * ld_head + (in_head - r * per_row) * 16u;
        }
#pragma unroll
        for (uint32_t i = 0; i < B; ++i)
            if (k0 + i * NT < units) put(w[i], sc[i], out[i]);
    }
}

template <typename F>
cudaError_t by_type(RowType t, const F &f) {
    switch (t) {
    case RowType::kF32: return f(std::integral_constant<RowType, RowType::kF32>{});
    case RowType::kF16: return f(std::integral_constant<RowType, RowType::kF16>{});
    default: return f(std::integral_constant<RowType, RowType::kBF16>{});
    }
}

bool aligned16(const void *p, uint64_t stride_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16u == 0 && stride_bytes % 16u == 0;
}

}  // namespace

cudaError_t paged_kv_append(const LaunchCtx &ctx, const PagedAppend &p) {
    const uint32_t elem = p.type == RowType::kF32 ? 4 : 2;
    const uint32_t vec = (aligned16(p.Q, 1ull * p.ldq * elem) ? 1u : 0u) |
                         (aligned16(p.K, 1ull * p.ldk * elem) ? 2u : 0u) |
                         (aligned16(p.V, 1ull * p.ldv * elem) ? 4u : 0u);
    const uint32_t q_align = common_align(reinterpret_cast<uintptr_t>(p.Q_out) | 1ull * p.ldqo * elem);
    PagedTurns turns{};
    for (uint32_t j = 0; j < p.rotary / 2; ++j) turns.t[j] = p.turns[j];
    const uint64_t items = segment_items(p.cache, p.batch) * 2 * p.cache.heads;
    // One token a sequence: a segment is one row, a warp's work (64 sequences of 32/8 heads of 128:
    // 13.1 us as a CTA's, 6.4 as a warp's).
    const bool single = p.batch.max_tokens == 1;
    const uint32_t nt = single ? 128 : 256, rows = kQueryRows(nt);
    const uint64_t kv = single ? (items + 3) / 4 : items;
    const uint64_t grid = kv + (p.Q ? (p.batch.tokens + rows - 1) / rows : 0);
    if (items > 0x7fffffffull || grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    // Units a thread holds: a page's worth, at most 4 (64 registers).
    const uint64_t units = (static_cast<uint64_t>(p.cache.head_dim) << p.cache.page_shift) / 16 / 256;
    if (ctx.launch_counter) ++*ctx.launch_counter;
    return by_type(p.type, [&](auto t) -> cudaError_t {
        constexpr RowType T = decltype(t)::value;
        auto kernel = single ? &paged_append_kernel<T, 128, 1, true>
                      : units <= 2 ? &paged_append_kernel<T, 256, 2, false>
                                   : &paged_append_kernel<T, 256, 4, false>;
        return launch_pdl(ctx.stream, kernel, dim3(static_cast<uint32_t>(grid)), dim3(nt), 0, p.cache,
                          p.batch, p.Q, p.K, p.V, p.Q_out, p.ldq, p.ldk, p.ldv, p.ldqo, p.q_heads,
                          p.rotary, p.interleaved, vec, q_align, static_cast<uint32_t>(kv),
                          static_cast<uint32_t>(items), turns, ctx.err);
    });
}

cudaError_t paged_kv_read(const LaunchCtx &ctx, const PagedRead &p) {
    const uint32_t elem = p.type == RowType::kF32 ? 4 : 2;
    const uint32_t align = common_align(reinterpret_cast<uintptr_t>(p.K_out) | reinterpret_cast<uintptr_t>(p.V_out) |
                                        p.ld_row * elem | p.ld_head * elem);
    // Heads of a CTA: enough for 4 units a thread, where pages are small.
    const uint32_t in_head = (p.cache.head_dim << p.cache.page_shift) / 16u;
    const uint32_t span = std::max(1u, std::min(p.cache.heads, 512u / in_head));
    const uint32_t spans = (p.cache.heads + span - 1) / span;
    const uint64_t grid = segment_items(p.cache, p.batch) * spans;
    if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    if (ctx.launch_counter) ++*ctx.launch_counter;
    return by_type(p.type, [&](auto t) -> cudaError_t {
        constexpr RowType T = decltype(t)::value;
        // K, then V; or the one of them that is wanted
        void *const first = p.K_out ? p.K_out : p.V_out;
        return launch_pdl(ctx.stream, &paged_read_kernel<T, 128>,
                          dim3(static_cast<uint32_t>(grid), p.K_out && p.V_out ? 2 : 1), dim3(128), 0, p.cache,
                          p.batch, first, p.V_out, p.ld_row, p.ld_head, span, spans, align, p.K_out == nullptr,
                          ctx.err);
    });
}

}  // namespace vnpu_b200
