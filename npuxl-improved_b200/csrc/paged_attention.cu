// paged_attention.cu - attention over the paged 8-bit key/value cache
// (VNPU_B200_OP_PAGED_ATTENTION): the kernel for few query rows, which is
// right for every shape, and the dispatch.
//
// The mathematics.  Scores are s_j = (q . c_j) * K_scale * scale with the int8
// codes c_j.  A value scale is folded into the softmax weight: with
//   t_j = s_j log2(e) + log2(V_scale of j),  m >= max t_j - 6,
//   p_j = 2^(t_j - m + 8),  l = sum p_j / V_scale of j,  o = sum p_j code_j / l,
// which is sum softmax(s)_j V_scale_j code_j: one addition a key and one
// product a page instead of a product a value, and every p_j fits a 16-bit
// float whatever the scales.  Codes are whole numbers below 128, exact in 16
// bits, so both products run on f16 tensor instructions with nothing lost on
// the cache's side.  A query row is scaled by a power of two to a largest
// element in [2^13, 2^14): f16 and bf16 queries are then exact too (down to
// 2^-27 of the row's largest), and f32 ones become hi + lo, 22 bits, two
// products on one accumulator; their weights p are split the same way.  Sums,
// maxima and accumulators are f32.
//
// The tensor core's sums are not rounded to nearest.  Over the steps of a long
// run that is a drift, at 131072 keys a CTA 5e-5 of the output: f32 rows take O
// from it 16 keys at a time and add in f32 (6 to 11 % of their time, 71.0 us to
// 76.8 at 32768 keys of 32 heads).  For 16-bit rows it stays below their rounding.
//
// m follows the running maximum only when that has grown by more than 2^6, so
// the accumulators are rescaled a few times a row instead of at every step.
//
// Measured, bf16, 32/8 heads of 128: one token each for 2 sequences of 131072
// keys 95 us (537 MB, 5.65 TB/s, 86 % of the copy bandwidth) and 6 us of
// joining; for 64 sequences of up to 4096 keys 68 us with joining (304 MB, 4.5
// TB/s: the starts and ends of rows beside the stream).
#include <algorithm>

#include "paged_attention.cuh"

namespace vnpu_b200 {
namespace {

constexpr uint32_t kWarps = 4, kThreadsA = kWarps * 32;
constexpr uint32_t kTile = 128;      // keys of a work unit, 32 for each warp
constexpr uint32_t kWarpKeys = kTile / kWarps;
// Reach of a table up to which row tiles are not split.  One token, 16 sequences of 32/8 heads of 128,
// us without and with splitting and joining: 256 keys 9.2 and 9.6, 384 keys 11.5 and 9.9; 64 sequences
// of 8 heads of 64: 12.4 and 13.3, 15.6 and 14.8.  (The lengths are the device's: the reach is what
// the host knows of them.)
constexpr uint32_t kWholeKeys = 256;

// As many CTAs an SM as the registers allow (the kernel is bound by the latency
// of its own instructions before it is by memory), rings as deep as that allows.
template <uint32_t DP, uint32_t MR>
struct AttnShape {
    static constexpr uint32_t kCtasPerSm = DP == 256 ? 1 : MR == 8 ? 3 : 2;
    static constexpr uint32_t kSlot = kWarpKeys * DP * 2;   // a warp's K and V codes of a unit
    static constexpr uint32_t kStages = (DP == 256 ? 200u : 208u / kCtasPerSm) * 1024 / (kWarps * kSlot);
    static constexpr uint32_t kSmem = kWarps * kStages * kSlot;
    static_assert(kStages >= 2 && kSlot >= 16 * DP * 4, "a slot also takes a warp's accumulators");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held as a product's fragment.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// The units (sequence, head, row tile, key tile) in that order, the last
// fastest: where a CTA stands in them.
struct Cursor {
    uint32_t b, h, rt;      // sequence, key/value head, row tile
    int32_t tile;           // key tile, lo <= tile < lo + nt
    int32_t lo, nt;
    uint32_t rts;           // row tiles of the sequence
    PagedSeq s;
};

// Row tiles and key tiles of a sequence; 0 row tiles when it has no rows (or
// bad numbers, which *bad reports).  An empty range of keys counts one tile, in
// which everything is masked, so that its rows are written.
template <uint32_t MR>
__device__ __forceinline__ void seq_units(const AttnParams &p, uint32_t b, Cursor &k, bool *bad) {
    k.b = b;
    k.rts = 0;
    k.lo = 0;
    k.nt = 1;
    const bool ok = load_seq(p.pb, p.c.page_shift, b, k.s);
    *bad = !ok;
    if (!ok || k.s.n == 0) return;
    k.rts = (static_cast<uint32_t>(k.s.n) * p.group + MR - 1) / MR;
    if (p.window && static_cast<uint32_t>(k.s.start) + 1u > p.window)
        k.lo = (k.s.start + 1 - static_cast<int32_t>(p.window)) / static_cast<int32_t>(kTile);
    const int32_t hi = (k.s.len + static_cast<int32_t>(kTile) - 1) / static_cast<int32_t>(kTile);
    k.nt = max(1, hi - k.lo);
}

// The next unit; true where it belongs to another row tile.  Loads the next
// sequence that has rows where one ends (the caller stops before the last
// unit's successor is asked for).
template <uint32_t MR>
__device__ __forceinline__ bool next_unit(const AttnParams &p, Cursor &k) {
    if (++k.tile < k.lo + k.nt) return false;
    if (++k.rt == k.rts) {
        k.rt = 0;
        if (++k.h == p.c.heads) {
            k.h = 0;
            bool bad;
            uint32_t b = k.b;
            do {
                if (++b >= p.pb.batch) break;
                seq_units<MR>(p, b, k, &bad);
            } while (k.rts == 0);
        }
    }
    k.tile = k.lo;
    return true;
}

// Persistent CTAs, each with an equal run of units (or, with `whole`, of row
// tiles, which are then not split and need no joining): sequences of any lengths
// give every CTA the same work, and a (sequence, head, row tile) is split over
// CTAs only where runs meet.  A warp keeps kStages - 1 units in flight through
// its own ring of cp.async copies (no CTA-wide waits within a run), across
// the ends of sequences too.
//
// The products are transposed: S^T = K Q^T and O^T += V^T P^T, so that the 16-row
// side of the tensor instruction is keys, then head_dim, and the query rows are
// its 8 columns.  For the few rows of a decode step that is half the products
// and half the accumulators of S = Q K^T.  P^T's fragment is S^T's transposed
// 8 x 8 by 8 x 8, one instruction each.  MR, the query rows of a tile, is 8, or
// 16 (two column tiles under one conversion of the codes) where a sequence has
// more.
template <RowType T, uint32_t DP, uint32_t MR>
__global__ void __launch_bounds__(kThreadsA, AttnShape<DP, MR>::kCtasPerSm)
    paged_attention_kernel(const __grid_constant__ AttnParams p, const bool whole) {
    using E = typename RowOf<T>::type;
    using Shape = AttnShape<DP, MR>;
    constexpr bool kSplit = T == RowType::kF32;
    static_assert(MR == 8 || MR == 16, "rows of a tile");
    constexpr uint32_t NT = MR / 8;                // column tiles
    constexpr uint32_t S = Shape::kStages, NC = DP / 16, NG = DP / 64, NJ = DP / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sh_scale[kWarps][S][4];       // K_scale and V_scale of a unit's 16-key groups
    __shared__ float2 sh_ml[kWarps][16];
    __shared__ unsigned long long sh_sum[kWarps];
    __shared__ Cursor sh_cursor;
    __shared__ unsigned long long sh_off;
    pdl_enter();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, n = lane >> 2, kq = lane & 3u;
    const uint32_t D = p.c.head_dim, cta = blockIdx.x;

    // ---- this CTA's run of units
    const uint32_t per_thread = (p.pb.batch + kThreadsA - 1) / kThreadsA;
    const uint32_t b_lo = min(tid * per_thread, p.pb.batch), b_hi = min(b_lo + per_thread, p.pb.batch);
    unsigned long long mine = 0;
    Cursor cur;
    for (uint32_t b = b_lo; b < b_hi; ++b) {
        bool bad;
        seq_units<MR>(p, b, cur, &bad);
        if (bad) record_error(p.err, kErrBadIndex);
        mine += static_cast<unsigned long long>(cur.rts) * p.c.heads * (whole ? 1 : cur.nt);
    }
    unsigned long long upto = mine;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sh_sum[warp] = upto;
    __syncthreads();
    unsigned long long total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) upto += sh_sum[w];
        total += sh_sum[w];
    }
    const unsigned long long run = max(1ull, (total + gridDim.x - 1) / gridDim.x);
    const unsigned long long t0 = run * cta;
    const bool countable = run <= 0xffffffffu;   // a run's units are counted in 32 bits; more are an hour's work
    if (t0 >= total || !countable) {
        if (tid == 0 && !countable) record_error(p.err, kErrBadIndex);
        if (tid == 0 && p.ws_meta) p.ws_meta[2 * cta].x = 0;
        return;
    }
    uint32_t left = static_cast<uint32_t>(min(run, total - t0));  // units (row tiles) of this CTA
    unsigned long long before = upto - mine;
    if (before <= t0 && t0 < upto) {
        for (uint32_t b = b_lo; b < b_hi; ++b) {
            bool bad;
            seq_units<MR>(p, b, cur, &bad);
            const unsigned long long w = static_cast<unsigned long long>(cur.rts) * p.c.heads * (whole ? 1 : cur.nt);
            if (t0 < before + w) {
                sh_cursor = cur;
                sh_off = t0 - before;
                break;
            }
            before += w;
        }
    }
    __syncthreads();
    {
        cur = sh_cursor;
        const unsigned long long off = sh_off;
        const unsigned long long nt = whole ? 1u : static_cast<uint32_t>(cur.nt), row_tile = off / nt;
        cur.h = static_cast<uint32_t>(row_tile / cur.rts);
        cur.rt = static_cast<uint32_t>(row_tile - static_cast<unsigned long long>(cur.h) * cur.rts);
        cur.tile = cur.lo + static_cast<int32_t>(off - row_tile * nt);
    }
    Cursor ahead = cur;         // the unit to copy next
    uint32_t ahead_left = left;
    uint32_t slot_in = 0;

    uint8_t *const ring = smem + warp * (S * Shape::kSlot);

    // Pages of the two 16-key groups of `ahead`'s part of this warp.
    int32_t page_next[2];
    const auto fetch_pages = [&]() {
        if (ahead_left == 0) return;
        const int32_t k0 = ahead.tile * static_cast<int32_t>(kTile) + static_cast<int32_t>(warp * kWarpKeys);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int32_t key = k0 + 16 * i;
            page_next[i] = key < ahead.s.len
                               ? __ldg(p.pb.table + static_cast<uint64_t>(ahead.b) * p.pb.table_stride +
                                       (static_cast<uint32_t>(key) >> p.c.page_shift))
                               : -1;
        }
    };
    // What the row tile to copy for sees at most, and the place of this lane's 16 bytes.
    int32_t ahead_min = 0, ahead_max = 0;
    const auto ahead_limits = [&]() {
        int32_t unused;
        row_limits(p, ahead.s, ahead.rt * MR, ahead_min, unused);
        row_limits(p, ahead.s, ahead.rt * MR + MR - 1, unused, ahead_max);
    };
    // 16-byte pieces of a row of codes change places by this: the readers below take pieces kq
    // of two rows next to each other (K), and pieces m, m + 4 of every second row (V)
    const auto swizzle = [](uint32_t row) {
        return DP == 64 ? (row >> 1) & 3u : (row & 1u) << 2 | ((row >> 1) & 3u);
    };
    const uint32_t my_row = lane / NC, my_ch = lane % NC, lane_src = my_row * D + my_ch * 16u;
    const bool my_ch_there = my_ch * 16u < D;
    constexpr uint32_t kStep = 32 / NC;                          // rows of a warp's copy
    const auto place = [&](uint32_t q) {                         // of its row q * kStep + my_row
        const uint32_t row = q * kStep + my_row;
        return row * DP + (my_ch ^ swizzle(row)) * 16u;
    };
    const auto issue = [&]() {
        if (ahead_left) {
            const int32_t k0 = ahead.tile * static_cast<int32_t>(kTile) + static_cast<int32_t>(warp * kWarpKeys);
            uint8_t *const dst = ring + slot_in * Shape::kSlot;
            uint64_t base[2], scale_at[2];
            bool ok[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t key = k0 + 16 * i;
                // a group with nothing to see is left as it is
                const bool live = key < ahead.s.len && key <= ahead_max && key + 16 > ahead_min;
                ok[i] = live && page_next[i] >= 0 && static_cast<uint32_t>(page_next[i]) < p.c.num_pages;
                if (live && !ok[i] && lane == 0) record_error(p.err, kErrBadIndex);
                const uint64_t at = ok[i] ? static_cast<uint64_t>(page_next[i]) * p.c.heads + ahead.h : 0;
                base[i] = ((at << p.c.page_shift) + (static_cast<uint32_t>(key) & ((1u << p.c.page_shift) - 1u))) * D;
                scale_at[i] = at;
            }
            if (lane < 4)   // K's of the two groups, then V's
                cp_async_4_zfill(&sh_scale[warp][slot_in][lane],
                                 (lane < 2 ? p.c.K_scale : p.c.V_scale) + (lane & 1u ? scale_at[1] : scale_at[0]),
                                 lane & 1u ? ok[1] : ok[0]);
            constexpr uint32_t kCopies = kWarpKeys / kStep;      // of K, and of V
            if (ok[0] && ok[1] && k0 + static_cast<int32_t>(kWarpKeys) <= ahead.s.len) {
                const auto copy = [&](uint32_t row_bytes) {
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const int8_t *const ks = p.c.K + base[i] + lane_src, *const vs = p.c.V + base[i] + lane_src;
#pragma unroll
                        for (uint32_t q = 0; q < kCopies / 2; ++q) {
                            cp_async_16(dst + place(i * (kCopies / 2) + q), ks + q * kStep * row_bytes);
                            cp_async_16(dst + kWarpKeys * DP + place(i * (kCopies / 2) + q), vs + q * kStep * row_bytes);
                        }
                    }
                };
                if (D == DP) copy(DP);               // offsets known to the compiler
                else if (my_ch_there) copy(D);
            } else {
#pragma unroll 1
                for (uint32_t q = 0; q < kCopies; ++q) {         // a sequence's last keys
                    const uint32_t i = q / (kCopies / 2);
                    const bool in = (i ? ok[1] : ok[0]) && k0 + static_cast<int32_t>(q * kStep + my_row) < ahead.s.len;
                    const uint64_t src = in ? (i ? base[1] : base[0]) + lane_src + (q % (kCopies / 2)) * kStep * D : 0;
                    if (my_ch_there) {
                        cp_async_16_zfill(dst + place(q), p.c.K + src, in);
                        cp_async_16_zfill(dst + kWarpKeys * DP + place(q), p.c.V + src, in);
                    }
                }
            }
            if (!whole || ahead.tile + 1 == ahead.lo + ahead.nt) --ahead_left;
            if (ahead_left && next_unit<MR>(p, ahead)) ahead_limits();
        }
        cp_async_commit();
        slot_in = slot_in + 1 == S ? 0 : slot_in + 1;
    };
    ahead_limits();

    fetch_pages();
#pragma unroll
    for (uint32_t i = 0; i + 1 < S; ++i) {
        issue();
        fetch_pages();
    }

    // ---- state of the current (sequence, head, row tile)
    uint32_t bq[NT][NG][4][2];             // query fragments
    uint32_t bl[kSplit ? NT : 1][NG][4][2];  // f32: their low halves
    float acc[NT][NJ][4];
    float m[NT][2], l[NT][2], qf[NT][2];   // of rows 8 t + 2 kq and + 1: running maximum, sum, score factor
    int32_t kmin[NT][2], kmax[NT][2], kmin_last = 0, kmax_first = 0, kmin_first = 0, kmax_last = 0;
    int32_t first_tile = 0;
    // The queries of the next row tile, read while the one before is written.
    alignas(16) E next_q[NT][NG][16];
    const auto read_rows = [&](const Cursor &k) {
        const uint32_t rows = static_cast<uint32_t>(k.s.n) * p.group;
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t) {
            const uint32_t r = k.rt * MR + 8 * t + n;       // the row of this lane's fragment
            const uint32_t token = token_of(p, r);
            const E *q = static_cast<const E *>(p.Q) +
                         static_cast<uint64_t>(k.s.row0 + static_cast<int32_t>(token)) * p.ldq +
                         (k.h * p.group + (r - token * p.group)) * D;
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g) {
                const uint32_t d = 16u * (kq + 4u * g);
                uint4 *v = reinterpret_cast<uint4 *>(next_q[t][g]);
                constexpr uint32_t NW = sizeof(E);          // 16-byte pieces of 16 elements
#pragma unroll
                for (uint32_t i = 0; i < NW; ++i) v[i] = make_uint4(0, 0, 0, 0);
                if (r >= rows || d >= D) continue;
                if (p.vec & 1u) {
#pragma unroll
                    for (uint32_t i = 0; i < NW; ++i) v[i] = __ldg(reinterpret_cast<const uint4 *>(q + d) + i);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 16; ++e) next_q[t][g][e] = q[d + e];
                }
            }
        }
    };
    const auto begin_rows = [&]() {
        first_tile = cur.tile;
        row_limits(p, cur.s, cur.rt * MR, kmin_first, kmax_first);
        row_limits(p, cur.s, cur.rt * MR + MR - 1, kmin_last, kmax_last);
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t) {
            float v[NG][16];
            float most = 0.0f;
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    v[g][e] = to_f32(next_q[t][g][e]);
                    most = fmaxf(most, fabsf(v[g][e]));
                }
            most = quad_max(most);
            const int ex = row_exponent(most);
            const float up = pow2(ex);
#pragma unroll
            for (uint32_t g = 0; g < NG; ++g)
#pragma unroll
                for (uint32_t s = 0; s < 4; ++s)
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        const float x0 = v[g][4 * s + 2 * k] * up, x1 = v[g][4 * s + 2 * k + 1] * up;
                        bq[t][g][s][k] = pack_half2(x0, x1);
                        if constexpr (kSplit) {
                            const float2 y = unpack_half2(bq[t][g][s][k]);
                            bl[t][g][s][k] = pack_half2(x0 - y.x, x1 - y.y);
                        }
                    }
            const float factor = p.scale_log2 * pow2(-ex);
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
                qf[t][e] = __shfl_sync(0xffffffffu, factor, 8 * kq + 4 * e);
                row_limits(p, cur.s, cur.rt * MR + 8 * t + 2 * kq + e, kmin[t][e], kmax[t][e]);
                m[t][e] = -INFINITY;
                l[t][e] = 0.0f;
            }
#pragma unroll
            for (uint32_t j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][j][e] = 0.0f;
        }
    };

    const auto compute = [&](uint32_t slot) {
        const int32_t k0 = cur.tile * static_cast<int32_t>(kTile) + static_cast<int32_t>(warp * kWarpKeys);
        if (k0 > kmax_last || k0 + static_cast<int32_t>(kWarpKeys) <= kmin_first) return;  // warp-uniform
        const uint8_t *kb = ring + slot * Shape::kSlot, *vb = kb + kWarpKeys * DP;
        const float *sc = sh_scale[warp][slot];
        // scores of two groups of 16 keys: element e of a fragment is key n + 8 (e >> 1) of the
        // group and row 2 kq + (e & 1).  The head_dim index is permuted, the same way in K and Q:
        // a lane's 16 codes are the elements of four products
        float s[2][NT][4];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t) s[i][t][0] = s[i][t][1] = s[i][t][2] = s[i][t][3] = 0.0f;
#pragma unroll
        for (uint32_t g = 0; g < NG; ++g) {
            uint4 w[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t row = 8u * i + n;
                w[i] = *reinterpret_cast<const uint4 *>(kb + row * DP + ((kq + 4u * g) ^ swizzle(row)) * 16u);
            }
            const auto word = [&](uint32_t i, uint32_t e) { return e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w; };
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half4(word(2 * i, e), a0, a2);
                    codes_to_half4(word(2 * i + 1, e), a1, a3);
#pragma unroll
                    for (uint32_t t = 0; t < NT; ++t) {
                        mma_f16(s[i][t], a0, a1, a2, a3, bq[t][g][e][0], bq[t][g][e][1]);
                        if constexpr (kSplit) mma_f16(s[i][t], a0, a1, a2, a3, bl[t][g][e][0], bl[t][g][e][1]);
                    }
                }
        }
        float lv[2], iv[2];
        bool on[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float vs = sc[2 + i];
            on[i] = vs >= kLeastScale;         // else a page of zeros, or nothing that is seen
            lv[i] = on[i] ? __log2f(vs) : kZeroLog;
            iv[i] = on[i] ? reciprocal(vs) : 1.0f;   // not 2^-lv: what lv is off by then cancels in o / l
        }
        const bool edge = k0 + static_cast<int32_t>(kWarpKeys) - 1 > kmax_first || k0 < kmin_last;
        float top[NT][2];
        bool grown = false;
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) {
                top[t][r] = -INFINITY;
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const float f = qf[t][r] * sc[i];
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        float x = fmaf(s[i][t][2 * e + r], f, lv[i]);
                        if (edge) {
                            const int32_t key = k0 + static_cast<int32_t>(16 * i + 8 * e + n);
                            if (key > kmax[t][r] || key < kmin[t][r]) x = -INFINITY;
                        }
                        s[i][t][2 * e + r] = x;
                        top[t][r] = fmaxf(top[t][r], x);
                    }
                }
#pragma unroll
                for (uint32_t o = 4; o < 32; o <<= 1)
                    top[t][r] = fmaxf(top[t][r], __shfl_xor_sync(0xffffffffu, top[t][r], o));
                grown |= top[t][r] > m[t][r] + kSlack;
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t) {
                float f[2];
#pragma unroll
                for (uint32_t r = 0; r < 2; ++r) {
                    const float to = fmaxf(m[t][r], top[t][r]);
                    f[r] = to > m[t][r] ? ex2(m[t][r] - to) : 1.0f;
                    l[t][r] *= f[r];
                    m[t][r] = to;
                }
#pragma unroll
                for (uint32_t j = 0; j < NJ; ++j)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) acc[t][j][e] *= f[e & 1];
            }
        }
        if (!(on[0] && on[1])) {               // warp-uniform: those count as they are
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) s[i][t][e] -= on[i] ? 0.0f : kZeroLog;
        }
        uint32_t pb[2][NT][2], pl[2][kSplit ? NT : 1][2];
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t) {
            float off[2];
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) off[r] = m[t][r] == -INFINITY ? 0.0f : m[t][r] - kLift;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
                    const float x = ex2(s[i][t][2 * e] - off[0]), y = ex2(s[i][t][2 * e + 1] - off[1]);
                    l[t][0] = fmaf(x, iv[i], l[t][0]);
                    l[t][1] = fmaf(y, iv[i], l[t][1]);
                    const uint32_t h = on[i] ? pack_half2(x, y) : 0u;
                    pb[i][t][e] = transpose8x8(h);
                    if constexpr (kSplit) {
                        const float2 u = unpack_half2(h);
                        pl[i][t][e] = transpose8x8(on[i] ? pack_half2(x - u.x, y - u.y) : 0u);
                    }
                }
        }
        // values: a lane's keys 2 kq, 2 kq + 1, + 8, + 9 of a group, and the dims of lane group n
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            constexpr uint32_t NW = DP / 32;       // words of a row for a thread
            uint32_t w[4][NW];
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                const uint32_t row = 16u * i + 2u * kq + (q & 1u) + 8u * (q >> 1);
                if constexpr (DP == 64) {
                    const uint2 x = *reinterpret_cast<const uint2 *>(vb + row * DP + ((n >> 1) ^ swizzle(row)) * 16u + (n & 1u) * 8u);
                    w[q][0] = x.x;
                    w[q][1] = x.y;
                } else {
#pragma unroll
                    for (uint32_t g = 0; g < DP / 128; ++g) {
                        const uint32_t ch = 8u * g + (((n >> 1) + 4u * (n & 1u)) ^ swizzle(row));
                        const uint4 x = *reinterpret_cast<const uint4 *>(vb + row * DP + ch * 16u);
                        w[q][4 * g] = x.x;
                        w[q][4 * g + 1] = x.y;
                        w[q][4 * g + 2] = x.z;
                        w[q][4 * g + 3] = x.w;
                    }
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < NW; ++k)
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half4(__byte_perm(w[0][k], w[1][k], half ? 0x7362 : 0x5140), a0, a1);
                    codes_to_half4(__byte_perm(w[2][k], w[3][k], half ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                    for (uint32_t t = 0; t < NT; ++t) {
                        if constexpr (kSplit) {   // 16 keys at a time, added in f32
                            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(part, a0, a1, a2, a3, pl[i][t][0], pl[i][t][1]);
                            mma_f16(part, a0, a1, a2, a3, pb[i][t][0], pb[i][t][1]);
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) acc[t][2 * k + half][e] += part[e];
                        } else {
                            mma_f16(acc[t][2 * k + half], a0, a1, a2, a3, pb[i][t][0], pb[i][t][1]);
                        }
                    }
                }
        }
    };

    // The warps' sums of a row tile joined through their consumed slots, and
    // written: as the output when this CTA saw all its keys, else as a part.
    const auto end_rows = [&](uint32_t slot, bool more, const Cursor *after) {
        const uint32_t rows = min(MR, static_cast<uint32_t>(cur.s.n) * p.group - cur.rt * MR);
        float *const mine_o = reinterpret_cast<float *>(ring + slot * Shape::kSlot);
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) {
#pragma unroll
                for (uint32_t o = 4; o < 32; o <<= 1) l[t][r] += __shfl_xor_sync(0xffffffffu, l[t][r], o);
                if (n == 0) sh_ml[warp][8 * t + 2 * kq + r] = make_float2(m[t][r], l[t][r]);
            }
        __syncwarp();  // all lanes are done with the slot's codes
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) {
                const uint32_t row = 8 * t + 2 * kq + r;
                if (row >= rows) continue;
                // a lane's sums of a row are the DP / 8 dims of the codes that it read
#pragma unroll
                for (uint32_t j = 0; j < NJ; j += 2) {
                    uint32_t d;
                    if constexpr (DP == 64) d = 8u * n + 2u * j;
                    else d = 128u * (j / 8u) + 16u * ((n >> 1) + 4u * (n & 1u)) + 2u * (j % 8u);
                    reinterpret_cast<float4 *>(mine_o)[row * (DP / 4) + ((d / 4) ^ (row & 7u))] =
                        make_float4(acc[t][j][r], acc[t][j][2 + r], acc[t][j + 1][r], acc[t][j + 1][2 + r]);
                }
            }
        if (after) read_rows(*after);
        __syncthreads();
        const bool started = first_tile == cur.lo;
        const uint32_t part = 2 * cta + (started ? 1 : 0);
        for (uint32_t i = tid; i < rows * (DP / 4); i += kThreadsA) {
            const uint32_t row = i / (DP / 4), d4 = i % (DP / 4);
            if (4u * d4 >= D) continue;
            float2 ml[kWarps];
            float mm = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                ml[w] = sh_ml[w][row];
                mm = fmaxf(mm, ml[w].x);
            }
            float4 o = make_float4(0, 0, 0, 0);
            float ll = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float f = row_factor(ml[w].x, mm);
                ll = fmaf(ml[w].y, f, ll);
                const float4 x = reinterpret_cast<const float4 *>(
                    smem + (w * S + slot) * Shape::kSlot)[row * (DP / 4) + (d4 ^ (row & 7u))];
                o.x = fmaf(x.x, f, o.x);
                o.y = fmaf(x.y, f, o.y);
                o.z = fmaf(x.z, f, o.z);
                o.w = fmaf(x.w, f, o.w);
            }
            if (started && !more) {
                const uint32_t r = cur.rt * MR + row, token = token_of(p, r);
                const float inv = inverse_sum(ll);
                E *out = static_cast<E *>(p.O) +
                         static_cast<uint64_t>(cur.s.row0 + static_cast<int32_t>(token)) * p.ldo +
                         (cur.h * p.group + (r - token * p.group)) * D + 4u * d4;
                const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
                alignas(16) E e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) from_f32(v[k], e[k]);
                if (p.vec & 2u) {
                    if constexpr (sizeof(E) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(e);
                    else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<uint2 *>(e);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) out[k] = e[k];
                }
            } else {
                reinterpret_cast<float4 *>(p.ws_o)[(static_cast<uint64_t>(part) * MR + row) * (DP / 4) + d4] = o;
                if (d4 == 0) p.ws_ml[part * MR + row] = make_float2(mm, ll);
            }
        }
        __syncthreads();  // the slots may be filled again
    };

    read_rows(cur);
    uint32_t slot = 0;
    bool fresh = true;
    uint32_t parts = 0;
    for (;;) {
        cp_async_wait_group<S - 2>();
        __syncwarp();
        issue();  // into the slot that the last step consumed
        fetch_pages();
        if (fresh) begin_rows();
        compute(slot);
        const bool row_end = cur.tile + 1 == cur.lo + cur.nt;
        if (!whole || row_end) --left;
        Cursor after = cur;
        fresh = left && next_unit<MR>(p, after);
        if (fresh || !left) {
            if (!row_end && first_tile == cur.lo)   // the tile's first CTA joins its parts
                parts = 1 + static_cast<uint32_t>((cur.lo + cur.nt - cur.tile - 1 + run - 1) / run);
            end_rows(slot, !row_end, fresh ? &after : nullptr);
        } else {
            __syncwarp();
        }
        if (!left) break;
        cur = after;
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    cp_async_wait_group<0>();
    if (tid == 0 && p.ws_meta) {
        p.ws_meta[2 * cta] = make_uint4(parts, static_cast<uint32_t>(cur.s.row0), cur.rt * MR, cur.h);
        p.ws_meta[2 * cta + 1] = make_uint4(
            min(MR, static_cast<uint32_t>(cur.s.n) * p.group - cur.rt * MR), 0, 0, 0);
    }
}

// Joins a row tile's parts: block (c, y) those of the tile that begins in CTA
// c and goes on in the next ones, 32 groups of 4 values of it; 8 lanes share
// the parts, added in a fixed order.
template <RowType T, uint32_t DP, uint32_t MR>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const AttnParams p) {
    using E = typename RowOf<T>::type;
    __shared__ float4 sh_o[8][32];
    __shared__ float2 sh_ml[8][32];
    pdl_enter();
    const uint32_t cta = blockIdx.x;
    const uint4 meta = p.ws_meta[2 * cta];
    if (meta.x < 2) return;
    const uint32_t rows = p.ws_meta[2 * cta + 1].x;
    const uint32_t x = threadIdx.x & 31u, y = threadIdx.x >> 5;
    const uint32_t i = blockIdx.y * 32u + x;
    const uint32_t row = i / (DP / 4), d4 = i % (DP / 4);
    const bool live = row < rows && 4u * d4 < p.c.head_dim;
    float mm = -INFINITY, ll = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    if (live) {
#pragma unroll 4
        for (uint32_t k = y; k < meta.x; k += 8) {
            const uint64_t part = k == 0 ? 2ull * cta + 1 : 2ull * (cta + k);
            const float2 ml = p.ws_ml[part * MR + row];
            const float4 v = reinterpret_cast<const float4 *>(p.ws_o)[(part * MR + row) * (DP / 4) + d4];
            const float to = fmaxf(mm, ml.x);
            const float f = row_factor(mm, to), g = row_factor(ml.x, to);
            mm = to;
            ll = ll * f + ml.y * g;
            o.x = o.x * f + v.x * g;
            o.y = o.y * f + v.y * g;
            o.z = o.z * f + v.z * g;
            o.w = o.w * f + v.w * g;
        }
    }
    sh_o[y][x] = o;
    sh_ml[y][x] = make_float2(mm, ll);
    __syncthreads();
    if (y != 0 || !live) return;
    for (uint32_t k = 1; k < 8; ++k) mm = fmaxf(mm, sh_ml[k][x].x);
    ll = 0.0f;
    o = make_float4(0, 0, 0, 0);
    for (uint32_t k = 0; k < 8; ++k) {
        const float2 ml = sh_ml[k][x];
        const float f = row_factor(ml.x, mm);
        const float4 v = sh_o[k][x];
        ll += ml.y * f;
        o.x += v.x * f;
        o.y += v.y * f;
        o.z += v.z * f;
        o.w += v.w * f;
    }
    const float inv = inverse_sum(ll);
    const uint32_t r = meta.z + row, token = token_of(p, r);
    E *out = static_cast<E *>(p.O) + static_cast<uint64_t>(meta.y + token) * p.ldo +
             (meta.w * p.group + (r - token * p.group)) * p.c.head_dim + 4u * d4;
    from_f32(o.x * inv, out[0]);
    from_f32(o.y * inv, out[1]);
    from_f32(o.z * inv, out[2]);
    from_f32(o.w * inv, out[3]);
}

template <RowType T, uint32_t DP, uint32_t MR>
cudaError_t launch_attention(const LaunchCtx &ctx, const PagedAttention &a) {
    using Shape = AttnShape<DP, MR>;
    const uint32_t elem = T == RowType::kF32 ? 4 : 2;
    AttnParams p{};
    p.c = a.cache;
    p.pb = a.batch;
    p.Q = a.Q;
    p.O = a.O;
    p.ldq = a.ldq;
    p.ldo = a.ldo;
    p.group = a.q_heads / a.cache.heads;
    p.group_inverse = inverse_of(p.group);
    p.causal = a.causal;
    p.window = a.window;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.vec = (reinterpret_cast<uintptr_t>(a.Q) % 16u == 0 && 1ull * a.ldq * elem % 16u == 0 ? 1u : 0u) |
            (reinterpret_cast<uintptr_t>(a.O) % (4u * elem) == 0 && a.ldo % 4u == 0 ? 2u : 0u);
    p.err = ctx.err;
    static thread_local int ready_device = -1;
    int device = 0;
    VNPU_LAUNCH(cudaGetDevice(&device));
    if (ready_device != device) {
        VNPU_LAUNCH(cudaFuncSetAttribute(paged_attention_kernel<T, DP, MR>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem));
        ready_device = device;
    }
    const uint32_t grid = static_cast<uint32_t>(ctx.num_sms) * Shape::kCtasPerSm;
    // A table that reaches a few key tiles only: row tiles are not split, and nothing is joined.
    const bool split = (static_cast<uint64_t>(a.batch.table_stride) << a.cache.page_shift) > kWholeKeys;
    void *ws = nullptr;
    const size_t o_bytes = 2ull * grid * MR * DP * sizeof(float);
    const size_t ml_bytes = 2ull * grid * MR * sizeof(float2);
    if (split) {
        VNPU_LAUNCH(cudaMallocAsync(&ws, o_bytes + ml_bytes + 2ull * grid * sizeof(uint4), ctx.stream));
        p.ws_o = static_cast<float *>(ws);
        p.ws_ml = reinterpret_cast<float2 *>(static_cast<char *>(ws) + o_bytes);
        p.ws_meta = reinterpret_cast<uint4 *>(static_cast<char *>(ws) + o_bytes + ml_bytes);
    }
    if (ctx.launch_counter) *ctx.launch_counter += split ? 2 : 1;
    cudaError_t e = launch_pdl(ctx.stream, &paged_attention_kernel<T, DP, MR>, dim3(grid), dim3(kThreadsA),
                               Shape::kSmem, p, !split);
    if (split) {
        const uint64_t rows = std::min<uint64_t>(MR, 1ull * a.batch.max_tokens * p.group);
        const uint32_t y = static_cast<uint32_t>((rows * (DP / 4) + 31) / 32);
        if (e == cudaSuccess)
            e = launch_pdl(ctx.stream, &paged_attention_join_kernel<T, DP, MR>, dim3(grid, y), dim3(256), 0, p);
        const cudaError_t f = cudaFreeAsync(ws, ctx.stream);
        if (e == cudaSuccess) e = f;
    }
    return e;
}

template <RowType T, uint32_t MR>
cudaError_t launch_by_dim(const LaunchCtx &ctx, const PagedAttention &a) {
    if (a.cache.head_dim <= 64) return launch_attention<T, 64, MR>(ctx, a);
    if (a.cache.head_dim <= 128) return launch_attention<T, 128, MR>(ctx, a);
    return launch_attention<T, 256, 8>(ctx, a);   // 16 rows' accumulators do not fit the registers
}

template <RowType T>
cudaError_t launch_few(const LaunchCtx &ctx, const PagedAttention &a) {
    return 1ull * a.batch.max_tokens * (a.q_heads / a.cache.heads) > 8 ? launch_by_dim<T, 16>(ctx, a)
                                                                       : launch_by_dim<T, 8>(ctx, a);
}

}  // namespace

cudaError_t paged_attention(const LaunchCtx &ctx, const PagedAttention &a) {
    // Rows of a key/value head in one sequence (tokens x group): the few-row kernel's 16-row tiles read
    // and convert the codes again for each tile, the many-row kernel has a block's start and end.  In
    // us, few and many, 16 sequences of 2048 keys, 64 of 512, 4 of 8192, 8 key/value heads:
    //   16-bit, 64:  48 rows 49 and 51, 55 and 66, 46 and 48; 56 rows 60 and 51, 67 and 66, 58 and 48
    //   16-bit, 128: 48 rows 65 and 61, 78 and 85, 60 and 57; 56 rows 79 and 62, 92 and 86, 76 and 57
    //   f32, 64:     64 rows 69 and 75, 78 and 89, 66 and 71; a fifth tile is 14 more
    //   f32, 128:    32 rows 77 and 97, 90 and 121, 73 and 88; 40 rows 107 and 98, 131 and 121, 99 and 89
    const uint64_t few = a.type != RowType::kF32 ? 48 : a.cache.head_dim <= 64 ? 64 : 32;
    if (1ull * a.batch.max_tokens * (a.q_heads / a.cache.heads) > few) {
        const cudaError_t e = paged_attention_many_rows(ctx, a);
        if (e != cudaErrorNotSupported) return e;
    }
    switch (a.type) {
    case RowType::kF32: return launch_few<RowType::kF32>(ctx, a);
    case RowType::kF16: return launch_few<RowType::kF16>(ctx, a);
    default: return launch_few<RowType::kBF16>(ctx, a);
    }
}

}  // namespace vnpu_b200
