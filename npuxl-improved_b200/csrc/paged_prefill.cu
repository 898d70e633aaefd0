// paged_prefill.cu - PAGED_ATTENTION for many query rows: both products on the
// 5th-generation tensor cores, accumulators in tensor memory.
//
// The mathematics is paged_attention.cu's.  A CTA, one an SM, works on 256 query
// rows of one key/value head (tokens x grouped heads, packed) and walks their
// keys in tiles of KT.  Its warps:
//   17, 18  copy a tile's codes of K and of V to shared memory (bulk copies, half a
//           tile at a time) and its page scales beside them, ahead of their use;
//   8-15    turn the codes into f16 (exact), in the swizzled layout of the
//           tensor core's operands, four warps the first halves of the tiles
//           and four the second;
//   16      issues S = Q K^T and O += P V for both halves of the rows;
//   0-3, 4-7  softmax of 128 rows each, one row a thread: S is read from tensor
//           memory, the weights go back over it as f16 (the second product takes
//           its A operand from there), and O is rescaled there when a row's
//           maximum grew.  One half's softmax runs under the other's products.
//
// f32 rows: Q = hi + lo in f16 (22 bits), P likewise; each product is two
// tensor instructions on the same accumulator, with tiles of 64 keys so that S
// and both halves of P fit beside each other.  The tensor core's sums are not
// rounded to nearest, which over the steps of a long run is a drift (at 131072
// keys 3e-4 of the output): every kRunTiles tiles O moves to a sum in memory,
// added in f32, a thread a row.
//
// What bounds it: at head_dim 128 a 256 x 128 tile costs 32768 exponentials at
// 16 a clock (2048 clocks) against 2048 clocks of the tensor core, with about
// 1400 issue slots a scheduler beside them.  Measured, bf16, 32/8 heads of 128:
// 2048 tokens over 32768 keys 1257 us (847 TFLOP/s, 52 % of the measured product
// rate); 880 us with the softmax's arithmetic left out, of which the products
// are 463: the rest is a tile's way through the roles.
//
// Work units are (head, block of 256 rows, key tile), counted exactly by a
// planning kernel of one block; every CTA gets an equal run of them, whatever
// the sequences' lengths, the mask and the number of rows, and blocks that
// are split over CTAs are joined afterwards.
#include <algorithm>

#include "paged_attention.cuh"

namespace vnpu_b200 {
namespace {

constexpr uint32_t kHalf = 128;              // rows of one accumulator (UMMA M)
constexpr uint32_t kRows = 2 * kHalf;        // query rows of a block
constexpr uint32_t kManyThreads = 640;       // 8 softmax, 8 converter, tensor-issue, 2 copy, a spare warp
constexpr uint32_t kScaleRing = 4;           // tiles whose scales are kept
constexpr uint32_t kRawRing = 4;             // half tiles of codes: two of K, two of V
constexpr uint32_t kPlanThreads = 1024;
// f32 rows: tiles whose O the tensor core adds up.  2048 tokens over 32768 keys, 32/8 heads of 128, in us, and
// the drift: all 2400 and 8e-5, 32 tiles 2440 and 5e-6, 16 tiles 2520 and 2.7e-6, 8 tiles 2700 and 1.3e-6.
constexpr int32_t kRunTiles = 16;
// What the start and the end of a block cost beside its key tiles, in tiles: runs are of equal cost.
// (8 ragged prompts, 32/8 heads: 308 us with 0, 263 with 2, 255 with 3, 258 with 5, 270 with 8.)
constexpr int32_t kBlockCost = 3;

// A block of rows and the key tiles that any of its rows sees.
struct RowBlock {
    uint32_t b, rb;
    int32_t lo, nt;
};

struct Plan {
    uint32_t *head;        // [0]: blocks, [1]: cost of one head's
    uint32_t *seq_base;    // [batch + 1]: blocks before sequence b
    RowBlock *blocks;
    PagedSeq *seqs;        // block e's sequence
    uint32_t *before;      // cost of the blocks before block e (one head)
    uint32_t capacity;     // entries of `blocks`, `seqs` and `before`
};

template <uint32_t KT>
__device__ __forceinline__ RowBlock block_tiles(const AttnParams &p, const PagedSeq &s, uint32_t b,
                                                uint32_t rb) {
    RowBlock x{b, rb, 0, 1};
    int32_t kmin, kmax, unused;
    row_limits(p, s, rb * kRows, kmin, unused);
    row_limits(p, s, rb * kRows + kRows - 1, unused, kmax);
    x.lo = kmin / static_cast<int32_t>(KT);
    x.nt = max(1, kmax / static_cast<int32_t>(KT) + 1 - x.lo);
    return x;
}

// Exclusive prefix of x over the block, and the sum.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t *sh, uint64_t *total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint64_t v = x;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    if (warp == 0) {
        uint64_t w = sh[lane];
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sh[lane] = w;
    }
    __syncthreads();
    const uint64_t base = warp ? sh[warp - 1] : 0;
    *total = sh[31];
    __syncthreads();
    return base + v - x;
}

// Sequences are looked at one by one, and rows that do not fall share no rows:
// their blocks are within the capacity.  Where the numbers do fall, the same rows
// can count many times over; no entry of the plan is written before the sum is
// known to fit.
template <uint32_t KT>
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const AttnParams p, const Plan plan) {
    __shared__ uint64_t sh[32];
    pdl_enter();
    const uint32_t tid = threadIdx.x, batch = p.pb.batch;
    uint64_t blocks = 0, total;
    for (uint32_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint32_t mine = 0;
        if (b < batch) {
            PagedSeq s;
            if (!load_seq(p.pb, p.c.page_shift, b, s)) record_error(p.err, kErrBadIndex);
            else mine = (static_cast<uint32_t>(s.n) * p.group + kRows - 1) / kRows;
        }
        const uint64_t at = blocks + block_scan(mine, sh, &total);
        if (b < batch) plan.seq_base[b] = static_cast<uint32_t>(at);
        blocks += total;
    }
    if (blocks > plan.capacity) {       // nothing is done
        if (tid == 0) {
            record_error(p.err, kErrBadIndex);
            plan.head[0] = 0;
            plan.head[1] = 0;
        }
        return;
    }
    if (tid == 0) plan.seq_base[batch] = static_cast<uint32_t>(blocks);
    __syncthreads();
    uint64_t tiles = 0;
    for (uint32_t e0 = 0; e0 < blocks; e0 += kPlanThreads) {
        const uint32_t e = e0 + tid;
        RowBlock x{0, 0, 0, 0};
        if (e < blocks) {
            uint32_t lo = 0, hi = batch;           // the last sequence that begins at or before e
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (plan.seq_base[mid] <= e) lo = mid;
                else hi = mid;
            }
            PagedSeq s;
            load_seq(p.pb, p.c.page_shift, lo, s);
            x = block_tiles<KT>(p, s, lo, e - plan.seq_base[lo]);
            plan.blocks[e] = x;
            plan.seqs[e] = s;
        }
        const uint64_t at = tiles + block_scan(e < blocks ? static_cast<uint32_t>(x.nt + kBlockCost) : 0u, sh, &total);
        if (e < blocks) plan.before[e] = static_cast<uint32_t>(at);
        tiles += total;
    }
    // A run's units, and so all of them, are counted in 32 bits: more than 2^32 tiles of 256 rows,
    // a minute's work, are refused.
    const bool fits = tiles <= 0xffffffffu / p.c.heads;
    if (tid == 0) {
        if (!fits) record_error(p.err, kErrBadIndex);
        plan.head[0] = fits ? static_cast<uint32_t>(blocks) : 0;
        plan.head[1] = fits ? static_cast<uint32_t>(tiles) : 0;
    }
}

// ---- tensor core wrappers -------------------------------------------------------
// The whole warp runs the issuing code and one elected lane's instructions take
// effect: descriptors then stay in uniform registers (issued from a branch of
// one lane, an instruction of 64 clocks took 75 to 97 to issue).
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t is;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(is));
    return is;
}
__device__ __forceinline__ void umma_f16_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
// A from tensor memory: f16 pairs, 8 columns for 16 elements of K.
__device__ __forceinline__ void umma_f16_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                            uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint32_t lead, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(lead)
        : "memory");
}
// f16 x f16 -> f32, A K-major; B K-major or, transposed, MN-major.
__host__ __device__ constexpr uint32_t umma_idesc_f16(uint32_t m, uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// MN-major operand in 128-byte swizzled rows of 64 elements: 8-row groups
// 1024 bytes apart along K, further 64-element columns `chunk` bytes apart.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t chunk) {
    uint64_t d = umma_desc_k_sw128(saddr);
    d &= ~(0x3fffull << 16);
    return d | (static_cast<uint64_t>(chunk >> 4) << 16);
}
__device__ __forceinline__ void tmem_st_32cols(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <RowType T, uint32_t DP>
struct ManyShape {
    static constexpr bool kSplit = T == RowType::kF32;
    static constexpr uint32_t KT = kSplit ? 64 : 128;          // keys of a tile
    static constexpr uint32_t kQHalf = kHalf * DP * 2 * (kSplit ? 2 : 1);
    static constexpr uint32_t kKvBytes = KT * DP * 2;           // a tile of K or V in f16
    static constexpr uint32_t kRawBytes = KT * DP / 2;          // the codes of half of it
    // queries, two tiles of K and of V, four half tiles of codes
    static constexpr uint32_t kSmem = 2 * kQHalf + 4 * kKvBytes + kRawRing * kRawBytes + 1024;
    // tensor memory of a half: S (KT columns; P over it, or for f32 hi and lo after it), O
    static constexpr uint32_t kPCol = kSplit ? 64 : 0, kOCol = 128, kHalfCols = 256;
};

// Where a CTA stands in its run: head, block, tiles; the roles walk alike.  A
// block is kBlockCost units, then one for each key tile; a CTA has the tiles
// whose units are in its run.
static_assert(sizeof(RowBlock) == 16 && sizeof(PagedSeq) == 16, "read as one word each");
struct Walk {
    uint32_t left, h, e, blocks;    // units left; current head and block
    int32_t used;                   // units of this segment
    int32_t tile, count;            // its first tile and its tiles
    RowBlock x;
    PagedSeq s;

    // Takes the segment that begins `off` units into block e; it may have no tile.
    __device__ __forceinline__ void take(const AttnParams &p, const Plan &plan, uint32_t off) {
        const int4 v = __ldcg(reinterpret_cast<const int4 *>(plan.blocks) + e);
        x.b = static_cast<uint32_t>(v.x);
        x.rb = static_cast<uint32_t>(v.y);
        x.lo = v.z;
        x.nt = v.w;
        const int32_t from = static_cast<int32_t>(off);
        used = min(x.nt + kBlockCost - from, static_cast<int32_t>(min(left, 0x7fffffffu)));
        const int32_t first = max(0, from - kBlockCost);
        tile = x.lo + first;
        count = max(0, from + used - kBlockCost) - first;
        // the numbers that the plan looked at, whatever the arrays hold by now
        const int4 u = __ldcg(reinterpret_cast<const int4 *>(plan.seqs) + e);
        s.row0 = u.x;
        s.n = u.y;
        s.start = u.z;
        s.len = u.w;
    }
    // The next segment that has tiles.
    __device__ __forceinline__ bool next(const AttnParams &p, const Plan &plan) {
        do {
            left -= static_cast<uint32_t>(used);
            if (!left) return false;
            if (++e == blocks) {
                e = 0;
                ++h;
            }
            take(p, plan, 0);
        } while (!count);
        return true;
    }
};

// kRuns: f32 rows whose runs may pass kRunTiles tiles (the code for that costs the others a tenth).
template <RowType T, uint32_t DP, bool kRuns>
__global__ void __launch_bounds__(kManyThreads, 1)
    paged_prefill_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ Plan plan) {
    using E = typename RowOf<T>::type;
    using Shape = ManyShape<T, DP>;
    constexpr bool kSplit = Shape::kSplit;
    constexpr uint32_t KT = Shape::KT, kGroups = KT / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *const sq = smem, *const sk = smem + 2 * Shape::kQHalf, *const sv = sk + 2 * Shape::kKvBytes;
    uint8_t *const raw = sv + 2 * Shape::kKvBytes;
    __shared__ uint64_t bar_q[2], bar_o[2], bar_s[2], bar_p[2];          // of a half
    __shared__ uint64_t bar_k[2], bar_k_free[2], bar_v[2], bar_v_free[2];   // f16 tiles
    __shared__ uint64_t bar_r[kRawRing], bar_r_free[kRawRing];              // codes
    __shared__ uint64_t bar_sc[kScaleRing];
    // a tile's 16-key groups: K scale, log2 of the V scale (for the maximum, and for the weights),
    // 1 / V scale; pages of zeros as bits
    __shared__ __align__(16) float sh_k[kScaleRing][8], sh_top[kScaleRing][8], sh_lv[kScaleRing][8], sh_iv[kScaleRing][8];
    __shared__ uint32_t sh_zeros[kScaleRing];
    __shared__ uint32_t sh_tmem;
    __shared__ int sh_abort;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, cta = blockIdx.x;
    const uint32_t D = p.c.head_dim;

    if (tid == 0) {
        sh_abort = 0;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&bar_q[i], 4);
            mbar_init(&bar_p[i], 4);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_o[i], 1);
            mbar_init(&bar_k[i], 8);
            mbar_init(&bar_v[i], 8);
            mbar_init(&bar_k_free[i], 1);
            mbar_init(&bar_v_free[i], 1);
        }
#pragma unroll
        for (uint32_t i = 0; i < kRawRing; ++i) {
            mbar_init(&bar_r[i], 1);
            mbar_init(&bar_r_free[i], 4);
        }
#pragma unroll
        for (uint32_t i = 0; i < kScaleRing; ++i) mbar_init(&bar_sc[i], 1);
        fence_barrier_init();
    }
    if (warp == 16) {
        tmem_alloc(&sh_tmem, 2 * Shape::kHalfCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh_tmem;
    pdl_enter();
    const auto wait = [&](uint64_t *bar, uint32_t parity) {
        return mbar_wait(bar, parity & 1u, p.limit_ns, p.err, &sh_abort);
    };
    // the same for a whole warp, which goes on together (tensor memory loads need that)
    const auto wait_warp = [&](uint64_t *bar, uint32_t parity) {
        return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    };
    // one arrival a warp, for all that its lanes did (32 arrivals would queue up)
    const auto arrive_warp = [&](uint64_t *bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    if (tid == 0) p.ws_meta[2 * cta].x = 0;   // nothing to join, unless the run says so at its end

    // ---- this CTA's run
    Walk w;
    w.blocks = __ldcg(plan.head);
    const uint32_t per_head = __ldcg(plan.head + 1);
    const uint64_t total = static_cast<uint64_t>(per_head) * p.c.heads;
    const uint64_t run = (total + gridDim.x - 1) / gridDim.x, t0 = run * cta;
    w.left = t0 < total ? static_cast<uint32_t>(min(run, total - t0)) : 0;
    bool busy = w.left != 0;
    if (busy) {
        w.h = static_cast<uint32_t>(t0 / per_head);
        const uint32_t off = static_cast<uint32_t>(t0 - static_cast<uint64_t>(w.h) * per_head);
        // the last block with before[e] <= off: 32 probes a step
        uint32_t lo = 0, hi = w.blocks;
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
            const bool le = at < hi && __ldcg(plan.before + at) <= off;
            const uint32_t k = 31u - __clz(__ballot_sync(0xffffffffu, le));
            lo += k * step;
            hi = min(hi, lo + step);
        }
        w.e = lo;
        w.take(p, plan, off - __ldcg(plan.before + lo));
        if (!w.count) busy = w.next(p, plan);
    }

    // The block's 640 x 96 registers go where they are needed: 256 x 152 + 384 x 56.  (The spare
    // warp makes up the fifth warpgroup, so that every scheduler's share adds up, too.)
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");

    if (busy && warp < 8) {
        // =============================== softmax ===============================
        const uint32_t half = warp >> 2, quad = warp & 3u;
        const uint32_t row = half * kHalf + quad * 32u + lane;       // of the block
        const uint32_t lanes = tmem + half * Shape::kHalfCols + (quad << 21);   // lane quad * 32
        uint8_t *const q_half = sq + half * Shape::kQHalf;
        uint64_t *const full_s = &bar_s[half], *const full_p = &bar_p[half];
        float f_next = 0.0f;
        // Query rows to shared memory as f16, scaled by a power of two.  DP / 8 lanes take a
        // row, so a warp reads whole rows, 4 steps in work and 4 in flight.
        const auto load_q = [&](const Walk &k) {
            constexpr uint32_t LR = DP / 8, RI = 32 / LR, NS = 4;    // lanes a row, rows a step, steps at once
            const uint32_t d = (lane % LR) * 8, rows = static_cast<uint32_t>(k.s.n) * p.group;
            const bool vec = p.vec & 1u;
            int ex_mine = 0;
            const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
            constexpr uint32_t NW = sizeof(E) / 2;
            uint4 next[NS][NW];
            const auto read = [&](uint32_t i0) {
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) {
                    const uint32_t r = k.x.rb * kRows + (row & ~31u) + (i0 + i) * RI + lane / LR;
                    const uint32_t token = token_of(p, r);
#pragma unroll
                    for (uint32_t e = 0; e < NW; ++e) next[i][e] = make_uint4(0, 0, 0, 0);
                    if (r >= rows || d >= D) continue;
                    const E *src = static_cast<const E *>(p.Q) +
                                   static_cast<uint64_t>(k.s.row0 + static_cast<int32_t>(token)) * p.ldq +
                                   (k.h * p.group + (r - token * p.group)) * D + d;
                    if (vec) {
#pragma unroll
                        for (uint32_t e = 0; e < NW; ++e) next[i][e] = __ldg(reinterpret_cast<const uint4 *>(src) + e);
                    } else {
                        alignas(16) E x[8];
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) x[e] = src[e];
#pragma unroll
                        for (uint32_t e = 0; e < NW; ++e) next[i][e] = reinterpret_cast<const uint4 *>(x)[e];
                    }
                }
            };
            read(0);
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < LR; i0 += NS) {
                float y[NS][8];
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) {
                    alignas(16) E x[8];
#pragma unroll
                    for (uint32_t e = 0; e < NW; ++e) reinterpret_cast<uint4 *>(x)[e] = next[i][e];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] = to_f32(x[e]);
                }
                if (i0 + NS < LR) read(i0 + NS);
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) {
                    float most = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(y[i][e]));
#pragma unroll
                    for (uint32_t o = 1; o < LR; o <<= 1)
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    const int ex = row_exponent(most);
                    const float up = sign * pow2(ex);
                    // the lane that owns the row takes its exponent
                    const uint32_t first = (i0 + i) * RI;
                    const int got = __shfl_sync(0xffffffffu, ex, ((lane - first) * LR) & 31u);
                    if (lane / RI == i0 + i) ex_mine = got;
                    uint4 hi, lo;
                    uint32_t *h = reinterpret_cast<uint32_t *>(&hi), *l = reinterpret_cast<uint32_t *>(&lo);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = y[i][2 * e] * up, b = y[i][2 * e + 1] * up;
                        h[e] = pack_half2(a, b);
                        if constexpr (kSplit) {
                            const float2 g = unpack_half2(h[e]);
                            l[e] = pack_half2(a - g.x, b - g.y);
                        }
                    }
                    const uint32_t rr = quad * 32u + first + lane / LR;
                    uint8_t *dst = q_half + (d / 64) * (kHalf * 128) + rr * 128 + ((((d / 8) & 7u) ^ (rr & 7u)) * 16);
                    *reinterpret_cast<uint4 *>(dst) = hi;
                    if constexpr (kSplit) *reinterpret_cast<uint4 *>(dst + kHalf * DP * 2) = lo;
                }
            }
            f_next = fabsf(p.scale_log2) * pow2(-ex_mine);
            fence_proxy_async_smem();
            arrive_warp(&bar_q[half]);
        };
        const auto takes = [&](const Walk &k) {   // this half has rows of the block
            return half == 0 || static_cast<uint32_t>(k.s.n) * p.group > k.x.rb * kRows + kHalf;
        };
        uint32_t tile_no = 0, done = 0, seg = 0;  // tiles of the run; tiles and segments of this half
        float m = 0.0f, l = 0.0f, m_run = 0.0f;   // m_run: the maximum that the sums in memory go by
        float *const run_sums = p.ws_run + (static_cast<uint64_t>(cta) * DP * kRows + row);
        const auto read_sums = [&](uint32_t c, float (&had)[32]) {
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) had[i] = run_sums[(32 * c + i) * kRows];
        };
        bool more = true, ok = true, write = false;
        Walk cur = w;                             // the segment in work, whose output comes last
        for (;;) {
            // The scores of the segment before are all computed: these queries may take the place
            // of its own, and their first scores be computed while its output is written.
            if (more && takes(w)) load_q(w);
            const float f = f_next;
            if (write) {
                if (!wait_warp(&bar_o[half], seg++)) break;
                tc_fence_after();
                const bool started = cur.tile == cur.x.lo, whole = started && cur.count == cur.x.nt;
                const uint32_t r = cur.x.rb * kRows + row, token = token_of(p, r);
                const bool live = r < static_cast<uint32_t>(cur.s.n) * p.group;
                const uint32_t part = 2 * cta + (started ? 1 : 0);
                const float inv = inverse_sum(l);
                E *out = static_cast<E *>(p.O) +
                         static_cast<uint64_t>(cur.s.row0 + static_cast<int32_t>(token)) * p.ldo +
                         (cur.h * p.group + (r - token * p.group)) * D;
                float *po = p.ws_o + (static_cast<uint64_t>(part) * kRows + row) * DP;
#pragma unroll
                for (uint32_t c = 0; c < DP / 32; ++c) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld_32cols(lanes + Shape::kOCol + 32 * c, v);
                    tmem_wait_ld();
                    if (!live) continue;
                    if (kRuns && cur.count > kRunTiles) {
                        float had[32];
                        read_sums(c, had);
                        const float k = row_factor(m_run, m);
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i)
                            v[i] = __float_as_uint(fmaf(had[i], k, __uint_as_float(v[i])));
                    }
                    if (whole) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; i += 8)
                            if (32 * c + i < D) {
                                float x[8];
#pragma unroll
                                for (uint32_t k = 0; k < 8; ++k) x[k] = __uint_as_float(v[i + k]) * inv;
                                store_n(out + 32 * c + i, p.vec & 4u ? 16u : 1u, x);
                            }
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(po + 32 * c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                }
                if (live && !whole) p.ws_ml[part * kRows + row] = make_float2(m, l);
                tc_fence_before();
            }
            if (!more) break;
            cur = w;
            more = w.next(p, plan);
            if (tid == 0 && !more) {
                // joined with the CTAs that go on with the block, when it begins here
                uint32_t parts = 0;
                if (cur.tile == cur.x.lo && cur.count != cur.x.nt) {
                    const uint64_t end = static_cast<uint64_t>(cur.h) * per_head + __ldcg(plan.before + cur.e) +
                                         static_cast<uint32_t>(cur.x.nt + kBlockCost);
                    parts = static_cast<uint32_t>((end - 1) / run) - cta + 1;
                }
                p.ws_meta[2 * cta] = make_uint4(parts, static_cast<uint32_t>(cur.s.row0), cur.x.rb * kRows, cur.h);
                p.ws_meta[2 * cta + 1] = make_uint4(
                    min(kRows, static_cast<uint32_t>(cur.s.n) * p.group - cur.x.rb * kRows), 0, 0, 0);
            }
            write = takes(cur);
            if (!write) {
                tile_no += static_cast<uint32_t>(cur.count);
                continue;
            }
            int32_t kmin, kmax, kmin_last, kmax_first, unused;
            row_limits(p, cur.s, cur.x.rb * kRows + row, kmin, kmax);
            row_limits(p, cur.s, cur.x.rb * kRows + half * kHalf, unused, kmax_first);
            row_limits(p, cur.s, cur.x.rb * kRows + half * kHalf + kHalf - 1, kmin_last, unused);
            m = -INFINITY;
            l = 0.0f;
            for (int32_t j0 = 0; ok && j0 < cur.count; j0 += kRuns ? kRunTiles : cur.count) {
                if (kRuns && j0) {                    // a run's sums to memory
                    if (!(ok = wait_warp(full_s, done))) break;   // S of the next tile is done, so the products are
                    tc_fence_after();
                    const float k = row_factor(m_run, m);
#pragma unroll 1
                    for (uint32_t c = 0; c < DP / 32; ++c) {
                        uint32_t v[32];
                        float had[32];
                        if (j0 > kRunTiles) read_sums(c, had);
                        tmem_ld_32cols(lanes + Shape::kOCol + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i)
                            run_sums[(32 * c + i) * kRows] =
                                j0 > kRunTiles ? fmaf(had[i], k, __uint_as_float(v[i])) : __uint_as_float(v[i]);
                    }
                    m_run = m;
                }
                const int32_t j1 = kRuns ? min(cur.count, j0 + kRunTiles) : cur.count;
                for (int32_t j = j0; j < j1; ++j, ++tile_no, ++done) {
                    const int32_t k0 = (cur.tile + j) * static_cast<int32_t>(KT);
                    const uint32_t ring = tile_no % kScaleRing;
                    const bool edge = k0 + static_cast<int32_t>(KT) - 1 > kmax_first || k0 < kmin_last;
                    if (!(ok = wait_warp(&bar_sc[ring], tile_no / kScaleRing) && wait_warp(full_s, done))) break;
                    tc_fence_after();
                    const uint32_t zeros = sh_zeros[ring];
                    // Loops over 64 keys are not unrolled: the code of all roles has to stay in the
                    // instruction caches (unrolled, a fifth of the stalls were for instructions).
                    const auto read = [&](uint32_t c, uint32_t (&x)[64]) {
                        tmem_ld_32cols(lanes + 64 * c, *reinterpret_cast<uint32_t(*)[32]>(x));
                        tmem_ld_32cols(lanes + 64 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32));
                        tmem_wait_ld();
                        if (edge) {   // bits of the keys that the row sees
                            const int64_t lo = max(0, min(64, kmin - k0 - static_cast<int32_t>(64 * c)));
                            const int64_t hi = max(0, min(64, kmax + 1 - k0 - static_cast<int32_t>(64 * c)));
                            const uint64_t seen = (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 64 ? ~0ull : (1ull << lo) - 1);
#pragma unroll
                            for (uint32_t i = 0; i < 64; ++i)
                                if (!(seen >> i & 1u)) x[i] = 0xff800000u;  // -infinity
                        }
                    };
                    // a factor of zero would make masked scores NaN
                    const auto factor = [&](uint32_t g) { return fmaxf(f * sh_k[ring][g], 1e-38f); };
                    float top = -INFINITY;
#pragma unroll 1
                    for (uint32_t c = 0; c < KT / 64; ++c) {
                        uint32_t x[64];
                        read(c, x);
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g) {
                            const auto score = [&](uint32_t i) { return __uint_as_float(x[16 * g + i]); };
                            const float y0 = max3(score(0), score(1), score(2)), y1 = max3(score(3), score(4), score(5));
                            const float y2 = max3(score(6), score(7), score(8)), y3 = max3(score(9), score(10), score(11));
                            const float y4 = max3(score(12), score(13), score(14));
                            // scales are not negative: the largest product is the largest score
                            top = fmaxf(top, fmaf(fmaxf(max3(y0, y1, y2), max3(y3, y4, score(15))),
                                                  factor(4 * c + g), sh_top[ring][4 * c + g]));
                        }
                    }
                    if (__any_sync(0xffffffffu, top > m + kSlack)) {
                        // some row's maximum grew by more than the slack
                        const float to = fmaxf(m, top);
                        const float a = to > m ? ex2(m - to) : 1.0f;
                        l *= a;
                        m = to;
                        if (j != j0) {   // S of this tile is done, so the products before it are
#pragma unroll 1
                            for (uint32_t c = 0; c < DP / 32; ++c) {
                                uint32_t r[32];
                                tmem_ld_32cols(lanes + Shape::kOCol + 32 * c, r);
                                tmem_wait_ld();
#pragma unroll
                                for (uint32_t i = 0; i < 32; ++i)
                                    r[i] = __float_as_uint(__uint_as_float(r[i]) * a);
                                tmem_st_32cols(lanes + Shape::kOCol + 32 * c, r);
                            }
                        }
                    }
                    const float off = m == -INFINITY ? 0.0f : m - kLift;
#pragma unroll 1
                    for (uint32_t c = 0; c < KT / 64; ++c) {
                        uint32_t x[64], h[32], lo[kSplit ? 32 : 1];
                        read(c, x);
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g) {
                            const float fg = factor(4 * c + g), b = sh_lv[ring][4 * c + g] - off;
                            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) {
                                const float u = ex2(fmaf(__uint_as_float(x[16 * g + 2 * i]), fg, b));
                                const float v = ex2(fmaf(__uint_as_float(x[16 * g + 2 * i + 1]), fg, b));
                                s0 += u;
                                s1 += v;
                                h[8 * g + i] = pack_half2(u, v);
                                if constexpr (kSplit) {
                                    const float2 y = unpack_half2(h[8 * g + i]);
                                    lo[8 * g + i] = pack_half2(u - y.x, v - y.y);
                                }
                            }
                            l = fmaf(s0 + s1, sh_iv[ring][4 * c + g], l);
                        }
                        const uint32_t zero4 = zeros >> (4 * c) & 15u;
                        if (zero4) {   // pages of zeros count in the sum alone
#pragma unroll
                            for (uint32_t i = 0; i < 32; ++i)
                                if (zero4 >> (i / 8) & 1u) {
                                    h[i] = 0;
                                    if constexpr (kSplit) lo[i] = 0;
                                }
                        }
                        tmem_st_32cols(lanes + Shape::kPCol + 32 * c, h);
                        if constexpr (kSplit) tmem_st_32cols(lanes + Shape::kPCol + 32, lo);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    arrive_warp(full_p);
                }
            }
            if (!ok) break;
        }
    } else if (busy && warp < 16) {
        // =============================== conversion ===============================
        constexpr uint32_t NC = DP / 16, RP = 128 / NC, NI = KT / 2 / RP;  // chunks a row, rows a step, steps
        const uint32_t ct = tid & 127u, chunk = ct % NC, row0 = ct / NC, second = warp >= 12 ? 1u : 0u;
        const bool there = chunk * 16u < D;      // columns past head_dim are zeros
        // 16 codes to two 16-byte pieces of a 128-byte swizzled row.  The columns' upper half
        // takes its second 8 codes first, so that 8 lanes of a row meet 8 banks.  (RP is a
        // multiple of 8: a thread's rows share their place in the swizzle.)
        const bool odd = chunk >= 4u;
        const uint32_t piece = (chunk & 3u) * 2u, turn = row0 & 7u;
        const uint32_t to = (chunk / 4u) * (KT * 128u) + row0 * 128u;
        const uint32_t at0 = to + (((piece + odd) ^ turn) * 16u), at1 = to + (((piece + !odd) ^ turn) * 16u);
        const auto convert = [&](const uint8_t *codes, uint8_t *dst) {
            codes += row0 * D + chunk * 16u;
#pragma unroll 4
            for (uint32_t i = 0; i < NI; ++i) {
                uint4 c = make_uint4(0, 0, 0, 0), h;
                if (there) c = *reinterpret_cast<const uint4 *>(codes + i * RP * D);
                if (odd) c = make_uint4(c.z, c.w, c.x, c.y);
                codes_to_half4(c.x, h.x, h.y);
                codes_to_half4(c.y, h.z, h.w);
                *reinterpret_cast<uint4 *>(dst + at0 + i * RP * 128u) = h;
                codes_to_half4(c.z, h.x, h.y);
                codes_to_half4(c.w, h.z, h.w);
                *reinterpret_cast<uint4 *>(dst + at1 + i * RP * 128u) = h;
            }
            fence_proxy_async_smem();
        };
        // this warp's half of a tile's K, then of its V, and on to the next tile
        uint32_t it = 0;
        bool ok = true, more = true;
        while (more && ok) {
            const int32_t count = w.count;
            more = w.next(p, plan);
#pragma unroll 1
            for (int32_t x = 0; x < 2 * count; ++x) {
                const uint32_t st = it & 1u, v = x & 1u, slot = 2 * v + second;
                if (!(ok = wait_warp(&bar_r[slot], it))) break;
                if (it >= 2 && !(ok = wait_warp(v ? &bar_v_free[st] : &bar_k_free[st], (it >> 1) - 1))) break;
                convert(raw + slot * Shape::kRawBytes, (v ? sv : sk) + st * Shape::kKvBytes + second * (KT / 2 * 128u));
                arrive_warp(v ? &bar_v[st] : &bar_k[st]);
                arrive_warp(&bar_r_free[slot]);
                it += v;
            }
        }
    } else if (busy && warp == 16) {
        // =============================== tensor products ===============================
        const uint32_t lead = elect_lane();
        constexpr uint32_t idesc_s = umma_idesc_f16(kHalf, KT, false);
        constexpr uint32_t idesc_o = umma_idesc_f16(kHalf, DP, true);
        const uint32_t aq = smem_addr(sq), ak = smem_addr(sk), av = smem_addr(sv);
        const auto scores = [&](uint32_t half, uint32_t st) {
#pragma unroll
            for (uint32_t x = 0; x < (kSplit ? 2u : 1u); ++x)
#pragma unroll
                for (uint32_t k = 0; k < DP / 16; ++k) {
                    const uint32_t q_off = half * Shape::kQHalf + x * (kHalf * DP * 2) + (k / 4) * (kHalf * 128) + (k % 4) * 32;
                    const uint32_t k_off = (k / 4) * (KT * 128) + (k % 4) * 32;
                    umma_f16_ss(lead, tmem + half * Shape::kHalfCols, umma_desc_k_sw128(aq + q_off),
                                umma_desc_k_sw128(ak + st * Shape::kKvBytes + k_off), idesc_s, x | k);
                }
            umma_commit_by(lead, &bar_s[half]);
        };
        const auto values = [&](uint32_t half, uint32_t st, bool add) {
            const uint32_t d = tmem + half * Shape::kHalfCols;
#pragma unroll
            for (uint32_t x = 0; x < (kSplit ? 2u : 1u); ++x)
#pragma unroll
                for (uint32_t k = 0; k < KT / 16; ++k)
                    umma_f16_ts(lead, d + Shape::kOCol, d + Shape::kPCol + 32 * x + 8 * k,
                                umma_desc_mn_sw128(av + st * Shape::kKvBytes + k * 2048, KT * 128), idesc_o,
                                (add ? 1u : 0u) | x | k);
        };
        uint32_t it = 0, done[2] = {0, 0}, seg[2] = {0, 0};
        bool ok = true, more = true;
        while (more && ok) {
            const int32_t count = w.count;
            const uint32_t halves = static_cast<uint32_t>(w.s.n) * p.group > w.x.rb * kRows + kHalf ? 2 : 1;
            more = w.next(p, plan);
            // step -1 only computes the first tile's scores; a half's values of a tile and its
            // scores of the next one follow each other, while the other half has its softmax
#pragma unroll 1
            for (int32_t j = -1; j < count && ok; ++j) {
                const bool last = j + 1 == count;
                const uint32_t st = it & 1u;
                const uint32_t next = j < 0 ? it : it + 1;     // the tile of the scores
                if (j >= 0 && !(ok = wait_warp(&bar_v[st], it >> 1))) break;
#pragma unroll 1
                for (uint32_t half = 0; half < halves; ++half) {
                    if (j >= 0) {
                        if (!(ok = wait_warp(&bar_p[half], done[half]++))) break;
                        tc_fence_after();
                        values(half, st, kRuns ? j % kRunTiles != 0 : j != 0);
                    } else if (!(ok = wait_warp(&bar_q[half], seg[half]++))) {
                        break;
                    }
                    if (last) {
                        umma_commit_by(lead, &bar_o[half]);
                    } else {
                        if (half == 0 && !(ok = wait_warp(&bar_k[next & 1u], next >> 1))) break;
                        tc_fence_after();
                        scores(half, next & 1u);
                    }
                }
                if (!last) umma_commit_by(lead, &bar_k_free[next & 1u]);
                if (j >= 0) {
                    umma_commit_by(lead, &bar_v_free[st]);
                    ++it;
                }
            }
        }
    } else if (busy && (warp == 17 || warp == 18)) {
        // =============================== copies ===============================
        // Warp 17 copies K, and gives the scales; warp 18 copies V.  Lane g looks after group g of
        // 16 keys.  A tile's pages are looked up two tiles before its codes are copied, and its
        // scales read one tile before, so that neither is waited for.
        const bool values_too = warp == 18;
        const int8_t *const pool = values_too ? p.c.V : p.c.K;
        struct Group {
            bool real;          // there is such a tile
            int32_t page;       // -1: not there
            uint32_t h, slot;   // head; slot of its first key in the page
            float ks, vs;
        };
        int32_t j = 0;          // tiles of the segment looked up
        bool more = true;
        const auto look_up = [&](Group &g) {
            g.page = -1;
            g.ks = g.vs = 0.0f;
            g.real = more;
            if (!more) return;
            const int32_t key = (w.tile + j) * static_cast<int32_t>(KT) + static_cast<int32_t>(lane * 16u);
            g.h = w.h;
            g.slot = static_cast<uint32_t>(key) & ((1u << p.c.page_shift) - 1u);
            if (lane < kGroups && key < w.s.len)
                g.page = __ldg(p.pb.table + static_cast<uint64_t>(w.x.b) * p.pb.table_stride +
                               (static_cast<uint32_t>(key) >> p.c.page_shift));
            else
                g.slot = 0xffffffffu;
            if (++j == w.count) {
                j = 0;
                more = w.next(p, plan);
            }
        };
        const auto read_scales = [&](Group &g) {
            if (g.slot == 0xffffffffu) return;
            if (g.page < 0 || static_cast<uint32_t>(g.page) >= p.c.num_pages) {
                record_error(p.err, kErrBadIndex);
                g.page = -1;
                return;
            }
            const uint64_t at = static_cast<uint64_t>(g.page) * p.c.heads + g.h;
            if (values_too) return;
            g.ks = __ldg(p.c.K_scale + at);
            g.vs = __ldg(p.c.V_scale + at);
        };
        const uint32_t per_copy = min(1u << (p.c.page_shift - 4u), kGroups / 2);   // groups of a page in half a tile
        Group now, next, later;
        now.slot = next.slot = later.slot = 0xffffffffu;
        now.h = next.h = later.h = 0;
        look_up(next);
        look_up(later);
        read_scales(next);
        uint32_t begun = 0;     // tiles whose copies were begun
        bool ok = true;
        for (uint32_t it = 0; next.real; ++it) {
            now = next;
            next = later;
            later.slot = 0xffffffffu;
            look_up(later);
            if (next.real) read_scales(next);
            const uint32_t ring = it % kScaleRing;
            // A group that is not there stays as it is in shared memory (whole numbers all the
            // same); its keys are masked or count as zeros.
            const uint64_t at = now.page >= 0 ? static_cast<uint64_t>(now.page) * p.c.heads + now.h : 0;
            const uint32_t there = __ballot_sync(0xffffffffu, now.page >= 0);
            const uint64_t src = ((at << p.c.page_shift) + now.slot) * D;
            const uint32_t zeros = __ballot_sync(0xffffffffu, lane < kGroups && !(now.vs >= kLeastScale));
#pragma unroll 1
            for (uint32_t part = 0; part < 2; ++part) {
                constexpr uint32_t kPart = kGroups / 2;      // groups of half a tile
                const uint32_t slot = 2 * values_too + part, first = part * kPart;
                // Half a tile is copied when its place's last one is converted.  K's first half:
                // K of tile it - 1 is then, so the scores of tile it - 3 are there (two tiles of K
                // are kept), and so the weights of tile it - 4: its scales' place is free, too.
                if (it && !(ok = wait_warp(&bar_r_free[slot], it - 1))) break;
                if (lane == 0)
                    mbar_arrive_expect_tx(&bar_r[slot], 16u * D * __popc(there >> first & ((1u << kPart) - 1u)));
                begun = it + 1;
                // one copy for the groups of a page, issued warp-uniformly (a branch of the lanes
                // that own them took 300 clocks)
#pragma unroll 1
                for (uint32_t g = first; g < first + kPart; g += per_copy) {
                    const uint32_t n = __popc(there >> g & ((1u << per_copy) - 1u));
                    const uint64_t from = __shfl_sync(0xffffffffu, src, g);
                    if (n && lane == 0)
                        bulk_load_1d(raw + slot * Shape::kRawBytes + (g - first) * 16u * D, pool + from, 16u * D * n,
                                     &bar_r[slot]);
                }
                if (part == 0 && !values_too) {
                    if (lane < kGroups) {
                        const bool on = now.vs >= kLeastScale;   // else a page of zeros
                        const float lv = on ? __log2f(now.vs) : 0.0f;
                        sh_k[ring][lane] = now.ks;
                        sh_top[ring][lane] = on ? lv : kZeroLog;
                        sh_lv[ring][lane] = lv;
                        sh_iv[ring][lane] = on ? reciprocal(now.vs) : 1.0f;   // what lv is off by cancels in o / l
                    }
                    if (lane == 0) sh_zeros[ring] = zeros;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_sc[ring]);
                }
            }
            if (!ok) break;
        }
        // a run that was given up may leave copies in flight: they end before the block does
        if (!ok && begun)
            for (uint32_t part = 0; part < 2; ++part) {
                const uint32_t slot = 2 * values_too + part;
                if (begun > 1) mbar_wait(&bar_r[slot], begun & 1u, p.limit_ns, nullptr, nullptr);
                mbar_wait(&bar_r[slot], (begun - 1) & 1u, p.limit_ns, nullptr, nullptr);
            }
    }
    __syncthreads();
    if (warp == 16) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 2 * Shape::kHalfCols);
    }
}

// Joins the parts of the block of rows that begins in CTA blockIdx.x and goes
// on in the next ones, in their order.
template <RowType T, uint32_t DP>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const AttnParams p) {
    using E = typename RowOf<T>::type;
    pdl_enter();
    const uint32_t cta = blockIdx.x;
    const uint4 meta = p.ws_meta[2 * cta];
    if (meta.x < 2) return;
    const uint32_t rows = p.ws_meta[2 * cta + 1].x;
    for (uint32_t i = blockIdx.y * 256u + threadIdx.x; i < rows * (DP / 4); i += gridDim.y * 256u) {
        const uint32_t row = i / (DP / 4), d4 = i % (DP / 4);
        if (4u * d4 >= p.c.head_dim) continue;
        float mm = -INFINITY, ll = 0.0f;
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (uint32_t k = 0; k < meta.x; ++k) {
            const uint64_t at = (k == 0 ? 2ull * cta + 1 : 2ull * (cta + k)) * kRows + row;
            const float2 ml = p.ws_ml[at];
            const float4 v = reinterpret_cast<const float4 *>(p.ws_o)[at * (DP / 4) + d4];
            const float to = fmaxf(mm, ml.x);
            const float f = row_factor(mm, to), g = row_factor(ml.x, to);
            mm = to;
            ll = ll * f + ml.y * g;
            o.x = o.x * f + v.x * g;
            o.y = o.y * f + v.y * g;
            o.z = o.z * f + v.z * g;
            o.w = o.w * f + v.w * g;
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
}

template <RowType T, uint32_t DP, bool kRuns>
cudaError_t launch_many(const LaunchCtx &ctx, const PagedAttention &a) {
    using Shape = ManyShape<T, DP>;
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
            (reinterpret_cast<uintptr_t>(a.O) % 16u == 0 && 1ull * a.ldo * elem % 16u == 0 ? 4u : 0u);
    p.err = ctx.err;
    p.limit_ns = ctx.wait_limit_ns;
    static thread_local int ready_device = -1;
    int device = 0;
    VNPU_LAUNCH(cudaGetDevice(&device));
    if (ready_device != device) {
        VNPU_LAUNCH(cudaFuncSetAttribute(paged_prefill_kernel<T, DP, kRuns>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem));
        ready_device = device;
    }
    const uint32_t grid = static_cast<uint32_t>(ctx.num_sms);
    const uint64_t blocks = static_cast<uint64_t>(a.batch.tokens) * p.group / kRows + a.batch.batch;
    const auto pad = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
    const size_t o_bytes = pad(2ull * grid * kRows * DP * sizeof(float));
    const size_t ml_bytes = pad(2ull * grid * kRows * sizeof(float2));
    const size_t meta_bytes = pad(2ull * grid * sizeof(uint4));
    const size_t block_bytes = pad(blocks * sizeof(RowBlock)), before_bytes = pad(blocks * sizeof(uint32_t));
    const size_t seqs_bytes = pad(blocks * sizeof(PagedSeq));
    const size_t run_bytes = kRuns ? pad(1ull * grid * kRows * DP * sizeof(float)) : 0;
    const size_t seq_bytes = pad((a.batch.batch + 1ull) * sizeof(uint32_t));
    char *ws = nullptr;
    VNPU_LAUNCH(cudaMallocAsync(reinterpret_cast<void **>(&ws),
                                o_bytes + ml_bytes + meta_bytes + block_bytes + seqs_bytes + before_bytes + seq_bytes + run_bytes +
                                    256,
                                ctx.stream));
    char *at = ws;
    const auto carve = [&](size_t n) {
        char *x = at;
        at += n;
        return x;
    };
    p.ws_o = reinterpret_cast<float *>(carve(o_bytes));
    p.ws_ml = reinterpret_cast<float2 *>(carve(ml_bytes));
    p.ws_meta = reinterpret_cast<uint4 *>(carve(meta_bytes));
    p.ws_run = reinterpret_cast<float *>(carve(run_bytes));
    Plan plan;
    plan.capacity = static_cast<uint32_t>(blocks);   // below 2^23 + 2^24
    plan.blocks = reinterpret_cast<RowBlock *>(carve(block_bytes));
    plan.seqs = reinterpret_cast<PagedSeq *>(carve(seqs_bytes));
    plan.before = reinterpret_cast<uint32_t *>(carve(before_bytes));
    plan.seq_base = reinterpret_cast<uint32_t *>(carve(seq_bytes));
    plan.head = reinterpret_cast<uint32_t *>(at);
    if (ctx.launch_counter) *ctx.launch_counter += 3;
    cudaError_t e = launch_pdl(ctx.stream, &paged_plan_kernel<Shape::KT>, dim3(1), dim3(kPlanThreads), 0, p, plan);
    if (e == cudaSuccess)
        e = launch_pdl(ctx.stream, &paged_prefill_kernel<T, DP, kRuns>, dim3(grid), dim3(kManyThreads), Shape::kSmem, p,
                       plan);
    if (e == cudaSuccess)
        e = launch_pdl(ctx.stream, &paged_prefill_join_kernel<T, DP>, dim3(grid, kRows * DP / 4 / 256), dim3(256), 0, p);
    const cudaError_t f = cudaFreeAsync(ws, ctx.stream);
    return e == cudaSuccess ? f : e;
}

template <RowType T, uint32_t DP>
cudaError_t many_by_reach(const LaunchCtx &ctx, const PagedAttention &a) {
    if constexpr (ManyShape<T, DP>::kSplit) {
        const uint64_t reach = static_cast<uint64_t>(a.batch.table_stride) << a.cache.page_shift;
        if (reach > static_cast<uint64_t>(kRunTiles) * ManyShape<T, DP>::KT) return launch_many<T, DP, true>(ctx, a);
    }
    return launch_many<T, DP, false>(ctx, a);
}
template <RowType T>
cudaError_t many_by_dim(const LaunchCtx &ctx, const PagedAttention &a) {
    if (a.cache.head_dim <= 64) return many_by_reach<T, 64>(ctx, a);
    return many_by_reach<T, 128>(ctx, a);
}

}  // namespace

cudaError_t paged_attention_many_rows(const LaunchCtx &ctx, const PagedAttention &a) {
    if (a.cache.head_dim > 128) return cudaErrorNotSupported;  // O and S of 256 columns do not fit twice
    switch (a.type) {
    case RowType::kF32: return many_by_dim<RowType::kF32>(ctx, a);
    case RowType::kF16: return many_by_dim<RowType::kF16>(ctx, a);
    default: return many_by_dim<RowType::kBF16>(ctx, a);
    }
}

}  // namespace vnpu_b200
