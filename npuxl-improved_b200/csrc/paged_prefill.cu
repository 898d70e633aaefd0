// paged_prefill.cu - PAGED_ATTENTION for many query rows: both products on the
// 5th-generation tensor cores, accumulators in tensor memory.
//
// The mathematics is paged_attention.cu's.  A CTA works on 128 query rows of
// one key/value head (tokens x grouped heads, packed) and walks their keys in
// tiles of KT: four converter warps turn the tile's codes into f16 in shared
// memory (exact), one thread issues S = Q K^T and O += P V, and four softmax
// warps, one row a thread, read S from tensor memory, write the weights P back
// over it as f16 (the A operand of the second product comes from tensor
// memory), and rescale O there when a maximum grew.  Two CTAs share an SM, so
// one's softmax runs under the other's products and under its own first and
// last tiles.
//
// f32 rows: Q = hi + lo in f16 (22 bits), P likewise; each product is two
// tensor instructions on the same accumulator, with tiles of 64 keys so that S
// and both halves of P fit beside each other.
//
// What bounds it: at head_dim 128 a 128 x 128 tile costs 16384 exponentials at
// 16 a clock (1024 clocks) against 512 clocks of the tensor core, and about as
// much again in issue slots for the conversion, the maxima and the scaling.
//
// Work units are (head, block of 128 rows, key tile), counted exactly by a
// planning kernel of one block; every CTA gets an equal run of them, whatever
// the sequences' lengths, the mask and the number of rows, and blocks that
// are split over CTAs are joined afterwards.
#include <algorithm>

#include "paged_attention.cuh"

namespace vnpu_b200 {
namespace {

constexpr uint32_t kRows = 128;              // query rows of a block (UMMA M)
constexpr uint32_t kManyThreads = 288;       // 4 softmax, 4 converter, 1 tensor-issue warps
constexpr uint32_t kPlanThreads = 1024;

// A block of rows and the key tiles that any of its rows sees.
struct RowBlock {
    uint32_t b, rb;
    int32_t lo, nt;
};

struct Plan {
    uint32_t *head;        // [0]: blocks, [1]: tiles of one head
    uint32_t *seq_base;    // [batch + 1]: blocks before sequence b
    RowBlock *blocks;
    uint32_t *before;      // tiles before block e (one head)
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
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *sh, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t v = x;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = sh[lane];
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sh[lane] = w;
    }
    __syncthreads();
    const uint32_t base = warp ? sh[warp - 1] : 0;
    *total = sh[31];
    __syncthreads();
    return base + v - x;
}

template <uint32_t KT>
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const AttnParams p, const Plan plan) {
    __shared__ uint32_t sh[32];
    pdl_enter();
    const uint32_t tid = threadIdx.x, batch = p.pb.batch;
    uint32_t blocks = 0, total;
    for (uint32_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint32_t mine = 0;
        if (b < batch) {
            PagedSeq s;
            if (!load_seq(p.pb, p.c.page_shift, b, s)) record_error(p.err, kErrBadIndex);
            else mine = (static_cast<uint32_t>(s.n) * p.group + kRows - 1) / kRows;
        }
        const uint32_t at = blocks + block_scan(mine, sh, &total);
        if (b < batch) plan.seq_base[b] = at;
        blocks += total;
    }
    if (tid == 0) plan.seq_base[batch] = blocks;
    __syncthreads();
    uint32_t tiles = 0;
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
        }
        const uint32_t at = tiles + block_scan(static_cast<uint32_t>(x.nt), sh, &total);
        if (e < blocks) plan.before[e] = at;
        tiles += total;
    }
    if (tid == 0) {
        plan.head[0] = blocks;
        plan.head[1] = tiles;
    }
}

// ---- tensor core wrappers -------------------------------------------------------
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// A from tensor memory: f16 pairs, 8 columns for 16 elements of K.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
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
__device__ __forceinline__ void tmem_st_16cols(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
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

template <RowType T, uint32_t DP>
struct ManyShape {
    static constexpr bool kSplit = T == RowType::kF32;
    static constexpr uint32_t KT = kSplit ? 64 : 128;          // keys of a tile
    static constexpr uint32_t NB = DP / 64;                     // 64-element column blocks
    static constexpr uint32_t kQBytes = kRows * DP * 2 * (kSplit ? 2 : 1);
    static constexpr uint32_t kKvBytes = KT * DP * 2;
    static constexpr uint32_t kSmem = kQBytes + 2 * kKvBytes + 1024;
    // tensor memory: S (KT columns; P over it, or for f32 hi and lo after it), O from column 128
    static constexpr uint32_t kPCol = kSplit ? 64 : 0, kOCol = 128, kCols = 256;
};

// Where a CTA stands in the units: head, block, tile; the roles walk alike.
struct Walk {
    const AttnParams *p;
    const Plan *plan;
    uint32_t left, h, e, blocks;    // tiles left; current head and block
    int32_t tile, count;            // first tile and tiles of this segment
    RowBlock x;
    PagedSeq s;

    // Takes the segment that begins `off` tiles into block e.
    __device__ __forceinline__ void take(uint32_t off) {
        const int4 v = __ldcg(reinterpret_cast<const int4 *>(plan->blocks) + e);
        x.b = static_cast<uint32_t>(v.x);
        x.rb = static_cast<uint32_t>(v.y);
        x.lo = v.z;
        x.nt = v.w;
        tile = x.lo + static_cast<int32_t>(off);
        count = min(x.nt - static_cast<int32_t>(off), static_cast<int32_t>(left));
        load_seq(p->pb, p->c.page_shift, x.b, s);
    }
    __device__ __forceinline__ bool next() {
        left -= static_cast<uint32_t>(count);
        if (!left) return false;
        if (++e == blocks) {
            e = 0;
            ++h;
        }
        take(0);
        return true;
    }
};

template <RowType T, uint32_t DP>
__global__ void __launch_bounds__(kManyThreads, 2)
    paged_prefill_kernel(const AttnParams p, const Plan plan) {
    using E = typename RowOf<T>::type;
    using Shape = ManyShape<T, DP>;
    constexpr bool kSplit = Shape::kSplit;
    constexpr uint32_t KT = Shape::KT, NB = Shape::NB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *const sq = smem, *const sk = smem + Shape::kQBytes, *const sv = sk + Shape::kKvBytes;
    __shared__ uint64_t bar_q, bar_o, bar_s, bar_p, bar_k, bar_k_free, bar_v, bar_v_free;
    __shared__ uint32_t sh_tmem;
    __shared__ int sh_abort;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, cta = blockIdx.x;
    const uint32_t D = p.c.head_dim;

    if (tid == 0) {
        sh_abort = 0;
        mbar_init(&bar_q, 128);
        mbar_init(&bar_p, 128);
        mbar_init(&bar_k, 128);
        mbar_init(&bar_v, 128);
        mbar_init(&bar_s, 1);
        mbar_init(&bar_o, 1);
        mbar_init(&bar_k_free, 1);
        mbar_init(&bar_v_free, 1);
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&sh_tmem, Shape::kCols);
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
    if (tid == 0) p.ws_meta[2 * cta].x = 0;   // nothing to join, unless the run says so at its end

    // ---- this CTA's run
    Walk w;
    w.p = &p;
    w.plan = &plan;
    w.blocks = __ldcg(plan.head);
    const uint32_t per_head = __ldcg(plan.head + 1);
    const uint64_t total = static_cast<uint64_t>(per_head) * p.c.heads;
    const uint64_t run = (total + gridDim.x - 1) / gridDim.x, t0 = run * cta;
    w.left = t0 < total ? static_cast<uint32_t>(min(run, total - t0)) : 0;
    const bool busy = w.left != 0;
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
        w.take(off - __ldcg(plan.before + lo));
    }
    // who joins what: the last segment, when its block begins here and goes on
    uint32_t parts = 0;

    if (busy && warp < 4) {
        // =============================== softmax ===============================
        const uint32_t row = tid;                                   // of the block; its TMEM lane
        const uint32_t lanes = tmem + (warp * 32u << 16);
        float f_next = 0.0f;
        // Query rows of a block to shared memory as f16, scaled by a power of two.
        const auto load_q = [&](const Walk &k) {
            const uint32_t r = k.x.rb * kRows + row, token = r / p.group;
            const bool live = r < static_cast<uint32_t>(k.s.n) * p.group;
            const E *q = static_cast<const E *>(p.Q) +
                         static_cast<uint64_t>(k.s.row0 + static_cast<int32_t>(token)) * p.ldq +
                         (k.h * p.group + (r - token * p.group)) * D;
            const bool vec = p.vec & 1u;
            float most = 0.0f;
            if (live)
                for (uint32_t d = 0; d < D; d += 8) {
                    float x[8];
                    load8(q + d, vec, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
                }
            const int ex = row_exponent(most);
            const float up = p.scale_log2 < 0.0f ? -pow2(ex) : pow2(ex);
            f_next = fabsf(p.scale_log2) * pow2(-ex);
#pragma unroll 4
            for (uint32_t d = 0; d < DP; d += 8) {
                float x[8] = {};
                if (live && d < D) load8(q + d, vec, x);
                uint4 hi, lo;
                uint32_t *h = reinterpret_cast<uint32_t *>(&hi), *l = reinterpret_cast<uint32_t *>(&lo);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = x[2 * i] * up, b = x[2 * i + 1] * up;
                    h[i] = pack_half2(a, b);
                    if constexpr (kSplit) {
                        const float2 g = unpack_half2(h[i]);
                        l[i] = pack_half2(a - g.x, b - g.y);
                    }
                }
                uint8_t *dst = sq + (d / 64) * (kRows * 128) + row * 128 + ((((d / 8) & 7u) ^ (row & 7u)) * 16);
                *reinterpret_cast<uint4 *>(dst) = hi;
                if constexpr (kSplit) *reinterpret_cast<uint4 *>(dst + kRows * DP * 2) = lo;
            }
            fence_proxy_async_smem();
            mbar_arrive(&bar_q);
        };
        // A tile's 16-key groups: lane g < KT / 16 holds group g's K scale, log2 of its V scale,
        // and 1 / V scale (0: a page of zeros, whose weights only count in the sum).
        constexpr uint32_t kGroups = KT / 16;
        float g_k = 0.0f, g_lv = 0.0f, g_iv = 1.0f, n_k = 0.0f, n_v = 0.0f;
        const auto fetch_scales = [&](const Walk &k, int32_t tile) {
            n_k = n_v = 0.0f;
            const int32_t key = tile * static_cast<int32_t>(KT) + static_cast<int32_t>(lane * 16u);
            if (lane >= kGroups || key >= k.s.len) return;
            const int32_t page = __ldg(p.pb.table + static_cast<uint64_t>(k.x.b) * p.pb.table_stride +
                                       (static_cast<uint32_t>(key) >> p.c.page_shift));
            if (page < 0 || static_cast<uint32_t>(page) >= p.c.num_pages) return;  // converters report it
            const uint64_t at = static_cast<uint64_t>(page) * p.c.heads + k.h;
            n_k = __ldg(p.c.K_scale + at);
            n_v = __ldg(p.c.V_scale + at);
        };
        load_q(w);
        fetch_scales(w, w.tile);
        uint32_t it = 0, seg = 0;
        bool more = true;
        while (more) {
            const float f = f_next;
            const Walk cur = w;
            int32_t kmin, kmax, kmin_last, kmax_first, unused;
            row_limits(p, cur.s, cur.x.rb * kRows + row, kmin, kmax);
            row_limits(p, cur.s, cur.x.rb * kRows, unused, kmax_first);
            row_limits(p, cur.s, cur.x.rb * kRows + kRows - 1, kmin_last, unused);
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int32_t j = 0; j < cur.count; ++j, ++it) {
                const int32_t k0 = (cur.tile + j) * static_cast<int32_t>(KT);
                g_k = n_k;
                g_lv = n_v > 0.0f ? __log2f(n_v) : 0.0f;
                g_iv = n_v > 0.0f ? ex2(-g_lv) : 1.0f;
                const uint32_t zeros = __ballot_sync(0xffffffffu, lane < kGroups && !(n_v > 0.0f));
                if (j + 1 < cur.count) fetch_scales(cur, cur.tile + j + 1);
                const bool edge = k0 + static_cast<int32_t>(KT) - 1 > kmax_first || k0 < kmin_last;
                if (!(ok = wait_warp(&bar_s, it))) break;
                tc_fence_after();
                // ---- the tile's maximum
                float top = -INFINITY;
#pragma unroll
                for (uint32_t c = 0; c < KT / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32cols(lanes + 32 * c, r);
                    tmem_wait_ld();
                    if (edge) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) {
                            const int32_t key = k0 + static_cast<int32_t>(32 * c + i);
                            if (key > kmax || key < kmin) r[i] = 0xff800000u;  // -infinity
                        }
                    }
#pragma unroll
                    for (uint32_t g = 0; g < 2; ++g) {
                        float x = __uint_as_float(r[16 * g]);
#pragma unroll
                        for (uint32_t i = 1; i < 16; ++i) x = fmaxf(x, __uint_as_float(r[16 * g + i]));
                        // scales are not negative: the largest product is the largest score
                        const float fg = f * __shfl_sync(0xffffffffu, g_k, 2 * c + g);
                        const float t = fmaf(x, fg, __shfl_sync(0xffffffffu, g_lv, 2 * c + g));
                        top = fmaxf(top, x == -INFINITY ? x : t);
                    }
                }
                // ---- rescale when some row's maximum grew by more than the slack
                const bool grown = top > m + kSlack;
                if (__any_sync(0xffffffffu, grown)) {
                    const float to = fmaxf(m, top);
                    const float a = to > m ? ex2(m - to) : 1.0f;
                    l *= a;
                    m = to;
                    if (j) {   // S of this tile is done, so the products before it are
#pragma unroll
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
                // ---- weights
#pragma unroll
                for (uint32_t c = 0; c < KT / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32cols(lanes + 32 * c, r);
                    tmem_wait_ld();
                    if (edge) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) {
                            const int32_t key = k0 + static_cast<int32_t>(32 * c + i);
                            if (key > kmax || key < kmin) r[i] = 0xff800000u;
                        }
                    }
                    uint32_t h[16], lo[16];
#pragma unroll
                    for (uint32_t g = 0; g < 2; ++g) {
                        // a zero factor keeps a masked key masked: -infinity * 0 is none
                        const float fg = fmaxf(f * __shfl_sync(0xffffffffu, g_k, 2 * c + g), 1e-38f);
                        const float b = __shfl_sync(0xffffffffu, g_lv, 2 * c + g) - off;
                        float sum = 0.0f;
#pragma unroll
                        for (uint32_t i = 0; i < 8; ++i) {
                            const float x = ex2(fmaf(__uint_as_float(r[16 * g + 2 * i]), fg, b));
                            const float y = ex2(fmaf(__uint_as_float(r[16 * g + 2 * i + 1]), fg, b));
                            sum += x + y;
                            h[8 * g + i] = pack_half2(x, y);
                            if constexpr (kSplit) {
                                const float2 u = unpack_half2(h[8 * g + i]);
                                lo[8 * g + i] = pack_half2(x - u.x, y - u.y);
                            }
                        }
                        l = fmaf(sum, __shfl_sync(0xffffffffu, g_iv, 2 * c + g), l);
                        if (zeros >> (2 * c + g) & 1u) {
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) h[8 * g + i] = lo[8 * g + i] = 0;
                        }
                    }
                    tmem_st_16cols(lanes + Shape::kPCol + 16 * c, h);
                    if constexpr (kSplit) tmem_st_16cols(lanes + Shape::kPCol + 32 + 16 * c, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&bar_p);
            }
            if (!ok) break;
            // All scores of this block are computed: the next block's queries may take its place.
            more = w.next();
            if (more) {
                load_q(w);
                fetch_scales(w, w.tile);
            }
            if (!wait_warp(&bar_o, seg++)) break;
            tc_fence_after();
            const uint32_t r = cur.x.rb * kRows + row, token = r / p.group;
            const bool live = r < static_cast<uint32_t>(cur.s.n) * p.group;
            const bool started = cur.tile == cur.x.lo;
            const bool whole = started && cur.count == cur.x.nt;
            const uint32_t part = 2 * cta + (started ? 1 : 0);
            if (started && !whole)
                parts = 1 + static_cast<uint32_t>((cur.x.nt - cur.count + run - 1) / run);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
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
                if (whole) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 8)
                        if (32 * c + i < D) {
                            float x[8];
#pragma unroll
                            for (uint32_t k = 0; k < 8; ++k) x[k] = __uint_as_float(v[i + k]) * inv;
                            store8(out + 32 * c + i, p.vec & 4u, x);
                        }
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4 *>(po + 32 * c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            if (live && !whole) p.ws_ml[part * kRows + row] = make_float2(m, l);
            if (tid == 0 && !more) {
                p.ws_meta[2 * cta] = make_uint4(parts, static_cast<uint32_t>(cur.s.row0), cur.x.rb * kRows, cur.h);
                p.ws_meta[2 * cta + 1] = make_uint4(
                    min(kRows, static_cast<uint32_t>(cur.s.n) * p.group - cur.x.rb * kRows), 0, 0, 0);
            }
            tc_fence_before();
        }
    } else if (busy && warp < 8) {
        // =============================== conversion ===============================
        constexpr uint32_t NC = DP / 16, RP = 128 / NC, NI = KT / RP;   // chunks a row, rows a step, steps
        const uint32_t ct = tid - 128, chunk = ct % NC, row0 = ct / NC;
        uint4 raw_k[NI], raw_v[NI];
        const uint32_t ps_mask = (1u << p.c.page_shift) - 1u;
        // A tile's codes of this thread; what is not there is zero.
        const auto fetch = [&](const Walk &k, int32_t tile, const int8_t *pool, uint4 (&raw)[NI]) {
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                const int32_t key = tile * static_cast<int32_t>(KT) + static_cast<int32_t>(i * RP + row0);
                raw[i] = make_uint4(0, 0, 0, 0);
                if (key >= k.s.len || chunk * 16u >= D) continue;
                const int32_t page = __ldg(p.pb.table + static_cast<uint64_t>(k.x.b) * p.pb.table_stride +
                                           (static_cast<uint32_t>(key) >> p.c.page_shift));
                if (page < 0 || static_cast<uint32_t>(page) >= p.c.num_pages) {
                    record_error(p.err, kErrBadIndex);
                    continue;
                }
                const uint64_t at = static_cast<uint64_t>(page) * p.c.heads + k.h;
                raw[i] = __ldg(reinterpret_cast<const uint4 *>(
                    pool + ((at << p.c.page_shift) + (static_cast<uint32_t>(key) & ps_mask)) * D + chunk * 16u));
            }
        };
        // 16 codes to two 16-byte pieces of a 128-byte swizzled row; the columns' upper half
        // writes its pieces in the other order, so that 8 lanes of a row meet 8 banks
        const auto put = [&](const uint4 (&raw)[NI], uint8_t *dst) {
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                const uint32_t row = i * RP + row0;
                uint4 a, b;
                codes_to_half4(raw[i].x, a.x, a.y);
                codes_to_half4(raw[i].y, a.z, a.w);
                codes_to_half4(raw[i].z, b.x, b.y);
                codes_to_half4(raw[i].w, b.z, b.w);
                uint8_t *at = dst + (chunk / 4u) * (KT * 128u) + row * 128u;
                const uint32_t piece = (chunk & 3u) * 2u, odd = chunk / 4u;
                *reinterpret_cast<uint4 *>(at + (((piece + odd) ^ (row & 7u)) * 16u)) = odd ? b : a;
                *reinterpret_cast<uint4 *>(at + (((piece + 1u - odd) ^ (row & 7u)) * 16u)) = odd ? a : b;
            }
            fence_proxy_async_smem();
        };
        uint32_t it = 0;
        bool ok = true, more = true;
        fetch(w, w.tile, p.c.K, raw_k);
        fetch(w, w.tile, p.c.V, raw_v);
        while (more && ok) {
            const Walk cur = w;
            for (int32_t j = 0; j < cur.count; ++j, ++it) {
                const bool last = j + 1 == cur.count;
                if (last) more = w.next();
                const int32_t tile = last ? w.tile : cur.tile + j + 1;   // the tile to fetch next
                if (it && !(ok = wait(&bar_k_free, it - 1))) break;
                put(raw_k, sk);
                mbar_arrive(&bar_k);
                if (!last || more) fetch(w, tile, p.c.K, raw_k);
                if (it && !(ok = wait(&bar_v_free, it - 1))) break;
                put(raw_v, sv);
                mbar_arrive(&bar_v);
                if (!last || more) fetch(w, tile, p.c.V, raw_v);
            }
        }
    } else if (busy && lane == 0) {
        // =============================== tensor products ===============================
        constexpr uint32_t idesc_s = umma_idesc_f16(kRows, KT, false);
        constexpr uint32_t idesc_o = umma_idesc_f16(kRows, DP, true);
        const uint32_t aq = smem_addr(sq), ak = smem_addr(sk), av = smem_addr(sv);
        uint32_t it = 0, seg = 0;
        bool ok = true, more = true;
        while (more && ok) {
            if (!(ok = wait(&bar_q, seg++))) break;
            for (int32_t j = 0; j < w.count; ++j, ++it) {
                if (!(ok = wait(&bar_k, it))) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t half = 0; half < (kSplit ? 2u : 1u); ++half)
#pragma unroll
                    for (uint32_t k = 0; k < DP / 16; ++k) {
                        const uint32_t q_off = half * (kRows * DP * 2) + (k / 4) * (kRows * 128) + (k % 4) * 32;
                        const uint32_t k_off = (k / 4) * (KT * 128) + (k % 4) * 32;
                        umma_f16_ss(tmem, umma_desc_k_sw128(aq + q_off), umma_desc_k_sw128(ak + k_off), idesc_s,
                                    half | k);
                    }
                umma_commit(&bar_k_free);
                umma_commit(&bar_s);
                if (!(ok = wait(&bar_p, it)) || !(ok = wait(&bar_v, it))) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t half = 0; half < (kSplit ? 2u : 1u); ++half)
#pragma unroll
                    for (uint32_t k = 0; k < KT / 16; ++k)
                        umma_f16_ts(tmem + Shape::kOCol, tmem + Shape::kPCol + 32 * half + 8 * k,
                                    umma_desc_mn_sw128(av + k * 2048, KT * 128), idesc_o,
                                    (j != 0) | half | k);
                umma_commit(&bar_v_free);
                if (j + 1 == w.count) umma_commit(&bar_o);
            }
            if (ok) more = w.next();
        }
    }
    __syncthreads();
    if (warp == 8) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, Shape::kCols);
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
            const float f = mm == -INFINITY ? 1.0f : ex2(mm - to), g = ml.x == -INFINITY ? 1.0f : ex2(ml.x - to);
            mm = to;
            ll = ll * f + ml.y * g;
            o.x = o.x * f + v.x * g;
            o.y = o.y * f + v.y * g;
            o.z = o.z * f + v.z * g;
            o.w = o.w * f + v.w * g;
        }
        const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
        const uint32_t r = meta.z + row, token = r / p.group;
        E *out = static_cast<E *>(p.O) + static_cast<uint64_t>(meta.y + token) * p.ldo +
                 (meta.w * p.group + (r - token * p.group)) * p.c.head_dim + 4u * d4;
        from_f32(o.x * inv, out[0]);
        from_f32(o.y * inv, out[1]);
        from_f32(o.z * inv, out[2]);
        from_f32(o.w * inv, out[3]);
    }
}

template <RowType T, uint32_t DP>
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
        VNPU_LAUNCH(cudaFuncSetAttribute(paged_prefill_kernel<T, DP>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem));
        ready_device = device;
    }
    const uint32_t grid = static_cast<uint32_t>(ctx.num_sms) * 2;
    const uint64_t blocks = static_cast<uint64_t>(a.batch.tokens) * p.group / kRows + a.batch.batch;
    const auto pad = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
    const size_t o_bytes = pad(2ull * grid * kRows * DP * sizeof(float));
    const size_t ml_bytes = pad(2ull * grid * kRows * sizeof(float2));
    const size_t meta_bytes = pad(2ull * grid * sizeof(uint4));
    const size_t block_bytes = pad(blocks * sizeof(RowBlock)), before_bytes = pad(blocks * sizeof(uint32_t));
    const size_t seq_bytes = pad((a.batch.batch + 1ull) * sizeof(uint32_t));
    char *ws = nullptr;
    VNPU_LAUNCH(cudaMallocAsync(reinterpret_cast<void **>(&ws),
                                o_bytes + ml_bytes + meta_bytes + block_bytes + before_bytes + seq_bytes + 256,
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
    Plan plan;
    plan.blocks = reinterpret_cast<RowBlock *>(carve(block_bytes));
    plan.before = reinterpret_cast<uint32_t *>(carve(before_bytes));
    plan.seq_base = reinterpret_cast<uint32_t *>(carve(seq_bytes));
    plan.head = reinterpret_cast<uint32_t *>(at);
    if (ctx.launch_counter) *ctx.launch_counter += 3;
    cudaError_t e = launch_pdl(ctx.stream, &paged_plan_kernel<Shape::KT>, dim3(1), dim3(kPlanThreads), 0, p, plan);
    if (e == cudaSuccess)
        e = launch_pdl(ctx.stream, &paged_prefill_kernel<T, DP>, dim3(grid), dim3(kManyThreads), Shape::kSmem, p, plan);
    if (e == cudaSuccess)
        e = launch_pdl(ctx.stream, &paged_prefill_join_kernel<T, DP>, dim3(grid, 4), dim3(256), 0, p);
    const cudaError_t f = cudaFreeAsync(ws, ctx.stream);
    return e == cudaSuccess ? f : e;
}

template <RowType T>
cudaError_t many_by_dim(const LaunchCtx &ctx, const PagedAttention &a) {
    if (a.cache.head_dim <= 64) return launch_many<T, 64>(ctx, a);
    return launch_many<T, 128>(ctx, a);
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
