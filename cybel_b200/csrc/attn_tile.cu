// Attention of many query rows over a paged cache on the 5th-generation tensor
// cores: whole prompts, chunks of a prompt, longer drafts.
//
// A CTA takes 256 rows (tokens x query heads of one kv head, row r = token
// r / group, head r % group) as two tiles of 128 and walks the positions they
// see 128 at a time. Per tile and step: S = Q K^T into tensor memory
// (tcgen05.mma kind::f16, M = N = 128), a warpgroup per tile turns S into
// weights -- one row per thread, so maximum and sum need no exchange -- and
// writes them back as fp16 over S, and O += P V takes P from tensor memory.
// While one tile's warpgroup works on its S, the tensor cores run the other
// tile's products: the exponentials (16 per clock and SM) and the products
// (1024 clocks a tile and step at head 128) bound the kernel together.
//
//  * warps 0-3, 4-7: softmax of tile 0, 1, and the tile's Q and output;
//  * warps 8-11: keys and values from the pages into a ring of 128-position
//    slots (128-byte swizzle, keys K-major, values MN-major as they lie).
//    Thread r looks up row r's page one step ahead; fp16 rows come by
//    cp.async, Q8 rows through registers, converted to their integer codes;
//  * warps 12, 13: issue the MMAs of tile 0, 1 (one warp for both took 4850
//    clocks a step, issuing one tile's while the other's were due).
//
// Q8 codes enter the products as they are; their scales multiply scores and
// weights in fp32, the latter relative to a power of two above the scales that
// the row has seen so far. (Code x scale rounded to fp16 for the products took 176 us instead of
// 208 at 4096 tokens, 32/8 heads, but each of the two roundings was as large as
// the output's own, and the error against 64 bits 2.4 times as large instead of
// 1.4 times. The weights' rounding to fp16 makes the rest of that factor.)
//
// fp32 rows: q and the weights are each two fp16 parts (22 bits), and both
// products run twice into the same accumulators, the low parts first. The
// tensor cores cut a sum off at each 16 products: over thousands of positions
// that shrank outputs by 0.035 x 2^-24 per position and spread them half as
// much. So a product covers a step (head 64) or 64 positions and 64 columns of
// the head (head 128) in an accumulator of its own, and the softmax warps add it
// to the output, which costs 370 us instead of 267 at 4096 tokens and makes the
// error 4e-7 instead of 2e-5 at 8000 positions. Values of one sign lose more: 0.11 x
// 2^-24 per position, 6.5e-3 over a million. fp16 rows keep the plain sum up to
// 32768 positions a CTA (2e-4, under half of their own rounding's 4.9e-4); longer
// ones are split further, and where eight CTAs do not reach, their products have
// accumulators of their own, too (head 128: 64 columns at a time beside the weights).
//
// The output is rescaled in tensor memory by the softmax warps themselves and
// only when a row's maximum rose by 2^kRise since the last time (fp32 rows: with
// the next addition): the product before is complete by then, because the
// barrier of S covers it. The weights
// are handed over in two halves, so that the product starts under the second
// half's exponentials.
//
// With few blocks of rows the positions are split over the CTAs of a cluster,
// which join their outputs through shared memory at the end (as in
// attn_few.cu). Every wait is bounded; a wait that gives up ends all roles.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn_ragged.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace b200q {

namespace {

constexpr int kThreads = 512;
constexpr int kRows = 128;       // rows of a tile (MMA M), positions of a step (N of S, K of P V)
constexpr int kTiles = 2;
constexpr int kCtaRows = kTiles * kRows;
constexpr int kMaxCluster = 8;
constexpr int kPlainSum = 32768;  // positions of a CTA whose sum the tensor cores keep (fp16 rows)
constexpr int kBadWords = 64;    // steps whose values were cleaned, one bit each
// Weights are 2^(score - reference maximum + kLift); the reference follows a
// row's maximum once that has risen by kRise, so they stay below 2^15 in fp16.
constexpr float kRise = 5.0f;
constexpr float kLift = 10.0f;
// Registers per thread after the split: 2 x softmax + loader + issuer = 512 =
// 4 x 128, what the block is launched with. (Q8 loaders hold a step's codes.)
constexpr int softmax_regs(bool q8) { return q8 ? 176 : 184; }
constexpr int loader_regs(bool q8) { return q8 ? 96 : 72; }
constexpr int issuer_regs(bool q8) { return 512 - 2 * softmax_regs(q8) - loader_regs(q8); }

template <bool SCALES>
struct Meta {
    uint32_t valid[4];           // bit: the position has a row that was loaded
    float vmax[4];               // largest finite value scale of each warp's 32
    float ks[kRows], vs[kRows];
};
template <>
struct Meta<false> {
    uint32_t valid[4];
};

// The rows and positions of one CTA.
struct Job {
    int live;
    int b, kvh;
    int row0;       // first row of the sequence's rows that the CTA takes
    int rows;       // of the sequence
    int first_tok;  // batch row of the sequence's first token
    int p0;         // its position
    Sight sight;
    int lo[kTiles], hi[kTiles];  // positions of the tiles' first and last rows (hi -1: no rows)
    // Whether a value that is not finite has to be kept out of the product
    // over positions j0 .. : some row does not see all of them, or the rows'
    // weights have low parts, which turn an infinity into NaN.
    template <bool PREC>
    __device__ __forceinline__ bool mixed(const Sight& s, int j0) const {
        return PREC || !s.all(lo[0], max(hi[0], hi[1]), j0, j0 + kRows - 1);
    }
};

// Which of a CTA's steps a tile takes part in: those of the prefix, and
// those that overlap what its own rows reach.
struct Steps {
    int prefix, from, to;
    __device__ __forceinline__ Steps(const Sight& s, const TileList<kRows>& list, int i0, int lo, int hi) {
        const bool any = hi >= max(lo, 0);
        prefix = any ? (s.pre + kRows - 1) / kRows - i0 : 0;
        from = list.before + max(s.first(max(lo, 0)) / kRows - list.from, 0) - i0;
        to = any && s.last(hi) >= 0 ? list.before + s.last(hi) / kRows - list.from - i0 : -1;
    }
    __device__ __forceinline__ bool has(int i) const { return i < prefix || (i >= from && i <= to); }
};

template <int D, bool PREC, bool Q8>
struct Tile {
    static constexpr int kHalf = kRows * 128;               // 128 rows x 64 fp16
    static constexpr int kMat = kHalf * (D / 64);           // one operand tile
    static constexpr int kParts = PREC ? 2 : 1;
    static constexpr int kQ = kTiles * kParts * kMat;
    static constexpr int kMeta = PREC ? 2 : 4;              // steps of per-position data in flight
    static constexpr int kMetaBytes = kMeta * static_cast<int>(sizeof(Meta<Q8>));
    static constexpr int kBarBytes = 320;
    static constexpr int kRest = kMetaBytes + kBarBytes + kBadWords * 4 + 128;
    static constexpr int kFree = (227 * 1024 - kQ - kRest) / kMat;
    static constexpr int NS = kFree > 6 ? 6 : kFree;        // ring slots
    static constexpr int kRing = kQ;
    static constexpr int kMetaAt = kRing + NS * kMat;
    static constexpr int kBars = kMetaAt + kMetaBytes;
    static constexpr int kBad = kBars + kBarBytes;
    static constexpr int kJob = kBad + kBadWords * 4;
    static constexpr int kTotal = kJob + 128;
    // after the loop, over Q and the ring: the tiles' outputs, then max and sum per row
    static constexpr int kMl = kTiles * kRows * D * 4;
    static constexpr int kNumBars = 2 * NS + 2 * kMeta + 4 * kTiles + 1 + 4 * kTiles;
    static_assert(NS >= 3 && kTotal <= 227 * 1024 && kMl + kCtaRows * 8 <= kMetaAt && kNumBars * 8 <= kBarBytes &&
                      sizeof(Job) <= 116,
                  "shared memory");
};

// ---- waits ----------------------------------------------------------------------
// A wait that runs out sets *dead, which ends every other wait too.
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* dead, volatile int* status) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1; it < kWaitMaxPolls; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
        if ((it & 7u) == 0u && global_timer_ns() - t0 > kWaitTimeoutNs) break;
    }
    *dead = 1;
    *status = STATUS_TIMEOUT;
    return false;
}
struct Waiter {
    volatile uint32_t* dead;
    volatile int* status;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        return mbar_test_wait(bar, parity) || mbar_try_wait(bar, parity) || wait_slow(bar, parity, dead, status);
    }
};

// Descriptors of operands with 128-byte swizzle: rows of 64 fp16, groups of 8
// rows 1024 bytes apart. Keys and Q are K-major (a row is 64 elements of the
// contraction, `other` unused); values are MN-major (a row is 64 elements of
// the output, halves of the head `other` bytes apart).
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t other) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>((other >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;  // descriptor version for sm_100
    d |= static_cast<uint64_t>(2) << 61;  // SWIZZLE_128B
    return d;
}
// fp16 operands, fp32 accumulator, M = 128; B K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc_of(int n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(kRows >> 4) << 24);
}

__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// The n lowest bits.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void put2(float* p, float2 v) { p[0] = v.x, p[1] = v.y; }

// Byte address of 16-byte chunk c (of D / 8) of row r of an operand tile.
template <int HALF>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The fp16 halves of w that are not finite set to 0.
__device__ __forceinline__ uint32_t clean16(uint32_t w) {
    if ((w & 0x7C00u) == 0x7C00u) w &= 0xFFFF0000u;
    if ((w & 0x7C000000u) == 0x7C000000u) w &= 0x0000FFFFu;
    return w;
}

// PREC: fp32 rows (two parts). OWN: products have accumulators of their own.
template <int D, bool PREC, bool OWN, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) b200q_attn_tile_kernel(const AttnArgs a) {
    using S = Tile<D, PREC, Q8>;
    using T = typename std::conditional<PREC, float, __half>::type;
    constexpr int NS = S::NS;
    constexpr int kMeta = S::kMeta;
    constexpr bool SC = Q8;  // scales beside the codes
    static_assert(OWN || !PREC, "fp32 rows' products have accumulators of their own");
    // Where they are: of a whole step (head 64: tensor memory has room), or of 64
    // columns at a time (and 64 positions, where the weights have two parts) beside
    // the weights, which the next product has to wait for.
    constexpr bool kWide = OWN && D == 64, kNarrow = OWN && D == 128;
    constexpr int kTurns = PREC ? 2 : 1;  // kNarrow: products of a step per 64 columns
    extern __shared__ __align__(1024) uint8_t smem[];
    Job* job_s = reinterpret_cast<Job*>(smem + S::kJob);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::kJob + 120);
    volatile uint32_t* dead = reinterpret_cast<volatile uint32_t*>(smem + S::kJob + 124);
    volatile uint32_t* any_bad = reinterpret_cast<volatile uint32_t*>(smem + S::kJob + 116);  // any of bad_bits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t C = cluster_size(), rank = cluster_rank();
    // What needs no input comes before the wait for the kernel ahead.
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    const uint32_t bar0 = smem_addr(bars);
    auto kvfull = [&](int i) { return bar0 + 8u * (i % NS); };
    auto kvempty = [&](int i) { return bar0 + 8u * (NS + i % NS); };
    auto mfull = [&](int i) { return bar0 + 8u * (2 * NS + i % kMeta); };
    auto mempty = [&](int i) { return bar0 + 8u * (2 * NS + kMeta + i % kMeta); };
    auto qfull = [&](int t) { return bar0 + 8u * (2 * NS + 2 * kMeta + t); };
    auto sready = [&](int t) { return bar0 + 8u * (2 * NS + 2 * kMeta + kTiles + t); };
    // Half of the weights is in place. kNarrow: the softmax warps are through with
    // what the next product overwrites (0), a product is complete (1).
    auto pready = [&](int t, int half) { return bar0 + 8u * (2 * NS + 2 * kMeta + 2 * kTiles + 2 * t + half); };
    const uint32_t done = bar0 + 8u * (2 * NS + 2 * kMeta + 4 * kTiles);
    auto turn = [&](int t, int w) { return done + 8u * (1 + 4 * t + w); };
    if (threadIdx.x == 32) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(kvfull(i), 4);
            mbar_init(kvempty(i), kTiles);
        }
        for (int i = 0; i < kMeta; ++i) {
            mbar_init(mfull(i), 4);
            mbar_init(mempty(i), 8);
        }
        for (int t = 0; t < kTiles; ++t) {
            mbar_init(qfull(t), kRows);
            mbar_init(sready(t), 1);
            mbar_init(pready(t, 0), 4);
            mbar_init(pready(t, 1), kNarrow ? 1 : 4);
            for (int w = 0; w < 4; ++w) mbar_init(turn(t, w), 1);
        }
        mbar_init(done, kTiles);
        fence_mbar_init();
    }
    if (warp == 12) {
        tmem_alloc(smem_addr(tmem_holder), 512);
        tmem_relinquish();
    }
    griddep_launch_dependents();
    griddep_wait();

    // ---- which rows: blocks of 256 rows of the sequences with more than
    // few_rows rows, the later blocks of a sequence (more positions) first
    const int cluster = blockIdx.x / C;
    if (warp == 0) {
        // the first 32 sequences' entries in one trip to memory
        const int b_lane = min(lane, a.r.batch - 1);
        const int2 rr_lane = seq_rows(a.r, b_lane);
        const Sight sight_lane = sight_of(a, b_lane);
        auto blocks = [&](int b) {
            if (b >= a.r.batch) return 0;
            const int2 rr = b < 32 ? rr_lane : seq_rows(a.r, b);
            const int rows = (rr.y - rr.x) * a.group;
            // (no more than the grid has room for, whatever the lengths say)
            return rows > a.few_rows ? (min(rows, a.most_rows) + kCtaRows - 1) / kCtaRows : 0;
        };
        int total = 0;
        for (int b0 = 0; b0 < a.r.batch; b0 += 32) total += blocks(b0 + lane);
        total = __reduce_add_sync(0xffffffffu, total);
        const int kvh = cluster % a.kv.n_kv;
        int x = total - 1 - cluster / a.kv.n_kv;
        if (lane == 0) {
            job_s->live = x >= 0;
            *dead = 0;
            *any_bad = 0;
        }
        for (int b0 = 0; b0 < a.r.batch && x >= 0; b0 += 32) {
            const int mine = blocks(b0 + lane);
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            if (x < upto && x >= upto - mine) {
                Job j;
                j.live = 1;
                const int2 rr = b0 == 0 ? rr_lane : seq_rows(a.r, b0 + lane);
                j.b = b0 + lane;
                j.kvh = kvh;
                j.rows = (rr.y - rr.x) * a.group;
                j.row0 = (x - (upto - mine)) * kCtaRows;
                j.first_tok = rr.x;
                j.sight = b0 == 0 ? sight_lane : sight_of(a, j.b);
                j.p0 = j.sight.n - (rr.y - rr.x);
                for (int t = 0; t < kTiles; ++t) {
                    const int r0 = j.row0 + t * kRows, r1 = min(r0 + kRows, j.rows) - 1;
                    j.lo[t] = j.p0 + div_by(r0, a.group_mul, a.group_shift);
                    j.hi[t] = r1 >= r0 ? j.p0 + div_by(r1, a.group_mul, a.group_shift) : -1;
                    if (r1 < r0) j.lo[t] = 0;
                }
                *job_s = j;
            }
            const int got = __shfl_sync(0xffffffffu, upto, 31);
            x = x < got ? -1 : x - got;
        }
    }
    for (int i = threadIdx.x; i < kBadWords; i += kThreads) reinterpret_cast<uint32_t*>(smem + S::kBad)[i] = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    if (!job_s->live) {  // the whole cluster
        if (warp == 12) tmem_dealloc(tmem, 512);
        return;
    }
    const Job& job = *job_s;
    const Sight sight = job.sight;
    const int lo = job.lo[0], hi = max(job.hi[0], job.hi[1]);
    const TileList<kRows> list(sight, lo, hi);
    const int n_all = hi < 0 ? 0 : list.count;
    if (threadIdx.x == 0 && sight.n > sight.limit) flag_bad_page(a.kv);
    const int i0 = static_cast<int>(static_cast<long long>(n_all) * rank / C);
    const int n = static_cast<int>(static_cast<long long>(n_all) * (rank + 1) / C) - i0;  // steps of this CTA
    const Waiter wait{dead, a.kv.status};
    const uint32_t sbase = smem_addr(smem);
    Meta<SC>* meta = reinterpret_cast<Meta<SC>*>(smem + S::kMetaAt);
    uint32_t* bad_bits = reinterpret_cast<uint32_t*>(smem + S::kBad);
    auto pos_of = [&](int i) { return list.at(i0 + i); };
    float2* ml = reinterpret_cast<float2*>(smem + S::kMl);
    // tensor-memory columns: S (then P) of the tiles, then their outputs, then kWide's accumulators
    constexpr uint32_t kO = 256, kF = 384;

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(issuer_regs(Q8)));
        if (warp < 12 + kTiles) {
            // ---------------- MMA issuer of tile t ----------------
            constexpr uint32_t idS = idesc_of(kRows, false), idO = idesc_of(kNarrow ? 64 : D, true);
            constexpr int kLast = S::kParts - 1;
            const int t = warp - 12;
            const Steps steps(sight, list, i0, job.lo[t], job.hi[t]);
            const uint32_t ts = tmem + t * kRows, to = tmem + kO + t * D;
            const uint64_t q0 = desc_sw128(sbase + t * S::kParts * S::kMat, 0);
            const uint64_t k0 = desc_sw128(sbase + S::kRing, 0), v0 = desc_sw128(sbase + S::kRing, S::kHalf);
            // One thread throughout, and the waits for operands that are early before
            // the wait for the weights, so that nothing stands between those and the
            // products (a wait by the whole warp costs 150 clocks even when it is over).
            if (elect_one()) {
                bool ok = wait(qfull(t), 0);
                int np = 0;  // steps so far
                int go = 0;  // kNarrow: products that waited for the softmax warps
                for (int s = 0; s <= n && ok; ++s) {
                    const int ki = 2 * s, vi = 2 * s - 1;
                    const bool pv = s > 0 && steps.has(s - 1), qk = s < n && steps.has(s);
                    ok = (s == n || wait(kvfull(ki), (ki / NS) & 1)) && (s == 0 || wait(kvfull(vi), (vi / NS) & 1));
                    if (pv) {
                        const uint64_t v = v0 + ((vi % NS) * (S::kMat >> 4));
#pragma unroll
                        for (int half = 0; half < (kNarrow ? kTurns : 2); ++half) {
                            if constexpr (kNarrow) {
#pragma unroll
                                for (int d = 0; d < D / 64; ++d) {
                                    ok = ok && wait(pready(t, 0), go++ & 1);
                                    if (!ok) break;
                                    tc_fence_after();
#pragma unroll
                                    for (int k = 0; k < 8; ++k)  // low parts first
                                        tc_mma_f16_ts(ts + 64, ts + (!PREC ? k * 8 : k < 4 ? 32 + k * 8 : (k - 4) * 8),
                                                      v + d * (S::kHalf >> 4) +
                                                          (PREC ? 4 * half + (k & 3) : k) * (2048 >> 4),
                                                      idO, k > 0 ? 1u : 0u);
                                    tc_commit(pready(t, 1));
                                }
                            } else {
                                ok = ok && wait(pready(t, half), (np - 1) & 1);
                                if (!ok) break;
                                tc_fence_after();
#pragma unroll
                                for (int part = kLast; part >= 0; --part)  // low parts first
#pragma unroll
                                    for (int k = 4 * half; k < 4 * half + 4; ++k)
                                        tc_mma_f16_ts(kWide ? tmem + kF + t * 64 : to, ts + part * 64 + k * 8,
                                                      v + k * (2048 >> 4), idO,
                                                      (!kWide && np > 1) || part < kLast || k > 0 ? 1u : 0u);
                            }
                        }
                    }
                    if (!ok) break;
                    if (qk) {
                        if (kNarrow && np > 0) ok = wait(pready(t, 0), go++ & 1);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t kk = k0 + ((ki % NS) * (S::kMat >> 4));
#pragma unroll
                        for (int part = kLast; part >= 0; --part)  // low parts first
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                const uint32_t off = ((k >> 2) * S::kHalf + (k & 3) * 32) >> 4;
                                tc_mma_f16(ts, q0 + ((part * S::kMat) >> 4) + off, kk + off, idS,
                                           part < kLast || k > 0 ? 1u : 0u);
                            }
                        tc_commit(sready(t));
                        ++np;
                    }
                    if (s > 0) tc_commit(kvempty(vi));
                    if (s < n) tc_commit(kvempty(ki));
                }
                tc_commit(done);  // what was issued still has to finish
            }
            __syncwarp();
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(loader_regs(Q8)));
        // ---------------- loader ----------------
        const int r = threadIdx.x - 256, w = warp - 8;
        const int hi_seen = sight.last(hi), lo_seen = sight.first(max(lo, 0));
        auto look = [&](int i) -> uint32_t {
            if (i >= n) return kNoRow;
            const int j = pos_of(i) + r;
            return (j <= hi_seen && (j < sight.pre || j >= lo_seen)) ? row_of(a, job.b, job.kvh, j) : kNoRow;
        };
        float ks_next = 0.0f, vs_next = 0.0f;  // Q8: the scales of the row looked up last
        // fp16 rows of one factor: it is part of the keys' scales where the scores are
        // shaped before the exponential.
        const float ks_mult = PREC || (a.cap == 0.0f && !a.slopes) ? 1.0f
                              : a.scale * (a.cap > 0.0f ? 1.0f / a.cap : kLog2e);
        auto scales_of = [&](uint32_t row) {
            if constexpr (Q8) {
                ks_next = row != kNoRow ? __ldg(a.kv.ks + row) : 0.0f;
                vs_next = row != kNoRow ? __ldg(a.kv.vs + row) : 0.0f;
            }
        };
        auto put_meta = [&](int i, uint32_t row) {
            Meta<SC>& m = meta[i % kMeta];
            const uint32_t bits = __ballot_sync(0xffffffffu, row != kNoRow);
            if (lane == 0) m.valid[w] = bits;
            if constexpr (Q8) {
                if (!(fabsf(vs_next) < INFINITY) && job.template mixed<PREC>(sight, pos_of(i))) {
                    vs_next = 0.0f;
                    atomicOr(bad_bits + (i >> 5) % kBadWords, 1u << (i & 31));
                    *any_bad = 1;
                }
            }
            if constexpr (SC) {
                m.ks[r] = ks_next * ks_mult;
                m.vs[r] = vs_next;
                const float mx = fabsf(vs_next) < INFINITY ? fabsf(vs_next) : 0.0f;
                const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
                if (lane == 0) m.vmax[w] = __uint_as_float(top);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(mfull(i));
        };
        bool ok = true;
        uint32_t ahead = look(0);
        if constexpr (!Q8) {
            constexpr int CH = D / 8, RPI = 32 / CH, NI = 32 / RPI;  // chunks per row, rows per copy, copies
            constexpr int LA = NS >= 5 ? 2 : 1;                      // items in flight behind the newest
            // Shared offsets of this thread's copies within the warp's 32 rows: they
            // repeat every 8 rows, up to the rows themselves.
            constexpr int PAT = 8 / RPI;
            uint32_t pat[PAT];
#pragma unroll
            for (int t = 0; t < PAT; ++t) pat[t] = chunk_at<S::kHalf>(w * 32 + t * RPI + lane / CH, lane % CH);
            // All of item x's copies of this thread have landed: clean what must
            // be, and hand it over.
            auto finish = [&](int x) {
                const uint32_t slot = sbase + S::kRing + (x % NS) * S::kMat;
                if ((x & 1) && job.template mixed<PREC>(sight, pos_of(x >> 1))) {
                    // An exponent of all ones plus one of its lowest bit carries into the
                    // sign's place, which the mask has cleared, and no further.
                    uint32_t found = 0;
#pragma unroll
                    for (int t = 0; t < NI; ++t) {
                        const uint4 v = lds128(slot + pat[t % PAT] + (t / PAT) * 1024);
                        found |= ((v.x & 0x7C007C00u) + 0x04000400u) | ((v.y & 0x7C007C00u) + 0x04000400u) |
                                 ((v.z & 0x7C007C00u) + 0x04000400u) | ((v.w & 0x7C007C00u) + 0x04000400u);
                    }
                    const bool bad = (found & 0x80008000u) != 0;
                    if (bad) {
#pragma unroll 1
                        for (int t = 0; t < NI; ++t) {
                            const uint32_t at = slot + chunk_at<S::kHalf>(w * 32 + t * RPI + lane / CH, lane % CH);
                            const uint4 v = lds128(at);
                            sts128(at, make_uint4(clean16(v.x), clean16(v.y), clean16(v.z), clean16(v.w)));
                        }
                    }
                    if (bad) {
                        atomicOr(bad_bits + (x >> 6) % kBadWords, 1u << ((x >> 1) & 31));
                        *any_bad = 1;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(kvfull(x));
            };
            // Waits for room before item x. Where there is none yet, what is on its way
            // is handed over first: the room may depend on it.
            int handed = 0;  // items finished
            auto room = [&](uint32_t bar, uint32_t parity, int x) {
                if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
                cp_async_wait<0>();
                while (handed < x) finish(handed++);
                ok = __all_sync(0xffffffffu, wait(bar, parity));
                return ok;
            };
            for (int i = 0; i < n && ok; ++i) {
                const uint32_t row = ahead;
                ahead = look(i + 1);
                if (!room(mempty(i), ((i / kMeta) & 1) ^ 1, 2 * i)) break;
                put_meta(i, row);
                // The warp's 32 rows one after the other in one page, as nearly always?
                const uint32_t row0 = __shfl_sync(0xffffffffu, row, 0);
                const bool run = __all_sync(0xffffffffu, row != kNoRow && row == row0 + lane);
                for (int part = 0; part < 2; ++part) {
                    const int x = 2 * i + part;
                    if (!room(kvempty(x), ((x / NS) & 1) ^ 1, x)) break;
                    const uint32_t slot = sbase + S::kRing + (x % NS) * S::kMat;
                    const uint8_t* src = static_cast<const uint8_t*>(part ? a.kv.v : a.kv.k) + (lane % CH) * 16;
                    if (run) {
                        src += static_cast<long long>(row0 + lane / CH) * (2 * D);
#pragma unroll
                        for (int t = 0; t < NI; ++t)
                            cp_async16(slot + pat[t % PAT] + (t / PAT) * 1024, src + t * (RPI * 2 * D), true);
                    } else {
#pragma unroll 4
                        for (int t = 0; t < NI; ++t) {
                            const uint32_t rw = __shfl_sync(0xffffffffu, row, t * RPI + lane / CH);
                            const bool have = rw != kNoRow;
                            cp_async16(slot + chunk_at<S::kHalf>(w * 32 + t * RPI + lane / CH, lane % CH),
                                       src + (have ? static_cast<long long>(rw) * (2 * D) : 0), have);
                        }
                    }
                    cp_async_commit();
                    if (handed <= x - LA) {
                        cp_async_wait<LA>();
                        finish(handed++);
                    }
                }
            }
            cp_async_wait<0>();
            if (ok)
                while (handed < 2 * n) finish(handed++);
        } else {
            constexpr int CH = D / 16, RPI = 32 / CH, NI = 32 / RPI;
            uint4 kreg[NI], vreg[NI];
            auto fetch = [&](uint4 (&reg)[NI], const void* base, uint32_t row) {
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    const uint32_t rw = __shfl_sync(0xffffffffu, row, t * RPI + lane / CH);
                    reg[t] = make_uint4(0u, 0u, 0u, 0u);
                    if (rw != kNoRow)
                        reg[t] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) +
                                                                      static_cast<long long>(rw) * D) +
                                       lane % CH);
                }
            };
            auto put = [&](const uint4 (&reg)[NI], int x) {
                const uint32_t slot = sbase + S::kRing + (x % NS) * S::kMat;
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    const int row = w * 32 + t * RPI + lane / CH, c = 2 * (lane % CH);
                    const uint32_t u[4] = {reg[t].x ^ 0x80808080u, reg[t].y ^ 0x80808080u, reg[t].z ^ 0x80808080u,
                                           reg[t].w ^ 0x80808080u};
                    uint32_t h[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) h[k] = codes_fp16(u[k >> 1], (k & 1) ? 0x4342 : 0x4140);
                    sts128(slot + chunk_at<S::kHalf>(row, c), make_uint4(h[0], h[1], h[2], h[3]));
                    sts128(slot + chunk_at<S::kHalf>(row, c + 1), make_uint4(h[4], h[5], h[6], h[7]));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(kvfull(x));
            };
            uint32_t row = ahead;
            ahead = look(1);
            if (n > 0) {
                scales_of(row);
                fetch(kreg, a.kv.k, row);
                fetch(vreg, a.kv.v, row);
            }
            for (int i = 0; i < n && ok; ++i) {
                ok = __all_sync(0xffffffffu, wait(mempty(i), ((i / kMeta) & 1) ^ 1));
                if (!ok) break;
                put_meta(i, row);
                row = ahead;
                scales_of(row);
                ahead = look(i + 2);
                ok = __all_sync(0xffffffffu, wait(kvempty(2 * i), ((2 * i / NS) & 1) ^ 1));
                if (!ok) break;
                put(kreg, 2 * i);
                fetch(kreg, a.kv.k, row);
                ok = __all_sync(0xffffffffu, wait(kvempty(2 * i + 1), (((2 * i + 1) / NS) & 1) ^ 1));
                if (!ok) break;
                put(vreg, 2 * i + 1);
                fetch(vreg, a.kv.v, row);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(softmax_regs(Q8)));
        // ---------------- softmax of tile t, row tid ----------------
        const int t = warp >> 2, tid = threadIdx.x & 127;
        const int row = job.row0 + t * kRows + tid;
        const bool have = row < job.rows;
        const int tok = have ? div_by(row, a.group_mul, a.group_shift) : 0, head = job.kvh * a.group + (have ? row - tok * a.group : 0);
        const int pos = job.p0 + tok;
        const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
        float mult = a.scale;
        {
            // Q of the warp's 32 rows, a row (fp32) or two (fp16) per load: fp16 as it
            // is, fp32 as two parts of q 2^10 / E, E a power of two above the row
            const uint32_t dst = sbase + t * S::kParts * S::kMat;
            const int w32 = (warp & 3) * 32;
            const long long mine = have ? (job.first_tok + tok) * a.q_stride + head * D : -1;  // of lane's row
            auto source = [&](int r) {  // row r of the warp's, NULL past the sequence
                const long long off = __shfl_sync(0xffffffffu, mine, r);
                return off >= 0 ? static_cast<const T*>(a.q) + off : nullptr;
            };
            if constexpr (!PREC) {
                constexpr int CH = D / 8, RPI = 32 / CH, NI = 32 / RPI;
#pragma unroll
                for (int k = 0; k < NI; ++k) {
                    const int r = k * RPI + lane / CH;
                    const T* src = source(r);
                    cp_async16(dst + chunk_at<S::kHalf>(w32 + r, lane % CH),
                               src ? src + (lane % CH) * 8 : static_cast<const T*>(a.q), src != nullptr);
                }
                cp_async_commit();
                cp_async_wait<0>();
            } else {
                constexpr int CH = D / 4, RPI = 32 / CH, NI = 32 / RPI, NB = 8;  // float4 per row; rows in flight
#pragma unroll 1
                for (int k0 = 0; k0 < NI; k0 += NB) {
                    float4 v[NB];
#pragma unroll
                    for (int k = 0; k < NB; ++k) {
                        const T* src = source((k0 + k) * RPI + lane / CH);
                        v[k] = src ? *reinterpret_cast<const float4*>(src + (lane % CH) * 4)
                                   : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
#pragma unroll
                    for (int k = 0; k < NB; ++k) {
                        const int r = (k0 + k) * RPI + lane / CH;
                        float amax = fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w)));
#pragma unroll
                        for (int o = CH / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                        const float E = fmaxf(pow2_above(amax < INFINITY ? amax : 0.0f), 7.8886090522e-31f);  // 2^-100
                        const float down = __fdiv_rn(1024.0f, E);
#pragma unroll
                        for (int h = 0; h < RPI; ++h) {
                            const float Eh = __shfl_sync(0xffffffffu, E, h * CH);
                            if (lane == (k0 + k) * RPI + h) mult = a.scale * (Eh * 0.0009765625f);
                        }
                        const float2 x = make_float2(v[k].x * down, v[k].y * down);
                        const float2 y = make_float2(v[k].z * down, v[k].w * down);
                        const uint32_t h0 = pack2(x.x, x.y), h1 = pack2(y.x, y.y);
                        const float2 f0 = unpack2(h0), f1 = unpack2(h1);
                        const uint32_t l0 = pack2(x.x - f0.x, x.y - f0.y), l1 = pack2(y.x - f1.x, y.y - f1.y);
                        const uint32_t at =
                            dst + chunk_at<S::kHalf>(w32 + r, (lane % CH) >> 1) + ((lane & 1) << 3);
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(h0), "r"(h1) : "memory");
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + S::kMat), "r"(l0), "r"(l1)
                                     : "memory");
                    }
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(qfull(t));
        }
        const bool shaped = a.cap > 0.0f || a.slopes != nullptr;
        const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
        // Factor left for the exponent: of a raw score, of tanh (cap alone), or none.
        const float to_log2 = !shaped ? mult * kLog2e : (a.slopes ? 1.0f : a.cap * kLog2e);
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + t * kRows, to = tmem + lanes + kO + t * D;
        const Steps mine(sight, list, i0, job.lo[t], job.hi[t]);
        const int t_lo = job.lo[t], t_hi = job.hi[t];
        float m = -INFINITY, l = 0.0f;
        float E = 0.0f, log_E = 0.0f;  // SC: the row's weights, their sum and its output are relative to E
        // OWN: 64 columns of the output, o keep + the product at f (o 0 before `add`).
        auto take = [&](uint32_t f, uint32_t o_at, bool add, float keep) {
#pragma unroll
            for (int c = 0; c < 64; c += 16) {
                float o[16], y[16];
                tmem_ld16(f + c, y);
                if (add) tmem_ld16(o_at + c, o);
                tmem_wait_ld();
                tmem_loaded16(y);
                if (add) {
                    tmem_loaded16(o);
#pragma unroll
                    for (int k = 0; k < 16; k += 2)
                        put2(y + k, fma2(make_float2(o[k], o[k + 1]), both(keep), make_float2(y[k], y[k + 1])));
                }
                tmem_st16(o_at + c, y);
            }
        };
        float last_keep = 1.0f;  // kWide: of the step whose product is not in the output yet
        int steps = 0;
        int drained = 0;  // kNarrow: products taken over so far
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            ok = __all_sync(0xffffffffu, wait(mfull(i), (i / kMeta) & 1));
            if (!ok) break;
            const Meta<SC>& md = meta[i % kMeta];
            // The exponentials' turn: the two warps that share a scheduler take
            // theirs one after the other, tile 0's first, so that one tile's
            // products run under the other's exponentials (left to themselves both
            // tiles fell in step and each unit idled half the time).
            const uint32_t my_turn = turn(t, warp & 3), next_turn = turn(t ^ 1, warp & 3);
            const bool wait_turn = t == 1 || i > 0;
            if (!mine.has(i)) {
                ok = __all_sync(0xffffffffu, !wait_turn || wait(my_turn, (i - 1 + t) & 1));
                if (lane == 0) {
                    mbar_arrive(next_turn);
                    mbar_arrive(mempty(i));
                }
                continue;
            }
            // Positions of the step that the row sees, 32 to a word: below the
            // prefix, or from a0 to a1.
            const int j0 = pos_of(i);
            const uint4 valid = *reinterpret_cast<const uint4*>(md.valid);
            const bool whole = (valid.x & valid.y & valid.z & valid.w) == 0xFFFFFFFFu &&
                               sight.all(t_lo, t_hi, j0, j0 + kRows - 1);
            uint32_t see[4] = {valid.x, valid.y, valid.z, valid.w};
            if (!whole) {
                const int pre = sight.pre - j0, a0 = sight.first(pos) - j0, a1 = pos - j0;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    see[w] &= below(pre - 32 * w) | (below(a1 + 1 - 32 * w) & ~below(a0 - 32 * w));
            }
            float unit = 1.0f;
            if constexpr (SC) {
                const float4 vm = *reinterpret_cast<const float4*>(md.vmax);
                float mx = fmaxf(fmaxf(vm.x, vm.y), fmaxf(vm.z, vm.w));
                if (mx >= E) {
                    if (!whole) {  // of the positions that the row sees: others' would push its weights below fp16
                        const uint32_t at = smem_addr(md.vs);
                        mx = 0.0f;
#pragma unroll
                        for (int c = 0; c < kRows; c += 4) {
                            const float4 v = lds_f4(at + c * 4);
                            const float f[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if ((see[c >> 5] & (1u << ((c + k) & 31))) && f[k] < INFINITY) mx = fmaxf(mx, f[k]);
                        }
                    }
                    if (mx >= E) {
                        const float e2 = fmaxf(pow2_above(mx), 8.6736173799e-19f);  // 2^-60
                        unit = E / e2;  // powers of two; 0 at the first step
                        E = e2;
                        log_E = static_cast<float>((__float_as_int(E) >> 23) - 127);
                    }
                }
            }
            ok = __all_sync(0xffffffffu, wait(sready(t), steps & 1));
            if (!ok) break;
            tc_fence_after();

            uint32_t ks_at = 0, vs_at = 0;
            if constexpr (SC) ks_at = smem_addr(md.ks), vs_at = smem_addr(md.vs);
            // ---- the step's exponents (times to_log2, plus row_off), from S
            float x[kRows];
            float row_off = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, x + 32 * c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_loaded32(x + 32 * c);
            if constexpr (SC) {
#pragma unroll
                for (int c = 0; c < kRows; c += 4) {
                    const float4 k = lds_f4(ks_at + c * 4);
                    // (multiplied as pairs, 120 registers of x were spilled: 272 us)
                    x[c] *= k.x, x[c + 1] *= k.y, x[c + 2] *= k.z, x[c + 3] *= k.w;
                }
            }
            if (shaped) {
                if (PREC || !SC) {
                    const float f1 = a.cap > 0.0f ? mult * inv_cap : mult * kLog2e;
#pragma unroll
                    for (int c = 0; c < kRows; c += 2) put2(x + c, mul2(make_float2(x[c], x[c + 1]), both(f1)));
                }
                if (a.cap > 0.0f) {
                    float far[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < kRows; c += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            far[u] = max3(far[u], fabsf(x[c + 2 * u]), fabsf(x[c + 2 * u + 1]));
                    // Far arguments take the other form one by one: it is off by 2^-22 absolutely,
                    // which the small scores beside them would feel (cap times as much).
                    constexpr float kFar = PREC ? 1.0f : 0.5f;
                    if (__any_sync(0xffffffffu, fmaxf(fmaxf(far[0], far[1]), fmaxf(far[2], far[3])) > kFar)) {
#pragma unroll
                        for (int c = 0; c < kRows; c += 2) {
                            const float2 z = make_float2(x[c], x[c + 1]), near = tanh_near<PREC>(z);
                            x[c] = fabsf(z.x) > kFar ? tanh_far(z.x) : near.x;
                            x[c + 1] = fabsf(z.y) > kFar ? tanh_far(z.y) : near.y;
                            // (four pairs at a time: all of them at once spill 300 to 500 bytes a thread)
                            if ((c & 6) == 6) asm volatile("" ::: "memory");
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < kRows; c += 2) put2(x + c, tanh_near<PREC>(make_float2(x[c], x[c + 1])));
                    }
                    if (a.slopes) {
#pragma unroll
                        for (int c = 0; c < kRows; c += 2)
                            put2(x + c, mul2(make_float2(x[c], x[c + 1]), both(a.cap * kLog2e)));
                    }
                }
                if (a.slopes) {
                    const float d0 = static_cast<float>(pos - j0);
                    if (j0 + kRows - 1 <= t_lo) {
                        // All behind the rows: the distance of the step's last position and the rest,
                        // so that the nearest biases, which matter most, are the smallest numbers.
                        constexpr int kEnd = kRows - 1;
                        row_off = -slope * (d0 - kEnd);
#pragma unroll
                        for (int c = 0; c < kRows; c += 2)
                            put2(x + c, fma2(both(slope), make_float2(c - kEnd, c + 1 - kEnd),
                                             make_float2(x[c], x[c + 1])));
                    } else {
#pragma unroll
                        for (int c = 0; c < kRows; ++c) x[c] = fmaf(-slope, fabsf(d0 - static_cast<float>(c)), x[c]);
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < kRows; ++c)
                    if (!(see[c >> 5] & (1u << (c & 31)))) x[c] = -INFINITY;
            }
            // ---- the reference maximum
            float keep = 1.0f;  // OWN: what the output so far is worth from here on
            {
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kRows; c += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) tops[u] = max3(tops[u], x[c + 2 * u], x[c + 2 * u + 1]);
                const float top = fmaf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), to_log2, row_off);
                const bool rise = top > m + kRise;
                if (__any_sync(0xffffffffu, rise || unit != 1.0f)) {
                    const float mn = rise ? top : m;
                    const float f = (m == -INFINITY ? 1.0f : ex2(m - mn)) * (steps > 0 ? unit : 1.0f);
                    m = mn;
                    l *= f;
                    keep = f;
                    if (!OWN && steps > 0) {
#pragma unroll
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            tmem_ld16(to + c, o);
                            tmem_wait_ld();
                            tmem_loaded16(o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] *= f;
                            tmem_st16(to + c, o);
                        }
                    }
                }
            }
            if constexpr (kWide) {  // the last step's product: complete, as S is
                if (steps > 0) {
                    take(tmem + lanes + kF + t * 64, to, steps > 1, last_keep);
                    tmem_wait_st();
                }
                last_keep = keep;
            }
            ok = __all_sync(0xffffffffu, !wait_turn || wait(my_turn, (i - 1 + t) & 1));
            if (!ok) break;
            // ---- weights, a quarter of the positions at a time
            const float base = m == -INFINITY ? 0.0f : kLift - m - log_E + row_off;
            float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            // kNarrow, two parts: the second half's, kept until the first half's products are done
            uint32_t parts[kNarrow && PREC ? 4 : 1][16];
#pragma unroll
            for (int quarter = 0; quarter < 4; ++quarter) {
                if (quarter == 3 && lane == 0) mbar_arrive(next_turn);  // its first loads run under this one's tail
                uint32_t hi16[16], lo16[16];
                float4 v4;
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float* xq = x + quarter * 32 + c;
                    if constexpr (SC) {
                        if (c % 4 == 0) v4 = lds_f4(vs_at + (quarter * 32 + c) * 4);
                    }
                    const float2 u = fma2(make_float2(xq[0], xq[1]), both(to_log2), both(base));
                    float2 p = make_float2(ex2(u.x), ex2(u.y));
                    s2[(c >> 1) & 1] = add2(s2[(c >> 1) & 1], p);
                    if constexpr (SC) p = mul2(p, c % 4 == 0 ? make_float2(v4.x, v4.y) : make_float2(v4.z, v4.w));
                    hi16[c / 2] = pack2(p.x, p.y);
                    if constexpr (PREC) {
                        const float2 h = unpack2(hi16[c / 2]);
                        lo16[c / 2] = pack2(p.x - h.x, p.y - h.y);
                    }
                }
                if (quarter == 2 && !(kNarrow && !PREC)) {  // the first half has arrived in tensor memory long ago
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pready(t, 0));
                }
                if constexpr (!kNarrow || !PREC) {
                    tmem_st16(ts + quarter * 16, hi16);
                    if constexpr (PREC) tmem_st16(ts + 64 + quarter * 16, lo16);
                } else if (quarter < 2) {
                    tmem_st16(ts + quarter * 16, hi16);
                    tmem_st16(ts + 32 + quarter * 16, lo16);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) parts[quarter - 2][k] = hi16[k], parts[quarter][k] = lo16[k];
                }
            }
            const float2 st = add2(s2[0], s2[1]);
            l += st.x + st.y;
            if constexpr (kNarrow) {
                if constexpr (!PREC) {
                    tmem_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) {
                    if constexpr (!PREC) mbar_arrive(pready(t, 0));
                    mbar_arrive(mempty(i));
                }
#pragma unroll
                for (int half = 0; half < kTurns; ++half) {
#pragma unroll
                    for (int d = 0; d < D / 64; ++d) {
                        ok = __all_sync(0xffffffffu, wait(pready(t, 1), drained++ & 1));
                        if (!ok) break;
                        tc_fence_after();
                        take(ts + 64, to + 64 * d, half > 0 || steps > 0, half > 0 ? 1.0f : keep);
                        if constexpr (PREC) {
                            if (half == 0 && d == D / 64 - 1) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) tmem_st16(ts + k * 16, parts[k]);
                            }
                        }
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(pready(t, 0));
                    }
                }
                if (!ok) break;
            } else {
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(pready(t, 1));
                    mbar_arrive(mempty(i));
                }
            }
            ++steps;
        }
        // ---------------- output ----------------
        ok = __all_sync(0xffffffffu, wait(done, 0));
        tc_fence_after();
        if constexpr (kWide) {
            if (steps > 0 && ok) {
                take(tmem + lanes + kF + t * 64, to, steps > 1, last_keep);
                tmem_wait_st();
            }
        }
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const float fin = C == 1 ? inv : (SC && l > 0.0f ? E : 1.0f);
        if (C > 1) ml[t * kRows + tid] = make_float2(m, l * fin);
        const bool bad = *any_bad != 0;
        // Through shared memory, so that rows leave in one piece: fp16 or fp32 rows
        // over the tile's Q (C = 1, this warp's rows only), or the fp32 parts of the
        // cluster over Q and the ring. `done` covers both tiles' products. 16-byte
        // chunks are spread by the row, so that a warp's rows fall on all banks.
        constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
        const uint32_t stage = C == 1 ? sbase + t * S::kParts * S::kMat + tid * kRowBytes
                                      : sbase + (t * kRows + tid) * (D * 4);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float o[32];
            if (steps > 0 && ok) {
                tmem_ld32(to + c, o);
                tmem_wait_ld();
                tmem_loaded32(o);
            } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= fin;
            if (bad && have) {  // values kept out of the product: to the rows that see them
#pragma unroll 1
                for (int i = 0; i < n; ++i) {
                    if (!((bad_bits[(i >> 5) % kBadWords] >> (i & 31)) & 1u)) continue;
                    const int j0 = pos_of(i);
                    if (!job.template mixed<PREC>(sight, j0)) continue;
#pragma unroll 1
                    for (int j = j0; j < min(j0 + kRows, sight.limit); ++j) {
                        const uint32_t rw = sight.sees(pos, j) ? row_of(a, job.b, job.kvh, j) : kNoRow;
                        if (rw == kNoRow) continue;
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const long long e = static_cast<long long>(rw) * D + c + k;
                            const float v = Q8 ? static_cast<const int8_t*>(a.kv.v)[e] * a.kv.vs[rw]
                                               : __half2float(static_cast<const __half*>(a.kv.v)[e]);
                            if (!(fabsf(v) < INFINITY)) o[k] += v;
                        }
                    }
                }
            }
            if (PREC || C > 1) {
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                    sts128(stage + ((((c + k) >> 2) ^ (tid & 7)) << 4),
                           make_uint4(__float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]),
                                      __float_as_uint(o[k + 3])));
            } else {
#pragma unroll
                for (int k = 0; k < 32; k += 8)
                    sts128(stage + ((((c + k) >> 3) ^ (tid & 7)) << 4),
                           make_uint4(pack2(o[k], o[k + 1]), pack2(o[k + 2], o[k + 3]), pack2(o[k + 4], o[k + 5]),
                                      pack2(o[k + 6], o[k + 7])));
            }
        }
        if (C == 1) {
            __syncwarp();
            constexpr int CH = kRowBytes / 16, RPI = 32 / CH, NI = 32 / RPI;
            const int w32 = (warp & 3) * 32;
            const long long to_out = have ? (job.first_tok + tok) * a.out_stride + head * D : -1;
#pragma unroll 8
            for (int k = 0; k < NI; ++k) {
                const int r = w32 + k * RPI + lane / CH;
                const long long off = __shfl_sync(0xffffffffu, to_out, k * RPI + lane / CH);
                if (off < 0) continue;
                const uint4 v = lds128(sbase + t * S::kParts * S::kMat + r * kRowBytes + (((lane % CH) ^ (r & 7)) << 4));
                *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + off + (lane % CH) * (16 / sizeof(T))) = v;
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 12) {
        mbar_wait_bounded(done, 0);  // complete already, unless a wait gave up
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (C == 1) return;
    // ---- join the parts of the cluster's CTAs: rows rank, rank + C, ... here
    cluster_sync();
    for (int it = threadIdx.x; it < kCtaRows / static_cast<int>(C) * (D / 4); it += kThreads) {
        const int r = it / (D / 4) * C + rank, e = it % (D / 4);
        const int row = job.row0 + r;
        if (row >= job.rows) continue;
        float2 part[kMaxCluster];
        float4 v[kMaxCluster];
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= static_cast<int>(C)) break;
            part[k] = ld_peer2(peer_addr(smem_addr(ml + r), k));
            v[k] = ld_peer4(peer_addr(sbase + r * (D * 4) + ((e ^ (r & 7)) << 4), k));
            M = fmaxf(M, part[k].x);
        }
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= static_cast<int>(C)) break;
            if (part[k].x == -INFINITY && part[k].y == 0.0f) continue;
            const float f = ex2(part[k].x - M);
            L += part[k].y * f;
            acc.x += v[k].x * f, acc.y += v[k].y * f, acc.z += v[k].z * f, acc.w += v[k].w * f;
        }
        const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
        const int tok = div_by(row, a.group_mul, a.group_shift), head = job.kvh * a.group + row - tok * a.group;
        T* out = static_cast<T*>(a.out) + (job.first_tok + tok) * a.out_stride + head * D + 4 * e;
        store_out4(out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool PREC, bool OWN, bool Q8>
int launch_tiles(const AttnArgs& a, long long units, int c, cudaStream_t st) {
    using S = Tile<D, PREC, Q8>;
    static std::mutex mu;
    static uint64_t done = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ECUDA;
    {
        std::lock_guard<std::mutex> lk(mu);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (!(done & bit)) {
            cudaFuncAttributes fa;
            // the register split adds up to 128 a thread: with fewer it would wait for ever
            if (cudaFuncGetAttributes(&fa, b200q_attn_tile_kernel<D, PREC, OWN, Q8>) != cudaSuccess ||
                fa.numRegs != 128 ||
                cudaFuncSetAttribute(b200q_attn_tile_kernel<D, PREC, OWN, Q8>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal) != cudaSuccess)
                return B200Q_ECUDA;
            done |= bit;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * c));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(c);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, b200q_attn_tile_kernel<D, PREC, OWN, Q8>, a) == cudaSuccess ? B200Q_OK
                                                                                                : B200Q_ECUDA;
}

}  // namespace

long long tile_blocks(int batch, long long total_rows, int most_rows, int few_rows) {
    const long long seqs = std::min<long long>(batch, total_rows / (few_rows + 1));
    return std::min(total_rows / kCtaRows + seqs, seqs * ((most_rows + kCtaRows - 1) / kCtaRows));
}

// While the blocks leave SMs idle, two steps a CTA at least (64 tokens of 32/8
// heads at 2000 positions, fp16: 22 us, 30 with four), and eight CTAs only for
// four fifths of the SMs: a GPC's are not a multiple of eight (16 clusters of
// eight took 37 us at 4000 positions, of four 26). More CTAs than that before a
// CTA's sum passes kPlainSum (fp16, 2048 tokens of 64/8 heads over 120 000
// positions: 8.0 ms unsplit, 8.7 over four CTAs, 11.2 with sums in fp32; over
// 250 000: 17.1, 21.6 over eight, 23.5; 1300 tokens of 32/1 heads over 120 000: 3.6,
// 2.3, 5.6). fp32 sums' own roundings add up, too: 3e-6 at 100 000 positions a CTA.
int tile_split(long long units, int max_kv, int sms) {
    int c = 1;
    while (c < kMaxCluster && units * c * 2 <= (c * 2 < kMaxCluster ? sms : sms * 4 / 5) && max_kv >= c * 2 * 2 * kRows)
        c *= 2;
    while (c < kMaxCluster && max_kv > c * kPlainSum) c *= 2;
    return c;
}

int launch_attn_tiles(const AttnArgs& a, int hd, bool fp32, bool q8, long long total_rows, int max_kv, int sms,
                      cudaStream_t st) {
    const long long units = tile_blocks(a.r.batch, total_rows, a.most_rows, a.few_rows) * a.kv.n_kv;
    if (units <= 0) return B200Q_OK;
    const int c = tile_split(units, max_kv, sms);
    if (units * c > 0x7fffffffll) return B200Q_ESHAPE;
    const bool own = max_kv > c * kPlainSum;
#define B200Q_TILES2(D, PREC, OWN) \
    (q8 ? launch_tiles<D, PREC, OWN, true>(a, units, c, st) : launch_tiles<D, PREC, OWN, false>(a, units, c, st))
#define B200Q_TILES(D) \
    (fp32 ? B200Q_TILES2(D, true, true) : own ? B200Q_TILES2(D, false, true) : B200Q_TILES2(D, false, false))
    return hd == 128 ? B200Q_TILES(128) : B200Q_TILES(64);
#undef B200Q_TILES
#undef B200Q_TILES2
}

}  // namespace b200q
