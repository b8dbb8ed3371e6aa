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
//  * warp 12: issues the MMAs.
//
// fp32 rows: q and the weights are each two fp16 parts (22 bits), both
// products run twice into the same accumulators. Q8 scales multiply scores
// and weights, the latter relative to a power of two above the scales so far.
// The output is rescaled in tensor memory by the softmax warps themselves and
// only when a row's maximum rose by 2^kRise since the last time: by then the
// product before is complete, because the barrier of S covers it.
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
constexpr int kBadWords = 64;    // steps whose values were cleaned, one bit each
constexpr float kRise = 5.0f;    // weights are at most 2^(kRise + kLift) = 2^15 in fp16
constexpr float kLift = 10.0f;
// Registers per thread after the split; 128 x (2 x 176 + 104 + 56) = 65536 =
// 512 x 128, what the block is launched with.
constexpr int kSoftmaxRegs = 176, kLoaderRegs = 104, kIssuerRegs = 56;

template <bool Q8>
struct Meta {
    uint32_t valid[4];           // bit: the position has a row that was loaded
    float vmax[4];               // Q8: largest finite value scale of each warp's 32
    float ks[kRows], vs[kRows];  // Q8
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
    int lo[kTiles], hi[kTiles];  // positions of the tiles' first and last rows (hi -1: no rows)
    __device__ __forceinline__ bool needs(const Sight& s, int t, int j0) const {
        const int top = max(hi[t], s.pre - 1);
        return hi[t] >= max(lo[t], 0) && j0 <= top && (j0 < s.pre || j0 + kRows > s.first(max(lo[t], 0)));
    }
    // Whether a value that is not finite has to be kept out of the product
    // over positions j0 .. : some row does not see all of them, or the rows'
    // weights have low parts, which turn an infinity into NaN.
    template <bool PREC>
    __device__ __forceinline__ bool mixed(const Sight& s, int j0) const {
        return PREC || !s.all(lo[0], max(hi[0], hi[1]), j0, j0 + kRows - 1);
    }
};

template <int D, bool PREC, bool Q8>
struct Tile {
    static constexpr int kHalf = kRows * 128;               // 128 rows x 64 fp16
    static constexpr int kMat = kHalf * (D / 64);           // one operand tile
    static constexpr int kParts = PREC ? 2 : 1;
    static constexpr int kQ = kTiles * kParts * kMat;
    static constexpr int kMeta = PREC ? 2 : 4;              // steps of per-position data in flight
    static constexpr int kMetaBytes = kMeta * static_cast<int>(sizeof(Meta<Q8>));
    static constexpr int kRest = kMetaBytes + 256 + kBadWords * 4 + 128;
    static constexpr int kFree = (227 * 1024 - kQ - kRest) / kMat;
    static constexpr int NS = kFree > 6 ? 6 : kFree;        // ring slots
    static constexpr int kRing = kQ;
    static constexpr int kMetaAt = kRing + NS * kMat;
    static constexpr int kBars = kMetaAt + kMetaBytes;
    static constexpr int kBad = kBars + 256;
    static constexpr int kJob = kBad + kBadWords * 4;
    static constexpr int kTotal = kJob + 128;
    // after the loop, over Q and the ring: the tiles' outputs, then max and sum per row
    static constexpr int kMl = kTiles * kRows * D * 4;
    static constexpr int kNumBars = 2 * NS + 2 * kMeta + 3 * kTiles + 1;
    static_assert(NS >= 3 && kTotal <= 227 * 1024 && kMl + kCtaRows * 8 <= kMetaAt && kNumBars * 8 <= 256 &&
                      sizeof(Job) + 8 <= 128,
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
    *status = *status | STATUS_TIMEOUT;
    return false;
}
struct Waiter {
    volatile uint32_t* dead;
    volatile int* status;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        return mbar_try_wait(bar, parity) || wait_slow(bar, parity, dead, status);
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
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// Byte address of 16-byte chunk c (of D / 8) of row r of an operand tile.
template <int HALF>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Two codes + 128 as fp16: 0x64 above a byte u is 1024 + u; less 1152 the code.
__device__ __forceinline__ uint32_t codes_fp16(uint32_t bytes, uint32_t sel) {
    const uint32_t h = __byte_perm(bytes, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// The fp16 halves of w that are not finite set to 0.
__device__ __forceinline__ uint32_t clean16(uint32_t w) {
    if ((w & 0x7C00u) == 0x7C00u) w &= 0xFFFF0000u;
    if ((w & 0x7C000000u) == 0x7C000000u) w &= 0x0000FFFFu;
    return w;
}

template <int D, bool PREC, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) b200q_attn_tile_kernel(const AttnArgs a) {
    using S = Tile<D, PREC, Q8>;
    using T = typename std::conditional<PREC, float, __half>::type;
    constexpr int NS = S::NS;
    constexpr int kMeta = S::kMeta;
    extern __shared__ __align__(1024) uint8_t smem[];
    Job* job_s = reinterpret_cast<Job*>(smem + S::kJob);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::kJob + 120);
    volatile uint32_t* dead = reinterpret_cast<volatile uint32_t*>(smem + S::kJob + 124);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t C = cluster_size(), rank = cluster_rank();
    griddep_launch_dependents();
    griddep_wait();

    // ---- which rows: blocks of 256 rows of the sequences with more than
    // few_rows rows, the later blocks of a sequence (more positions) first
    const int cluster = blockIdx.x / C;
    if (warp == 0) {
        auto blocks = [&](int b) {
            if (b >= a.r.batch) return 0;
            const int2 rr = seq_rows(a.r, b);
            const int rows = (rr.y - rr.x) * a.group;
            return rows > a.few_rows ? (rows + kCtaRows - 1) / kCtaRows : 0;
        };
        int total = 0;
        for (int b0 = 0; b0 < a.r.batch; b0 += 32) total += blocks(b0 + lane);
        total = __reduce_add_sync(0xffffffffu, total);
        const int kvh = cluster % a.kv.n_kv;
        int x = total - 1 - cluster / a.kv.n_kv;
        if (lane == 0) {
            job_s->live = x >= 0;
            *dead = 0;
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
                const int2 rr = seq_rows(a.r, b0 + lane);
                j.b = b0 + lane;
                j.kvh = kvh;
                j.rows = (rr.y - rr.x) * a.group;
                j.row0 = (x - (upto - mine)) * kCtaRows;
                j.first_tok = rr.x;
                j.p0 = a.r.kv_len[j.b] - (rr.y - rr.x);
                for (int t = 0; t < kTiles; ++t) {
                    const int r0 = j.row0 + t * kRows, r1 = min(r0 + kRows, j.rows) - 1;
                    j.lo[t] = j.p0 + r0 / a.group;
                    j.hi[t] = r1 >= r0 ? j.p0 + r1 / a.group : -1;
                    if (r1 < r0) j.lo[t] = 0;
                }
                *job_s = j;
            }
            const int got = __shfl_sync(0xffffffffu, upto, 31);
            x = x < got ? -1 : x - got;
        }
    }
    for (int i = threadIdx.x; i < kBadWords; i += kThreads) reinterpret_cast<uint32_t*>(smem + S::kBad)[i] = 0;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    const uint32_t bar0 = smem_addr(bars);
    auto kvfull = [&](int i) { return bar0 + 8u * (i % NS); };
    auto kvempty = [&](int i) { return bar0 + 8u * (NS + i % NS); };
    auto mfull = [&](int i) { return bar0 + 8u * (2 * NS + i % kMeta); };
    auto mempty = [&](int i) { return bar0 + 8u * (2 * NS + kMeta + i % kMeta); };
    auto qfull = [&](int t) { return bar0 + 8u * (2 * NS + 2 * kMeta + t); };
    auto sready = [&](int t) { return bar0 + 8u * (2 * NS + 2 * kMeta + kTiles + t); };
    auto pready = [&](int t) { return bar0 + 8u * (2 * NS + 2 * kMeta + 2 * kTiles + t); };
    const uint32_t done = bar0 + 8u * (2 * NS + 2 * kMeta + 3 * kTiles);
    if (threadIdx.x == 32) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(kvfull(i), kRows);
            mbar_init(kvempty(i), 1);
        }
        for (int i = 0; i < kMeta; ++i) {
            mbar_init(mfull(i), 4);
            mbar_init(mempty(i), 8);
        }
        for (int t = 0; t < kTiles; ++t) {
            mbar_init(qfull(t), kRows);
            mbar_init(sready(t), 1);
            mbar_init(pready(t), 4);
        }
        mbar_init(done, 1);
        fence_mbar_init();
    }
    __syncthreads();
    if (!job_s->live) return;  // the whole cluster
    if (warp == 12) {
        tmem_alloc(smem_addr(tmem_holder), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    const Job& job = *job_s;
    const Sight sight = sight_of(a, job.b);
    const int lo = job.lo[0], hi = max(job.hi[0], job.hi[1]);
    const TileList<kRows> list(sight, lo, hi);
    const int n_all = hi < 0 ? 0 : list.count;
    const int i0 = static_cast<int>(static_cast<long long>(n_all) * rank / C);
    const int n = static_cast<int>(static_cast<long long>(n_all) * (rank + 1) / C) - i0;  // steps of this CTA
    const Waiter wait{dead, a.kv.status};
    const uint32_t sbase = smem_addr(smem);
    Meta<Q8>* meta = reinterpret_cast<Meta<Q8>*>(smem + S::kMetaAt);
    uint32_t* bad_bits = reinterpret_cast<uint32_t*>(smem + S::kBad);
    auto pos_of = [&](int i) { return list.at(i0 + i); };
    float2* ml = reinterpret_cast<float2*>(smem + S::kMl);
    constexpr uint32_t kO = 256;  // tensor-memory columns: S (then P) of the tiles, then their outputs

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssuerRegs));
        if (warp == 12) {
            // ---------------- MMA issuer ----------------
            constexpr uint32_t idS = idesc_of(kRows, false), idO = idesc_of(D, true);
            bool ok = true;
            int np[kTiles] = {0, 0};  // steps of each tile so far
            for (int s = 0; s <= n && ok; ++s) {
                for (int t = 0; t < kTiles && ok; ++t) {
                    if (s > 0 && job.needs(sight, t, pos_of(s - 1))) {
                        const int item = 2 * (s - 1) + 1;
                        ok = wait(pready(t), (np[t] - 1) & 1) && wait(kvfull(item), (item / NS) & 1);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t d = tmem + kO + t * D, p = tmem + t * kRows;
                        const uint64_t v = desc_sw128(sbase + S::kRing + (item % NS) * S::kMat, S::kHalf);
                        if (elect_one()) {
#pragma unroll
                            for (int part = 0; part < S::kParts; ++part)
#pragma unroll
                                for (int k = 0; k < kRows / 16; ++k)
                                    tc_mma_f16_ts(d, p + part * 64 + k * 8, v + k * (2048 >> 4), idO,
                                                  np[t] > 1 || part > 0 || k > 0 ? 1u : 0u);
                        }
                        __syncwarp();
                    }
                    if (s < n && job.needs(sight, t, pos_of(s))) {
                        const int item = 2 * s;
                        if (np[t] == 0) ok = wait(qfull(t), 0);
                        ok = ok && wait(kvfull(item), (item / NS) & 1);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t d = tmem + t * kRows;
                        const uint64_t k0 = desc_sw128(sbase + S::kRing + (item % NS) * S::kMat, 0);
                        const uint64_t q0 = desc_sw128(sbase + t * S::kParts * S::kMat, 0);
                        if (elect_one()) {
#pragma unroll
                            for (int part = 0; part < S::kParts; ++part)
#pragma unroll
                                for (int k = 0; k < D / 16; ++k) {
                                    const uint32_t off = ((k >> 2) * S::kHalf + (k & 3) * 32) >> 4;
                                    tc_mma_f16(d, q0 + ((part * S::kMat) >> 4) + off, k0 + off, idS,
                                               part > 0 || k > 0 ? 1u : 0u);
                                }
                            tc_commit(sready(t));
                        }
                        __syncwarp();
                        ++np[t];
                    }
                }
                if (ok && elect_one()) {
                    if (s > 0) tc_commit(kvempty(2 * (s - 1) + 1));
                    if (s < n) tc_commit(kvempty(2 * s));
                    if (s == n) tc_commit(done);
                }
                __syncwarp();
            }
            if (!ok && elect_one()) tc_commit(done);  // what was issued still has to finish
            __syncwarp();
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoaderRegs));
        // ---------------- loader ----------------
        const int r = threadIdx.x - 256, w = warp - 8;
        const int hi_seen = max(hi, sight.pre - 1), lo_seen = sight.first(max(lo, 0));
        auto look = [&](int i) -> uint32_t {
            if (i >= n) return kNoRow;
            const int j = pos_of(i) + r;
            return (j <= hi_seen && (j < sight.pre || j >= lo_seen)) ? row_of(a, job.b, job.kvh, j) : kNoRow;
        };
        auto put_meta = [&](int i, uint32_t row) {
            Meta<Q8>& m = meta[i % kMeta];
            const uint32_t bits = __ballot_sync(0xffffffffu, row != kNoRow);
            if (lane == 0) m.valid[w] = bits;
            if constexpr (Q8) {
                float ks = 0.0f, vs = 0.0f;
                if (row != kNoRow) ks = a.kv.ks[row], vs = a.kv.vs[row];
                if (!(fabsf(vs) < INFINITY) && job.template mixed<PREC>(sight, pos_of(i))) {
                    vs = 0.0f;
                    atomicOr(bad_bits + (i >> 5) % kBadWords, 1u << (i & 31));
                }
                m.ks[r] = ks;
                m.vs[r] = vs;
                const float mx = fabsf(vs) < INFINITY ? fabsf(vs) : 0.0f;
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
            // All of item x's copies of this thread have landed: clean what must
            // be, and hand it over.
            auto finish = [&](int x) {
                const uint32_t slot = sbase + S::kRing + (x % NS) * S::kMat;
                if ((x & 1) && job.template mixed<PREC>(sight, pos_of(x >> 1))) {
                    bool bad = false;
#pragma unroll 4
                    for (int t = 0; t < NI; ++t) {
                        const uint32_t at = slot + chunk_at<S::kHalf>(w * 32 + t * RPI + lane / CH, lane % CH);
                        const uint4 v = lds128(at);
                        const uint4 u = make_uint4(clean16(v.x), clean16(v.y), clean16(v.z), clean16(v.w));
                        if (u.x != v.x || u.y != v.y || u.z != v.z || u.w != v.w) {
                            bad = true;
                            sts128(at, u);
                        }
                    }
                    if (bad) atomicOr(bad_bits + (x >> 6) % kBadWords, 1u << ((x >> 1) & 31));
                }
                fence_proxy_async_smem();
                mbar_arrive(kvfull(x));
            };
            for (int i = 0; i < n && ok; ++i) {
                const uint32_t row = ahead;
                ahead = look(i + 1);
                ok = __all_sync(0xffffffffu, wait(mempty(i), ((i / kMeta) & 1) ^ 1));
                if (!ok) break;
                put_meta(i, row);
                for (int part = 0; part < 2; ++part) {
                    const int x = 2 * i + part;
                    ok = __all_sync(0xffffffffu, wait(kvempty(x), ((x / NS) & 1) ^ 1));
                    if (!ok) break;
                    const uint32_t slot = sbase + S::kRing + (x % NS) * S::kMat;
                    const uint8_t* src = static_cast<const uint8_t*>(part ? a.kv.v : a.kv.k) + (lane % CH) * 16;
#pragma unroll
                    for (int t = 0; t < NI; ++t) {
                        const int rl = t * RPI + lane / CH;
                        const uint32_t rw = __shfl_sync(0xffffffffu, row, rl);
                        const bool have = rw != kNoRow;
                        cp_async16(slot + chunk_at<S::kHalf>(w * 32 + rl, lane % CH),
                                   src + (have ? static_cast<long long>(rw) * (2 * D) : 0), have);
                    }
                    cp_async_commit();
                    if (x >= LA) {
                        cp_async_wait<LA>();
                        finish(x - LA);
                    }
                }
            }
            cp_async_wait<0>();
            if (ok)
                for (int x = max(0, 2 * n - LA); x < 2 * n; ++x) finish(x);
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
                    sts128(slot + chunk_at<S::kHalf>(row, c),
                           make_uint4(codes_fp16(u[0], 0x4140), codes_fp16(u[0], 0x4342), codes_fp16(u[1], 0x4140),
                                      codes_fp16(u[1], 0x4342)));
                    sts128(slot + chunk_at<S::kHalf>(row, c + 1),
                           make_uint4(codes_fp16(u[2], 0x4140), codes_fp16(u[2], 0x4342), codes_fp16(u[3], 0x4140),
                                      codes_fp16(u[3], 0x4342)));
                }
                fence_proxy_async_smem();
                mbar_arrive(kvfull(x));
            };
            uint32_t row = ahead;
            ahead = look(1);
            if (n > 0) {
                fetch(kreg, a.kv.k, row);
                fetch(vreg, a.kv.v, row);
            }
            for (int i = 0; i < n && ok; ++i) {
                ok = __all_sync(0xffffffffu, wait(mempty(i), ((i / kMeta) & 1) ^ 1));
                if (!ok) break;
                put_meta(i, row);
                row = ahead;
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---------------- softmax of tile t, row tid ----------------
        const int t = warp >> 2, tid = threadIdx.x & 127;
        const int row = job.row0 + t * kRows + tid;
        const bool have = row < job.rows;
        const int tok = have ? row / a.group : 0, head = job.kvh * a.group + (have ? row - tok * a.group : 0);
        const int pos = job.p0 + tok;
        const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
        float mult = a.scale;
        {
            // Q: this row, fp16 as it is, fp32 as two parts of q 2^10 / E
            const T* q = static_cast<const T*>(a.q) + (job.first_tok + tok) * a.q_stride + head * D;
            const uint32_t dst = sbase + t * S::kParts * S::kMat;
            if constexpr (!PREC) {
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c)
                    sts128(dst + chunk_at<S::kHalf>(tid, c),
                           have ? *(reinterpret_cast<const uint4*>(q) + c) : make_uint4(0u, 0u, 0u, 0u));
            } else {
                float amax = 0.0f;
                if (have)
#pragma unroll 8
                    for (int c = 0; c < D / 4; ++c) {
                        const float4 v = *(reinterpret_cast<const float4*>(q) + c);
                        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                    }
                const float E = fmaxf(pow2_above(amax < INFINITY ? amax : 0.0f), 7.8886090522e-31f);  // 2^-100
                const float down = __fdiv_rn(1024.0f, E);
                mult *= E * 0.0009765625f;
#pragma unroll 2
                for (int c = 0; c < D / 8; ++c) {
                    uint4 h = make_uint4(0u, 0u, 0u, 0u), l = h;
                    if (have) {
                        const float4 x = *(reinterpret_cast<const float4*>(q) + 2 * c);
                        const float4 y = *(reinterpret_cast<const float4*>(q) + 2 * c + 1);
                        const float v[8] = {x.x * down, x.y * down, x.z * down, x.w * down,
                                            y.x * down, y.y * down, y.z * down, y.w * down};
                        uint32_t hh[4], ll[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            hh[k] = pack2(v[2 * k], v[2 * k + 1]);
                            const float2 f = unpack2(hh[k]);
                            ll[k] = pack2(v[2 * k] - f.x, v[2 * k + 1] - f.y);
                        }
                        h = make_uint4(hh[0], hh[1], hh[2], hh[3]);
                        l = make_uint4(ll[0], ll[1], ll[2], ll[3]);
                    }
                    sts128(dst + chunk_at<S::kHalf>(tid, c), h);
                    sts128(dst + S::kMat + chunk_at<S::kHalf>(tid, c), l);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(qfull(t));
        }
        const bool shaped = a.cap > 0.0f || a.slopes != nullptr;
        const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
        const float to_log2 = shaped ? 1.0f : mult * kLog2e;  // factor left for the exponent
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + t * kRows, to = tmem + lanes + kO + t * D;
        float m = -INFINITY, l = 0.0f;
        float E = 0.0f, inv_E = 0.0f;
        int steps = 0;
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            const int j0 = pos_of(i);
            ok = __all_sync(0xffffffffu, wait(mfull(i), (i / kMeta) & 1));
            if (!ok) break;
            const Meta<Q8>& md = meta[i % kMeta];
            if (!job.needs(sight, t, j0)) {
                __syncwarp();
                if (lane == 0) mbar_arrive(mempty(i));
                continue;
            }
            ok = __all_sync(0xffffffffu, wait(sready(t), steps & 1));
            if (!ok) break;
            tc_fence_after();
            float x[kRows];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, x + 32 * c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_loaded32(x + 32 * c);
            const uint4 valid = *reinterpret_cast<const uint4*>(md.valid);
            const bool whole = (valid.x & valid.y & valid.z & valid.w) == 0xFFFFFFFFu &&
                               sight.all(job.lo[t], job.hi[t], j0, j0 + kRows - 1);
            if constexpr (Q8) {
#pragma unroll
                for (int c = 0; c < kRows; c += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(md.ks + c);
                    x[c] *= k.x, x[c + 1] *= k.y, x[c + 2] *= k.z, x[c + 3] *= k.w;
                }
            }
            if (shaped) {
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int c = 0; c < kRows; ++c) x[c] = capped<PREC>(x[c] * mult, a.cap, inv_cap) * kLog2e;
                } else {
#pragma unroll
                    for (int c = 0; c < kRows; ++c) x[c] *= mult * kLog2e;
                }
                if (a.slopes) {
                    const float d0 = static_cast<float>(pos - j0);
#pragma unroll
                    for (int c = 0; c < kRows; ++c) x[c] -= slope * fabsf(d0 - static_cast<float>(c));
                }
            }
            if (!whole) {
                // positions of the step that the row sees: below `pre`, or from `a0` to `a1`
                const int pre = sight.pre - j0, a0 = sight.first(pos) - j0, a1 = pos - j0;
                const uint32_t vw[4] = {valid.x, valid.y, valid.z, valid.w};
#pragma unroll
                for (int c = 0; c < kRows; ++c) {
                    const bool see = ((vw[c >> 5] >> (c & 31)) & 1u) && (c < pre || (c >= a0 && c <= a1));
                    if (!see) x[c] = -INFINITY;
                }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kRows; c += 8)
#pragma unroll
                for (int u = 0; u < 4; ++u) tops[u] = fmaxf(tops[u], fmaxf(x[c + 2 * u], x[c + 2 * u + 1]));
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * to_log2;
            float unit = 1.0f;
            if constexpr (Q8) {
                const float4 vm = *reinterpret_cast<const float4*>(md.vmax);
                const float mx = fmaxf(fmaxf(vm.x, vm.y), fmaxf(vm.z, vm.w));
                if (mx >= E) {
                    const float e2 = pow2_above(mx);
                    unit = E / e2;  // powers of two; 0 at the first step
                    E = e2;
                    inv_E = 1.0f / E;
                }
            }
            const bool rise = top > m + kRise;
            if (__any_sync(0xffffffffu, rise) || unit != 1.0f) {
                const float mn = rise ? top : m;
                const float f = m == -INFINITY ? 1.0f : ex2(m - mn);
                m = mn;
                l *= f;
                if (steps > 0) {
                    const float fu = f * unit;
#pragma unroll
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        tmem_ld16(to + c, o);
                        tmem_wait_ld();
                        tmem_loaded16(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] *= fu;
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : kLift - m;
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t hi32[32], lo32[32];
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    float p[4];
                    float4 v = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                    if constexpr (Q8) v = *reinterpret_cast<const float4*>(md.vs + half * 64 + c);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        p[u] = ex2(fmaf(x[half * 64 + c + u], to_log2, base));
                        sums[u] += p[u];
                    }
                    if constexpr (Q8) p[0] *= v.x * inv_E, p[1] *= v.y * inv_E, p[2] *= v.z * inv_E, p[3] *= v.w * inv_E;
                    hi32[c / 2] = pack2(p[0], p[1]);
                    hi32[c / 2 + 1] = pack2(p[2], p[3]);
                    if constexpr (PREC) {
                        const float2 h0 = unpack2(hi32[c / 2]), h1 = unpack2(hi32[c / 2 + 1]);
                        lo32[c / 2] = pack2(p[0] - h0.x, p[1] - h0.y);
                        lo32[c / 2 + 1] = pack2(p[2] - h1.x, p[3] - h1.y);
                    }
                }
                tmem_st32(ts + half * 32, hi32);
                if constexpr (PREC) tmem_st32(ts + 64 + half * 32, lo32);
            }
            l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(pready(t));
                mbar_arrive(mempty(i));
            }
            ++steps;
        }
        // ---------------- output ----------------
        ok = __all_sync(0xffffffffu, wait(done, 0));
        tc_fence_after();
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const float fin = C == 1 ? (Q8 ? inv * E : inv) : (Q8 ? E : 1.0f);
        if (C > 1) ml[t * kRows + tid] = make_float2(m, l);
        bool bad = false;
        for (int k = 0; k < kBadWords; ++k) bad |= bad_bits[k] != 0;
        T* out = static_cast<T*>(a.out) + (job.first_tok + tok) * a.out_stride + head * D;
        // The other tile's products may still read the ring: its outputs go
        // over Q and the ring only once both are done (`done` covers all).
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
                    for (int j = j0; j < min(j0 + kRows, sight.n); ++j) {
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
            if (C == 1) {
                if (have) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        store_out4(out + c + k, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                }
            } else {
                // chunk (of 4 floats) spread by the row, so that a warp's rows fall on all banks
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                    sts128(sbase + (t * kRows + tid) * (D * 4) + ((((c + k) >> 2) ^ (tid & 7)) << 4),
                           make_uint4(__float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]),
                                      __float_as_uint(o[k + 3])));
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
        const int tok = row / a.group, head = job.kvh * a.group + row - tok * a.group;
        T* out = static_cast<T*>(a.out) + (job.first_tok + tok) * a.out_stride + head * D + 4 * e;
        store_out4(out, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool PREC, bool Q8>
int launch_tiles(const AttnArgs& a, long long total_rows, int max_kv, int sms, cudaStream_t st) {
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
            if (cudaFuncGetAttributes(&fa, b200q_attn_tile_kernel<D, PREC, Q8>) != cudaSuccess || fa.numRegs != 128 ||
                cudaFuncSetAttribute(b200q_attn_tile_kernel<D, PREC, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     S::kTotal) != cudaSuccess)
                return B200Q_ECUDA;
            done |= bit;
        }
    }
    // An upper bound of the blocks of rows: the lengths are on the device.
    const long long seqs = std::min<long long>(a.r.batch, total_rows / (a.few_rows + 1));
    const long long blocks = total_rows / kCtaRows + seqs;
    if (blocks <= 0) return B200Q_OK;
    const long long units = blocks * a.kv.n_kv;
    // Split the positions while the blocks leave SMs idle, four steps a CTA at least.
    int c = 1;
    while (c < kMaxCluster && units * c * 2 <= sms && max_kv >= c * 2 * 4 * kRows) c *= 2;
    if (units * c > 0x7fffffffll) return B200Q_ESHAPE;
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
    return cudaLaunchKernelEx(&cfg, b200q_attn_tile_kernel<D, PREC, Q8>, a) == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

}  // namespace

int launch_attn_tiles(const AttnArgs& a, int hd, bool fp32, bool q8, long long total_rows, int max_kv, int sms,
                      cudaStream_t st) {
#define B200Q_TILES(D)                                                                 \
    (fp32 ? (q8 ? launch_tiles<D, true, true>(a, total_rows, max_kv, sms, st)          \
                : launch_tiles<D, true, false>(a, total_rows, max_kv, sms, st))        \
          : (q8 ? launch_tiles<D, false, true>(a, total_rows, max_kv, sms, st)         \
                : launch_tiles<D, false, false>(a, total_rows, max_kv, sms, st)))
    return hd == 128 ? B200Q_TILES(128) : B200Q_TILES(64);
#undef B200Q_TILES
}

}  // namespace b200q
