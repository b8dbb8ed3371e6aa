// Attention of a few query rows per sequence over a paged cache (decode
// steps, drafted tokens): bound by the cache's bytes.
//
// The query heads that share a kv head, of one or several tokens, are the
// rows of one matrix product: row r of a sequence is token r / group, head
// r % group. 16 rows (fp16) fill the M of mma.m16n8k16; fp32 rows come 8 at a
// time, each as two fp16 parts hi + lo of its value (22 bits, after scaling
// the row by a power of two) in rows r and r + 8, so that one product gives
// both and their sum stays in a lane. The softmax weights of fp32 rows are
// split in the same way before the second product. So are those of fp16 rows
// where no sequence has more than 8 of them (a decode step): the upper half of
// the product would stay empty, and a lane has one row's exponentials instead
// of two: 64 rows of 64/8 heads over 100-8000 Q8 positions 135 -> 125 us, one
// row of 32/8 heads over 2048 9.5 -> 8.6, and the error against 64 bits 1.0
// times the plain form's instead of 1.4 times.
//
// A warp takes every (4 C)-th tile of 16 or 32 positions through a cp.async ring of
// its own and keeps a running maximum, sum and output: the warps share
// nothing until the end, so no barrier stands between the loads. The CTAs of
// a cluster (C, up to 16) share one block of rows; their partial outputs are
// joined in shared memory over the cluster, in a fixed order, without a
// workspace, a counter or a second launch. The page of the next tile to load
// is looked up one tile ahead of its loads.
//
// Q8 rows enter as their integer codes, exact in fp16; a key's scale
// multiplies its score, a value's scale its softmax weight, relative to a
// power of two E above the scales that its row has seen so far, so that the
// weight in fp16 neither over- nor underflows. Weights are kept 2^10 above 1 for
// the same reason.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn_ragged.cuh"
#include "internal.h"

namespace b200q {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxCluster = 16;  // beyond 8 only where the device allows it
constexpr int kPlainSum = 32768;  // positions of a warp whose sum the tensor cores keep: 2^-12.2 of it are lost
constexpr float kRise = 4.0f;    // a row's reference maximum follows once exceeded by this (log2)
constexpr float kLift = 10.0f;   // weights are 2^(score - maximum + kLift): at most 2^14 in fp16

template <int D, bool SPLIT, bool Q8>
struct Few {
    static constexpr int R = SPLIT ? 8 : 16;               // rows per block
    static constexpr int RB = Q8 ? D : 2 * D;             // bytes per stored row
    static constexpr int CH = RB / 16;                    // 16-byte chunks per row
    // Positions per tile: more of them give a warp more independent products;
    // rows of 256 bytes leave room for 16 only.
    static constexpr int kTile = RB == 256 ? 16 : 32;
    static constexpr int kScales = Q8 ? 2 * kTile * 4 : 0;  // the tile's key and value scales
    static constexpr int kStage = 2 * kTile * RB + kScales;
    static constexpr int NS = RB == 64 ? 3 : 2;
    static constexpr int kRing = NS * kStage;
    static constexpr int kPart = R * D * 4;               // a warp's output, in its ring after the loop
    static constexpr int kWarpBytes = kRing > kPart ? kRing : kPart;
    static constexpr int kTotal = kWarps * kWarpBytes + kWarps * R * 8 + R * 8;
};

// Resident CTAs per SM, which registers and rings are cut to: twelve warps with
// one tile on its way each beat eight with two (64 sequences of 100-8000
// positions in Q8 pages 148 -> 134 us, two of 60-120 thousand in fp16 pages 198
// -> 156; four times eight rows of 2000 positions 17 -> 20).
constexpr int kCtasPerSm = 3;

__device__ __forceinline__ void ldsm4(uint32_t (&v)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&v)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The tensor cores cut an accumulator off with each product: 0.11 x 2^-24 of a
// sum of one sign per position. fp32 rows add the products themselves: their
// error at 8000 positions is 3e-7 instead of 6e-6, for 1 to 3 percent of the time
// (one row of 32/8 heads over 2048 positions 9.0 -> 9.2 us, 64 over 4000 175 -> 177;
// Q8, the two parts joined at once, 110 -> 112; apart they spilled: 133).
// fp16 rows, which it would cost 5 percent, keep the accumulator for up to kPlainSum
// positions a warp.
__device__ __forceinline__ void add4(float (&d)[4], const float (&t)[4]) {
    const float2 x = add2(make_float2(d[0], d[1]), make_float2(t[0], t[1]));
    const float2 y = add2(make_float2(d[2], d[3]), make_float2(t[2], t[3]));
    d[0] = x.x, d[1] = x.y, d[2] = y.x, d[3] = y.y;
}
// The product's two parts (rows g and g + 8) added to d's first two.
__device__ __forceinline__ void add_parts(float (&d)[4], const float (&t)[4]) {
    const float2 p = add2(make_float2(t[0], t[1]), make_float2(t[2], t[3]));
    const float2 x = add2(make_float2(d[0], d[1]), p);
    d[0] = x.x, d[1] = x.y;
}
// d plus the product. OWN: the product gets an accumulator of its own and is
// added to d in fp32; else the tensor core adds it, and cuts the sum off.
template <bool OWN>
__device__ __forceinline__ void mma_onto(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (OWN) {
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma16(t, a, b0, b1);
        add4(d, t);
    } else {
        mma16(d, a, b0, b1);
    }
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
    return v;
}

__device__ __forceinline__ bool not_finite16(uint32_t h) {
    return (h & 0x7C00u) == 0x7C00u || (h & 0x7C000000u) == 0x7C000000u;
}

// Where 16-byte chunk c of row r of a tile lies in its row: spread so that
// the fragment reads below touch all banks (fp16: ldmatrix reads the same
// chunk of 8 rows; Q8: 8 lanes read 4 chunks of 2 rows of keys, 2 chunks of 4
// even rows of values).
template <int D, bool Q8>
__device__ __forceinline__ int k_chunk(int r, int c) {
    if constexpr (!Q8) return c ^ (r & 7);
    return D == 128 ? c ^ ((r & 1) << 2) : c;
}
template <int D, bool Q8>
__device__ __forceinline__ int v_chunk(int r, int c) {
    if constexpr (!Q8) return c ^ (r & 7);
    return D == 128 ? c ^ (r & 6) : c ^ ((r >> 1) & 3);
}

template <int D, bool FP32, bool SPLIT, bool Q8>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) b200q_attn_few_kernel(const AttnArgs a) {
    using F = Few<D, SPLIT, Q8>;
    using T = typename std::conditional<FP32, float, __half>::type;
    static_assert(SPLIT || !FP32, "fp32 rows have two parts");
    constexpr int R = F::R, KS = D / 16, NB = D / 8, NS = F::NS, kTile = F::kTile;
    constexpr int NK = kTile / 8;  // blocks of 8 positions
    constexpr uint32_t kAll = kTile == 32 ? 0xFFFFFFFFu : 0xFFFFu;
    // o holds the sum of the two parts (in o[.][0] and o[.][1]) where products are
    // added to it in fp32 and no value is infinite by itself, but by its scale.
    constexpr bool kJoined = Q8 && FP32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t present[kWarps][8];  // per stage: which of its positions have a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float2* ml = reinterpret_cast<float2*>(smem + kWarps * F::kWarpBytes);  // [kWarps][R] max, sum
    float2* ml_cta = ml + kWarps * R;                                       // [R]
    const uint32_t ring = smem_addr(smem) + warp * F::kWarpBytes;
    const uint32_t C = cluster_size(), rank = cluster_rank();
    int unit = blockIdx.x / C;
    const int rb = unit % a.row_blocks;
    unit /= a.row_blocks;
    const int kvh = unit % a.kv.n_kv, b = unit / a.kv.n_kv;
    griddep_launch_dependents();
    griddep_wait();
    const int2 rr = seq_rows(a.r, b);
    const int rows = (rr.y - rr.x) * a.group;
    const int r0 = rb * R;
    if (rows > a.few_rows || r0 >= rows) return;  // the same for the whole cluster
    const Sight s = sight_of(a, b);
    if (threadIdx.x == 0 && s.n > s.limit) flag_bad_page(a.kv);
    const int nr = min(R, rows - r0);
    const int p0 = s.n - (rr.y - rr.x);
    const int p_lo = p0 + r0 / a.group, p_hi = p0 + (r0 + nr - 1) / a.group;

    // This lane's rows: g, and without low parts g + 8.
    constexpr int NR = SPLIT ? 1 : 2;
    int pos[NR];
    float slope[NR], mult[NR];
    uint32_t qa[KS][4];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = r0 + g + 8 * i;
        const bool have = r < rows;
        const int tok = have ? div_by(r, a.group_mul, a.group_shift) : 0, head = kvh * a.group + (have ? r - tok * a.group : 0);
        pos[i] = p0 + tok;
        slope[i] = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
        const T* q = static_cast<const T*>(a.q) + (rr.x + tok) * a.q_stride + head * D;
        // Elements of k-step ks that this lane holds: the fragment's own order
        // for fp16 rows; for Q8 four consecutive ones, so that a lane reads 16
        // codes of a key for four steps at once (any order does, if the keys'
        // is the same).
        float v[KS][4];
        float amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int e0 = Q8 ? (ks >> 2) * 64 + c * 16 + (ks & 3) * 4 : ks * 16 + 2 * c;
            const int e1 = Q8 ? e0 + 2 : e0 + 8;
            if constexpr (FP32) {
                const float2 x = have ? *reinterpret_cast<const float2*>(q + e0) : make_float2(0.0f, 0.0f);
                const float2 y = have ? *reinterpret_cast<const float2*>(q + e1) : make_float2(0.0f, 0.0f);
                v[ks][0] = x.x, v[ks][1] = x.y, v[ks][2] = y.x, v[ks][3] = y.y;
#pragma unroll
                for (int t = 0; t < 4; ++t) amax = fmaxf(amax, fabsf(v[ks][t]));
            } else {
                qa[ks][i] = have ? *reinterpret_cast<const uint32_t*>(q + e0) : 0u;
                qa[ks][2 + i] = have ? *reinterpret_cast<const uint32_t*>(q + e1) : 0u;
                if constexpr (SPLIT) qa[ks][1] = qa[ks][3] = 0u;  // fp16 as it is
            }
        }
        mult[i] = a.scale;
        if constexpr (FP32) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // |q| / E below 1: parts of q 2^10 / E, the smallest of them 2^-34 of the largest element
            const float E = fmaxf(pow2_above(amax < INFINITY ? amax : 0.0f), 7.8886090522e-31f);  // 2^-100
            const float down = __fdiv_rn(1024.0f, E);
            mult[i] *= E * 0.0009765625f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float x = v[ks][2 * t] * down, y = v[ks][2 * t + 1] * down;
                    const uint32_t hi = pack2(x, y);
                    const float2 h = unpack2(hi);
                    qa[ks][2 * t] = hi;
                    qa[ks][2 * t + 1] = pack2(x - h.x, y - h.y);
                }
            }
        }
    }
    const bool shaped = a.cap > 0.0f || a.slopes != nullptr;
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    if (!shaped) {
#pragma unroll
        for (int i = 0; i < NR; ++i) mult[i] *= kLog2e;
    }

    float o[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) m[i] = -INFINITY, l[i] = 0.0f;
    // Q8: the power of two that a row's o is in units of, above the scales that the
    // row has seen in this warp's tiles; the warp's least.
    float E[NR], least = 0.0f;
#pragma unroll
    for (int i = 0; i < NR; ++i) E[i] = 0.0f;

    const TileList<kTile> tiles(s, p_lo, p_hi);
    const int stride = kWarps * static_cast<int>(C);
    const int first = static_cast<int>(rank) * kWarps + warp;
    const int n_mine = p_hi < 0 || tiles.count <= first ? 0 : (tiles.count - first + stride - 1) / stride;
    const int hi_seen = s.last(p_hi), lo_seen = s.first(max(p_lo, 0));

    // Position lane % kTile of my tile i: its pool row, if some row of the block sees it.
    auto look = [&](int i) -> uint32_t {
        if (i >= n_mine) return kNoRow;
        const int j = tiles.at(first + i * stride) + lane % kTile;
        return (j <= hi_seen && (j < s.pre || j >= lo_seen)) ? row_of(a, b, kvh, j) : kNoRow;
    };
    uint32_t ahead = look(0);  // row of the next tile to load
    auto load = [&](int i) {
        const uint32_t rowi = ahead;
        ahead = look(i + 1);
        if (i < n_mine) {
            const uint32_t st = ring + (i % NS) * F::kStage;
            constexpr int RPI = 32 / F::CH;  // rows a warp copies at once
            const int ch = lane % F::CH;
#pragma unroll
            for (int t = 0; t < kTile / RPI; ++t) {
                const int r = t * RPI + lane / F::CH;
                const uint32_t row = __shfl_sync(0xffffffffu, rowi, r);
                const bool ok = row != kNoRow;
                const long long off = ok ? static_cast<long long>(row) * F::RB + ch * 16 : 0;
                cp_async16(st + r * F::RB + k_chunk<D, Q8>(r, ch) * 16, static_cast<const uint8_t*>(a.kv.k) + off, ok);
                cp_async16(st + (kTile + r) * F::RB + v_chunk<D, Q8>(r, ch) * 16,
                           static_cast<const uint8_t*>(a.kv.v) + off, ok);
            }
            if constexpr (Q8) {
                static_assert(!Q8 || kTile == 32, "a lane per position");
                const bool ok = rowi != kNoRow;
                cp_async4(st + 2 * kTile * F::RB + lane * 4, a.kv.ks + (ok ? rowi : 0), ok);
                cp_async4(st + 2 * kTile * F::RB + (kTile + lane) * 4, a.kv.vs + (ok ? rowi : 0), ok);
            }
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, rowi != kNoRow) & kAll;
        if (lane == 0) present[warp][i % NS] = bits;
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) load(i);

    for (int i = 0; i < n_mine; ++i) {
        cp_async_wait<NS - 2>();
        __syncwarp();
        load(i + NS - 1);  // into the stage that the previous tile left
        const uint32_t st = ring + (i % NS) * F::kStage;
        const uint32_t kt = st, vt = st + kTile * F::RB;
        const uint32_t bits = present[warp][i % NS];
        const int j0 = tiles.at(first + i * stride);
        // ---- scores: S[rows][positions], with 16 positions in two halves of the
        // head, so that four chains of products run side by side
        constexpr int HV = NK == 2 ? 2 : 1;
        float sc[NK][4];
        {
            float acc[HV][NK][4];
#pragma unroll
            for (int hv = 0; hv < HV; ++hv)
#pragma unroll
                for (int nb = 0; nb < NK; ++nb) acc[hv][nb][0] = acc[hv][nb][1] = acc[hv][nb][2] = acc[hv][nb][3] = 0.0f;
            if constexpr (!Q8) {
#pragma unroll
                for (int ks = 0; ks < KS / HV; ks += 2)
#pragma unroll
                    for (int nb = 0; nb < NK; ++nb)
#pragma unroll
                        for (int hv = 0; hv < HV; ++hv) {
                            uint32_t k4[4];
                            const int r = nb * 8 + (lane & 7), kk = hv * (KS / 2) + ks;
                            ldsm4(k4, kt + r * F::RB + k_chunk<D, Q8>(r, kk * 2 + (lane >> 3)) * 16);
                            mma16(acc[hv][nb], qa[kk], k4[0], k4[1]);
                            mma16(acc[hv][nb], qa[kk + 1], k4[2], k4[3]);
                        }
            } else {
#pragma unroll
                for (int kq = 0; kq < D / 64; ++kq) {
                    uint4 w[NK];
#pragma unroll
                    for (int nb = 0; nb < NK; ++nb) {
                        const int r = nb * 8 + g;
                        w[nb] = lds128(kt + r * F::RB + k_chunk<D, Q8>(r, kq * 4 + c) * 16);
                    }
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int nb = 0; nb < NK; ++nb) {
                            const uint32_t u =
                                (t == 0 ? w[nb].x : t == 1 ? w[nb].y : t == 2 ? w[nb].z : w[nb].w) ^ 0x80808080u;
                            mma16(acc[0][nb], qa[kq * 4 + t], codes_fp16(u, 0x4140), codes_fp16(u, 0x4342));
                        }
                }
            }
#pragma unroll
            for (int nb = 0; nb < NK; ++nb)
#pragma unroll
                for (int v = 0; v < 4; ++v) sc[nb][v] = HV == 2 ? acc[0][nb][v] + acc[HV - 1][nb][v] : acc[0][nb][v];
        }
        // ---- exponents (log2); position of value v of block nb: j0 + 8 nb + 2 c + (v & 1)
        constexpr int NX = 2 * NK;
        float x[NR][NX];
#pragma unroll
        for (int nb = 0; nb < NK; ++nb) {
            float ks0 = 1.0f, ks1 = 1.0f;
            if constexpr (Q8) {
                const float2 k2 = lds_f2(st + 2 * kTile * F::RB + (nb * 8 + 2 * c) * 4);
                ks0 = k2.x, ks1 = k2.y;
            }
            if constexpr (FP32) {
                x[0][2 * nb] = (sc[nb][0] + sc[nb][2]) * ks0;
                x[0][2 * nb + 1] = (sc[nb][1] + sc[nb][3]) * ks1;
            } else {
                x[0][2 * nb] = sc[nb][0] * ks0, x[0][2 * nb + 1] = sc[nb][1] * ks1;
                if constexpr (!SPLIT)
                    x[NR - 1][2 * nb] = sc[nb][2] * ks0, x[NR - 1][2 * nb + 1] = sc[nb][3] * ks1;
            }
        }
        const bool whole = bits == kAll && s.all(p_lo, p_hi, j0, j0 + kTile - 1);
#pragma unroll
        for (int i2 = 0; i2 < NR; ++i2) {
#pragma unroll
            for (int v = 0; v < NX; ++v) x[i2][v] *= mult[i2];
            if (shaped) {
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int v = 0; v < NX; v += 2) {
                        const float2 z = mul2(make_float2(x[i2][v], x[i2][v + 1]), both(inv_cap));
                        const float2 near = tanh_near<true>(z);
                        x[i2][v] = a.cap * (fabsf(z.x) > 1.0f ? tanh_far(z.x) : near.x);
                        x[i2][v + 1] = a.cap * (fabsf(z.y) > 1.0f ? tanh_far(z.y) : near.y);
                    }
                }
#pragma unroll
                for (int v = 0; v < NX; ++v) {
                    const int j = j0 + 8 * (v >> 1) + 2 * c + (v & 1);
                    x[i2][v] = x[i2][v] * kLog2e - slope[i2] * fabsf(static_cast<float>(pos[i2] - j));
                }
            }
            if (!whole) {
#pragma unroll
                for (int v = 0; v < NX; ++v) {
                    const int jj = 8 * (v >> 1) + 2 * c + (v & 1);
                    if (!((bits >> jj) & 1u) || !s.sees(pos[i2], j0 + jj)) x[i2][v] = -INFINITY;
                }
            }
        }
        // ---- the running maximum, raised only when a row passes it by kRise
        float top[NR];
        bool rise = false;
#pragma unroll
        for (int i2 = 0; i2 < NR; ++i2) {
            top[i2] = fmaxf(fmaxf(x[i2][0], x[i2][1]), fmaxf(x[i2][2], x[i2][3]));
#pragma unroll
            for (int v = 4; v < NX; ++v) top[i2] = fmaxf(top[i2], x[i2][v]);
            top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 1));
            top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 2));
            rise |= top[i2] > m[i2] + kRise;
        }
        float unit[NR];  // Q8: change of o's unit
#pragma unroll
        for (int i2 = 0; i2 < NR; ++i2) unit[i2] = 1.0f;
        float vs[NX];
        if constexpr (Q8) {
            const float mine = fabsf(__uint_as_float(lds32(st + 2 * kTile * F::RB + (kTile + lane) * 4)));
            const float mx = mine < INFINITY ? mine : 0.0f;
#pragma unroll
            for (int nb = 0; nb < NK; ++nb) {
                const float2 v2 = lds_f2(st + 2 * kTile * F::RB + (kTile + 8 * nb + 2 * c) * 4);
                vs[2 * nb] = v2.x, vs[2 * nb + 1] = v2.y;
            }
            if (__any_sync(0xffffffffu, mx >= least)) {
                const float all = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
                least = INFINITY;
#pragma unroll
                for (int i2 = 0; i2 < NR; ++i2) {
                    float most = all;
                    if (!whole) {  // of the positions that the row sees: others' would push its weights below fp16
                        most = 0.0f;
#pragma unroll
                        for (int v = 0; v < NX; ++v) {
                            const float y = x[i2][v] == -INFINITY ? 0.0f : fabsf(vs[v]);
                            most = y < INFINITY ? fmaxf(most, y) : most;
                        }
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    }
                    if (most >= E[i2]) {
                        const float e2 = fminf(pow2_above(most), 8.5070591730e37f);  // 2^126
                        unit[i2] = E[i2] / e2;  // both powers of two (0 at the first tile, where o is 0)
                        E[i2] = e2;
                        rise = true;
                    }
                    least = fminf(least, E[i2]);
                }
                least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
            }
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int i2 = 0; i2 < NR; ++i2) {
                const float mn = top[i2] > m[i2] + kRise ? top[i2] : m[i2];
                const float f = m[i2] == -INFINITY ? 1.0f : ex2(m[i2] - mn);
                m[i2] = mn;
                l[i2] *= f;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int v = 0; v < (kJoined ? 2 : 4); ++v) o[n][v] *= f * unit[i2];
                    } else {
                        o[n][2 * i2] *= f * unit[i2];
                        o[n][2 * i2 + 1] *= f * unit[i2];
                    }
                }
            }
        }
        // ---- weights, a fragment per 16 positions
        uint32_t pa[kTile / 16][4];
#pragma unroll
        for (int i2 = 0; i2 < NR; ++i2) {
            const float base = m[i2] == -INFINITY ? 0.0f : kLift - m[i2];
            // (of a power of two, 2^126 at most)
            const float inv_E = __int_as_float(0x7F000000 - __float_as_int(E[i2]));
#pragma unroll
            for (int f = 0; f < kTile / 16; ++f) {
                float p[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    p[v] = ex2(x[i2][4 * f + v] + base);
                    l[i2] += p[v];
                    if constexpr (Q8) p[v] = x[i2][4 * f + v] == -INFINITY ? 0.0f : p[v] * (vs[4 * f + v] * inv_E);
                }
                if constexpr (SPLIT) {
                    pa[f][0] = pack2(p[0], p[1]);
                    pa[f][2] = pack2(p[2], p[3]);
                    const float2 h0 = unpack2(pa[f][0]), h1 = unpack2(pa[f][2]);
                    float low[4] = {p[0] - h0.x, p[1] - h0.y, p[2] - h1.x, p[3] - h1.y};
                    if constexpr (kJoined) {  // an infinity is the upper part's alone
#pragma unroll
                        for (int v = 0; v < 4; ++v) low[v] = fabsf(p[v]) < INFINITY ? low[v] : 0.0f;
                    }
                    pa[f][1] = pack2(low[0], low[1]);
                    pa[f][3] = pack2(low[2], low[3]);
                } else {
                    pa[f][i2] = pack2(p[0], p[1]);
                    pa[f][2 + i2] = pack2(p[2], p[3]);
                }
            }
        }
        if constexpr (!Q8) {
            // Rows of the block see different positions of this tile: a value
            // that is not finite must reach only the rows that see it, so it is
            // added to theirs here and leaves the product.
            if (!whole && p_lo != p_hi) {
                uint32_t bad = 0;
#pragma unroll 1
                for (int t = lane; t < kTile * F::CH; t += 32) {
                    const uint4 w = lds128(vt + t * 16);
                    if (not_finite16(w.x) || not_finite16(w.y) || not_finite16(w.z) || not_finite16(w.w))
                        bad |= 1u << (t / F::CH);
                }
                bad = __reduce_or_sync(0xffffffffu, bad);
                while (bad) {
                    const int jj = __ffs(bad) - 1;
                    bad &= bad - 1;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const uint32_t w = lds32(vt + jj * F::RB + v_chunk<D, Q8>(jj, n) * 16 + c * 4);
                        if (!not_finite16(w)) continue;
                        const float2 f = unpack2(w);
#pragma unroll
                        for (int i2 = 0; i2 < NR; ++i2) {
                            if (!s.sees(pos[i2], j0 + jj)) continue;
                            if ((w & 0x7C00u) == 0x7C00u) o[n][2 * i2] += f.x;
                            if ((w & 0x7C000000u) == 0x7C000000u) o[n][2 * i2 + 1] += f.y;
                        }
                    }
                    __syncwarp();
                    for (int t = lane; t < F::RB / 4; t += 32) {
                        uint32_t w = lds32(vt + jj * F::RB + t * 4);
                        if ((w & 0x7C00u) == 0x7C00u) w &= 0xFFFF0000u;
                        if ((w & 0x7C000000u) == 0x7C000000u) w &= 0x0000FFFFu;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(vt + jj * F::RB + t * 4), "r"(w) : "memory");
                    }
                    __syncwarp();
                }
            }
        }
        // ---- O += P V
        if constexpr (kJoined) {
            // As below, but two words of the values at a time, so that both fragments'
            // products share an accumulator.
            constexpr int NF = kTile / 16;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                uint32_t wv[NF][4][2];
#pragma unroll
                for (int f = 0; f < NF; ++f)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int r = 2 * c + (t & 1) + 8 * (t >> 1);
                        const int at = D == 128 ? v_chunk<D, Q8>(r, g) * 16 + h * 8
                                                : v_chunk<D, Q8>(r, g >> 1) * 16 + (g & 1) * 8;
                        const uint2 w = lds64(vt + (f * 16 + r) * F::RB + at);
                        wv[f][t][0] = w.x ^ 0x80808080u, wv[f][t][1] = w.y ^ 0x80808080u;
                    }
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint32_t sel = hf ? 0x7362u : 0x5140u;
                        float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int f = 0; f < NF; ++f) {
                            const uint32_t b0 = __byte_perm(wv[f][0][w], wv[f][1][w], sel);
                            const uint32_t b1 = __byte_perm(wv[f][2][w], wv[f][3][w], sel);
                            mma16(s0, pa[f], codes_fp16(b0, 0x4140), codes_fp16(b1, 0x4140));
                            mma16(s1, pa[f], codes_fp16(b0, 0x4342), codes_fp16(b1, 0x4342));
                        }
                        add_parts(o[4 * (2 * h + w) + 2 * hf], s0);
                        add_parts(o[4 * (2 * h + w) + 2 * hf + 1], s1);
                    }
            }
            continue;
        }
#pragma unroll
        for (int f = 0; f < kTile / 16; ++f) {
            const uint32_t vf = vt + f * 16 * F::RB;
            if constexpr (!Q8) {
#pragma unroll
                for (int n = 0; n < NB; n += 2) {
                    uint32_t v4[4];
                    const int r = (lane & 7) + 8 * ((lane >> 3) & 1);
                    ldsm4t(v4, vf + r * F::RB + v_chunk<D, Q8>(r, n + (lane >> 4)) * 16);
                    mma_onto<FP32>(o[n], pa[f], v4[0], v4[1]);
                    mma_onto<FP32>(o[n + 1], pa[f], v4[2], v4[3]);
                }
            } else {
                // Block n, column g: element g * NB + n, so that a lane's elements of
                // a value are consecutive bytes.
                constexpr int W = D / 32;  // 32-bit words per lane and value
                uint32_t wv[4][W];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int r = 2 * c + (t & 1) + 8 * (t >> 1);
                    if constexpr (D == 128) {
                        const uint4 w = lds128(vf + r * F::RB + v_chunk<D, Q8>(r, g) * 16);
                        wv[t][0] = w.x, wv[t][1] = w.y, wv[t][W - 2] = w.z, wv[t][W - 1] = w.w;
                    } else {
                        const uint32_t ad = vf + r * F::RB + v_chunk<D, Q8>(r, g >> 1) * 16 + (g & 1) * 8;
                        wv[t][0] = lds32(ad), wv[t][1] = lds32(ad + 4);
                    }
#pragma unroll
                    for (int w = 0; w < W; ++w) wv[t][w] ^= 0x80808080u;
                }
#pragma unroll
                for (int w = 0; w < W; ++w) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint32_t sel = hf ? 0x7362u : 0x5140u;
                        const uint32_t b0 = __byte_perm(wv[0][w], wv[1][w], sel);
                        const uint32_t b1 = __byte_perm(wv[2][w], wv[3][w], sel);
                        mma16(o[4 * w + 2 * hf], pa[f], codes_fp16(b0, 0x4140), codes_fp16(b1, 0x4140));
                        mma16(o[4 * w + 2 * hf + 1], pa[f], codes_fp16(b0, 0x4342), codes_fp16(b1, 0x4342));
                    }
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- join the warps of the CTA, then the CTAs of the cluster
    float* part = reinterpret_cast<float*>(smem + warp * F::kWarpBytes);  // [R][D]
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (c == 0) ml[warp * R + g + 8 * i] = make_float2(m[i], l[i]);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int col = 2 * c + v;
                const int e = Q8 ? col * NB + n : n * 8 + col;
                // (the low parts of weights turn an infinite value into NaN: leave them out then)
                const float val = !SPLIT    ? o[n][2 * i + v]
                                  : kJoined ? o[n][v]
                                            : o[n][v] + (fabsf(o[n][2 + v]) < INFINITY ? o[n][2 + v] : 0.0f);
                part[(g + 8 * i) * D + e] = Q8 ? val * E[i] : val;
            }
        }
    }
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(smem);
    constexpr int kItems = R * D / 4;
    auto put = [&](int r, int e, float4 v, float lsum) {
        const int row = r0 + r;
        if (r >= nr) return;
        const float inv = lsum > 0.0f || lsum != lsum ? 1.0f / lsum : 0.0f;
        const int tok = div_by(row, a.group_mul, a.group_shift), head = kvh * a.group + row - tok * a.group;
        T* out = static_cast<T*>(a.out) + (rr.x + tok) * a.out_stride + head * D + e;
        store_out4(out, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    };
    for (int it = threadIdx.x; it < kItems; it += kWarps * 32) {
        const int r = it / (D / 4), e = it % (D / 4) * 4;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * R + r].x);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 t = ml[w * R + r];
            const float4 v = *reinterpret_cast<const float4*>(parts + w * (F::kWarpBytes / 4) + r * D + e);
            const float f = t.x == -INFINITY ? (t.y == 0.0f ? 0.0f : 1.0f) : ex2(t.x - M);
            if (f == 0.0f && t.y == 0.0f) continue;
            L += t.y * f;
            acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
        if (C == 1) {
            put(r, e, acc, L);
        } else {
            *reinterpret_cast<float4*>(smem + (r * D + e) * 4) = acc;  // over warp 0's, read by this thread only
            if (e == 0) ml_cta[r] = make_float2(M, L);
        }
    }
    if (C == 1) return;
    cluster_sync();
    for (int it = rank * kWarps * 32 + threadIdx.x; it < kItems; it += C * kWarps * 32) {
        const int r = it / (D / 4), e = it % (D / 4) * 4;
        if (r >= nr) continue;
        float2 t[kMaxCluster];
        float4 v[kMaxCluster];
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= static_cast<int>(C)) break;
            t[k] = ld_peer2(peer_addr(smem_addr(ml_cta + r), k));
            v[k] = ld_peer4(peer_addr(smem_addr(smem) + (r * D + e) * 4, k));
            M = fmaxf(M, t[k].x);
        }
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k >= static_cast<int>(C)) break;
            if (t[k].x == -INFINITY && t[k].y == 0.0f) continue;
            const float f = ex2(t[k].x - M);
            L += t[k].y * f;
            acc.x += v[k].x * f, acc.y += v[k].y * f, acc.z += v[k].z * f, acc.w += v[k].w * f;
        }
        put(r, e, acc, L);
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool FP32, bool SPLIT, bool Q8>
int launch_few(const AttnArgs& a0, int max_rows, int max_kv, int sms, cudaStream_t st) {
    using F = Few<D, SPLIT, Q8>;
    static_assert(F::kTotal <= 226 * 1024 / kCtasPerSm - 1024, "resident CTAs");
    AttnArgs a = a0;
    a.row_blocks = (max_rows + F::R - 1) / F::R;
    static std::mutex mu;
    static uint64_t done = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ECUDA;
    {
        std::lock_guard<std::mutex> lk(mu);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (!(done & bit)) {
            if (cudaFuncSetAttribute(b200q_attn_few_kernel<D, FP32, SPLIT, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     F::kTotal) != cudaSuccess ||
                cudaFuncSetAttribute(b200q_attn_few_kernel<D, FP32, SPLIT, Q8>, cudaFuncAttributeNonPortableClusterSizeAllowed,
                                     1) != cudaSuccess)
                return B200Q_ECUDA;
            done |= bit;
        }
    }
    const long long units = static_cast<long long>(a.r.batch) * a.kv.n_kv * a.row_blocks;
    const int c = few_split(units, max_kv, sms);
    if (units * c > 0x7fffffffll) return B200Q_ESHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * c));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = F::kTotal;
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
    cudaError_t e = cudaLaunchKernelEx(&cfg, b200q_attn_few_kernel<D, FP32, SPLIT, Q8>, a);
    if (e != cudaSuccess && c > 8) {  // no room for clusters of 16 (a partitioned device): the portable size
        cudaGetLastError();
        attr[0].val.clusterDim.x = 8;
        cfg.gridDim.x = static_cast<unsigned>(units * 8);
        e = cudaLaunchKernelEx(&cfg, b200q_attn_few_kernel<D, FP32, SPLIT, Q8>, a);
    }
    return e == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

}  // namespace

int few_slots(int sms) { return sms * kCtasPerSm; }

int few_block_rows(bool fp32, int max_rows) { return fp32 || max_rows <= 8 ? 8 : 16; }

// CTAs per block of rows: as many as one wave holds while the blocks leave SMs
// idle, two where they fill more than half a wave (ragged lengths even out over
// the halves), and about 64 positions a warp. Measured at 4 x 8 rows of 2000
// positions: 17 us for one wave, 24 for two; 64 sequences of 100-8000: 191, 175,
// 186 us for 1, 2, 4. More than 8 only up to three quarters of a wave: larger
// clusters do not fill the GPCs (24 of 16 took 36 us at 8000 positions, of 13 23),
// or for sums of more than kPlainSum positions a warp.
int few_split(long long units, int max_kv, int sms) {
    const long long slots = few_slots(sms);
    long long c = std::max<long long>(slots / units, 2);
    if (c > 8) c = std::max<long long>(8, std::min<long long>(kMaxCluster, slots * 3 / 4 / units));
    c = std::max(c, std::min<long long>(kMaxCluster, (max_kv + kWarps * kPlainSum - 1ll) / (kWarps * kPlainSum)));
    return static_cast<int>(std::max<long long>(1, std::min<long long>(c, (max_kv + kWarps * 64 - 1) / (kWarps * 64))));
}

int launch_attn_few(const AttnArgs& a, int hd, bool fp32, bool q8, int max_rows, int max_kv, int sms, cudaStream_t st) {
#define B200Q_FEW3(D, FP32, SPLIT)                                             \
    (q8 ? launch_few<D, FP32, SPLIT, true>(a, max_rows, max_kv, sms, st) \
        : launch_few<D, FP32, SPLIT, false>(a, max_rows, max_kv, sms, st))
    const bool split = few_block_rows(fp32, max_rows) == 8;
#define B200Q_FEW(D) (fp32 ? B200Q_FEW3(D, true, true) : split ? B200Q_FEW3(D, false, true) : B200Q_FEW3(D, false, false))
    return hd == 128 ? B200Q_FEW(128) : B200Q_FEW(64);
#undef B200Q_FEW
#undef B200Q_FEW3
}

}  // namespace b200q
