// Rotary positions and paged-cache appends for batches of sequences of
// different lengths, and the host side of the ragged operators.
//
// Angles. Pair p of a row at position pos turns by pos * f_p radians. In fp32
// the product loses the phase of far positions (at pos = 1e6 its last bit is
// 0.06 rad), so the table holds f_p / (2 pi) as a 64-bit fraction of a turn
// and the kernels form pos * turn modulo 2^64: the whole turns drop out of
// the product exactly and what is left is off by at most pos * 2^-63 turns
// (the table's rounding, and that of the 64-bit mantissas it is computed in).
// The fraction's nearest quarter turn is taken out as an integer too, so that
// sincospi sees at most an eighth of a turn, with all 24 bits of it.
//
// Q8 keys are rotated in fp64: the page's quantizer rounds the fp32 row to
// codes, and a key that is off by an fp32 rounding would fall on the other
// side of a border of two codes now and then (2e-5 of all codes measured at
// 2^-24 relative).
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "internal.h"
#include "ragged.cuh"

namespace b200q {

namespace {

constexpr int kRopeThreads = 128;
constexpr int kMaxRot = 256;    // rotated elements of a head
constexpr int kMaxRows = 4;     // rows of one CTA
// Units a thread loads before it stores the first (rotated rows: 62 / 53 / 58
// us for 2 / 3 / 4 at 8191 x 64 heads), and the units of query heads that a
// thread of an append takes one after the other (6 x 1000 tokens into Q8 pages:
// 77 us for 4, 72 for 8, two of them in flight; 84 with four).
constexpr int kRowsInFlight = 3, kAppendInFlight = 2, kHeadsPerThread = 8;

template <typename T>
__device__ __forceinline__ float load1(const T* p) {
    return static_cast<float>(*p);
}

// V consecutive elements of T as loaded, 16 bytes at a time (V = 4 or 8 fp32, 8
// fp16), 8 bytes (4 fp16) or one element.
template <typename T, int V>
struct Vec {
    static constexpr int W = sizeof(T) * V / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (W >= 4) {
#pragma unroll
            for (int k = 0; k < W; k += 4) {
                const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p) + k / 4);
                w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
            }
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            w[0] = x.x, w[1] = x.y;
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)))));
    }
};
template <typename T>
struct Vec<T, 1> {
    T x;
    __device__ __forceinline__ void load(const T* p) { x = *p; }
    __device__ __forceinline__ float get(int) const { return static_cast<float>(x); }
};
template <int V>
__device__ __forceinline__ void store_v(float* p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = v[0];
    } else {
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
}
template <int V>
__device__ __forceinline__ void store_v(__half* p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = __float2half_rn(v[0]);
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
            w[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if constexpr (V == 8) __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
}

// cos and sin (times mag) of pos * turn, turn in 2^-64 turns.
__device__ __forceinline__ float2 cos_sin(int pos, uint64_t turn, float mag) {
    const uint64_t a = static_cast<uint64_t>(static_cast<uint32_t>(pos)) * turn;
    const uint32_t top = static_cast<uint32_t>(a >> 32);
    const uint32_t quarter = (top + 0x20000000u) >> 30;
    const int rest = static_cast<int>(top - (quarter << 30));  // 2^-32 turns, within an eighth
    float s, c;
    sincospif(static_cast<float>(rest) * 4.656612873077392578125e-10f, &s, &c);  // 2^-31: half turns
    const float cc = (quarter & 1u) ? -s : c, ss = (quarter & 1u) ? c : s;
    return (quarter & 2u) ? make_float2(-cc * mag, -ss * mag) : make_float2(cc * mag, ss * mag);
}
// The same in fp64, by the Taylor series about 0: an eighth of a turn is
// pi / 4 at most, where the first terms left out are below 2^-54 (sin: x^17 /
// 17!) and 2^-58 (cos: x^18 / 18!).
__device__ __forceinline__ double2 cos_sin64(int pos, uint64_t turn, double mag) {
    const uint64_t a = static_cast<uint64_t>(static_cast<uint32_t>(pos)) * turn;
    const uint64_t quarter = (a + (1ull << 61)) >> 62;
    const long long rest = static_cast<long long>(a - (quarter << 62));
    const double x = static_cast<double>(rest) * (6.283185307179586476925 / 18446744073709551616.0);  // 2 pi 2^-64
    const double u = -x * x;
    double s = 1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;  // 1 / 15!, 1 / 16!
    s = fma(s, u, 1.0 / 6227020800.0);
    s = fma(s, u, 1.0 / 39916800.0);
    s = fma(s, u, 1.0 / 362880.0);
    s = fma(s, u, 1.0 / 5040.0);
    s = fma(s, u, 1.0 / 120.0);
    s = fma(s, u, 1.0 / 6.0);
    s = fma(s * u, x, x);
    c = fma(c, u, 1.0 / 87178291200.0);
    c = fma(c, u, 1.0 / 479001600.0);
    c = fma(c, u, 1.0 / 3628800.0);
    c = fma(c, u, 1.0 / 40320.0);
    c = fma(c, u, 1.0 / 720.0);
    c = fma(c, u, 1.0 / 24.0);
    c = fma(c, u, 0.5);
    c = fma(c, u, 1.0);
    const double cc = (quarter & 1u) ? -s : c, ss = (quarter & 1u) ? c : s;
    return (quarter & 2u) ? make_double2(-cc * mag, -ss * mag) : make_double2(cc * mag, ss * mag);
}

// How one head's elements are cut into units that read and write the same
// elements: a pair unit is V elements of each half of the pairs (half layout)
// or V elements of V / 2 pairs (interleaved); a copy unit the V elements after
// the rotated part. V = 1: one pair, one element.
struct RopeShape {
    int hd;
    int rot;
    int half;        // layout: pairs (p, p + rot / 2) instead of (2p, 2p + 1)
    int units;       // per head
    int pair_units;  // the first of them
    uint32_t unit_mul;  // index / units = div_by
    int unit_shift;
};

// Rotates `heads` heads of one row by the threads of the CTA: src heads hd
// elements apart, dst heads dst_step. A thread keeps to one unit and its
// angles and walks the heads, kFlight of them loaded before the first is
// stored. cs: cos, sin of the row's pairs (unused when nothing is rotated).
// A copy unit goes the same way and keeps what it read.
template <int V, int kFlight, typename T, typename TO>
__device__ __forceinline__ void rotate_heads(const RopeShape& s, const float2* cs, const T* src, TO* dst,
                                             long long dst_step, int heads) {
    int u = threadIdx.x, h0 = 0, ustep = kRopeThreads, hstep = 1;
    if (s.units <= kRopeThreads) {
        h0 = div_by(threadIdx.x, s.unit_mul, s.unit_shift);
        u = threadIdx.x - h0 * s.units;
        ustep = s.units;
        hstep = div_by(kRopeThreads, s.unit_mul, s.unit_shift);
        if (h0 >= hstep) return;  // the remainder of the threads
    }
    for (; u < s.units; u += ustep) {
        const bool turn = u < s.pair_units;
        const bool two = turn && (s.half || V == 1);
        const int p = two ? u * V : u * V / 2;
        const int i = !turn ? s.rot + (u - s.pair_units) * V : (V == 1 && !s.half ? 2 * u : u * V);
        const int j = i + (s.half ? s.rot / 2 : 1);
        float c[V], n[V];  // per element of the first vector (half), or per pair (interleaved)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 t = turn && (two || e < V / 2) ? cs[p + e] : make_float2(1.0f, 0.0f);
            c[e] = t.x, n[e] = t.y;
        }
#pragma unroll 1
        for (int h = h0; h < heads; h += hstep * kFlight) {
            Vec<T, V> a[kFlight], b[kFlight];
#pragma unroll
            for (int k = 0; k < kFlight; ++k) {
                const int hh = h + k * hstep;
                if (hh >= heads) continue;
                a[k].load(src + hh * s.hd + i);
                if (two) b[k].load(src + hh * s.hd + j);
            }
#pragma unroll
            for (int k = 0; k < kFlight; ++k) {
                const int hh = h + k * hstep;
                if (hh >= heads) continue;
                TO* y = dst + hh * dst_step;
                float o[V];
                if (two) {
                    float o2[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 r = fma2(both(b[k].get(e)), make_float2(-n[e], c[e]),
                                              mul2(both(a[k].get(e)), make_float2(c[e], n[e])));
                        o[e] = r.x, o2[e] = r.y;
                    }
                    store_v(y + j, o2);
                } else if (V > 1 && turn) {
#pragma unroll
                    for (int e = 0; e + 1 < V; e += 2) {
                        const float2 r = fma2(both(a[k].get(e + 1)), make_float2(-n[e / 2], c[e / 2]),
                                              mul2(both(a[k].get(e)), make_float2(c[e / 2], n[e / 2])));
                        o[e] = r.x, o[e + 1] = r.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = a[k].get(e);
                }
                store_v(y + i, o);
            }
        }
    }
}

// One unit of one head, loaded and stored apart, for threads that take units
// of any head and row in turn.
template <typename T, int V>
struct RopeUnit {
    Vec<T, V> a, b;
    int i, p;       // first element; first pair, -1 for a copy
    bool two;       // a second vector, rot / 2 elements on
    __device__ __forceinline__ void load(const RopeShape& s, const T* x, int u) {
        two = u < s.pair_units && (s.half || V == 1);
        p = u >= s.pair_units ? -1 : (two ? u * V : u * V / 2);
        i = u >= s.pair_units ? s.rot + (u - s.pair_units) * V : (V == 1 && !s.half ? 2 * u : u * V);
        a.load(x + i);
        if (two) b.load(x + i + (s.half ? s.rot / 2 : 1));
    }
    template <typename TO>
    __device__ __forceinline__ void store(const RopeShape& s, const float2* cs, TO* y) const {
        float o[V];
        if (p < 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = a.get(e);
        } else if (two) {
            float o2[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = cs[p + e];
                o[e] = a.get(e) * t.x - b.get(e) * t.y;
                o2[e] = a.get(e) * t.y + b.get(e) * t.x;
            }
            store_v(y + i + (s.half ? s.rot / 2 : 1), o2);
        } else {
#pragma unroll
            for (int e = 0; e + 1 < V; e += 2) {
                const float2 t = cs[p + e / 2];
                o[e] = a.get(e) * t.x - a.get(e + 1) * t.y;
                o[e + 1] = a.get(e) * t.y + a.get(e + 1) * t.x;
            }
        }
        store_v(y + i, o);
    }
};

struct RopeRowsArgs {
    const void* x;
    void* y;
    const int* pos;          // [rows]
    const uint64_t* turns;   // [rot / 2]
    long long x_stride, y_stride;
    int rows, heads, rows_per_cta, heads_per_cta;
    float mag;
    RopeShape s;
};

// Bound by its bytes for prompts, by latency for a step: a thread's loads go
// out before the angles are computed, which need positions from memory first.
template <int V, typename T>
__global__ void __launch_bounds__(kRopeThreads) b200q_rope_rows_kernel(const RopeRowsArgs a) {
    __shared__ float2 cs[kMaxRows * kMaxRot / 2];
    griddep_launch_dependents();
    griddep_wait();
    const int np = a.s.rot / 2;
    const int r0 = blockIdx.x * a.rows_per_cta, h0 = blockIdx.y * a.heads_per_cta;
    const int nr = min(a.rows_per_cta, a.rows - r0);
    const int per_row = min(a.heads_per_cta, a.heads - h0) * a.s.units, total = nr * per_row;
    const T* x = static_cast<const T*>(a.x) + r0 * a.x_stride + h0 * a.s.hd;
    T* y = static_cast<T*>(a.y) + r0 * a.y_stride + h0 * a.s.hd;
    bool angles = false;
    for (int i0 = threadIdx.x; i0 - static_cast<int>(threadIdx.x) < total; i0 += kRopeThreads * kRowsInFlight) {
        RopeUnit<T, V> u[kRowsInFlight];
        int at[kRowsInFlight], row[kRowsInFlight];  // head's first element, row (-1: none)
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k) {
            int i = i0 + k * kRopeThreads;
            row[k] = -1;
            if (i >= total) continue;
            int r = 0;
            while (i >= per_row) i -= per_row, ++r;
            const int h = div_by(i, a.s.unit_mul, a.s.unit_shift);
            row[k] = r;
            at[k] = h * a.s.hd;
            u[k].load(a.s, x + r * a.x_stride + at[k], i - h * a.s.units);
        }
        if (!angles) {
            for (int i = threadIdx.x; i < nr * np; i += kRopeThreads)
                cs[i] = cos_sin(a.pos[r0 + i / np], a.turns[i % np], a.mag);
            __syncthreads();
            angles = true;
        }
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k)
            if (row[k] >= 0) u[k].store(a.s, cs + row[k] * np, y + row[k] * a.y_stride + at[k]);
    }
}

struct AppendArgs {
    RaggedView r;
    PagedView kv;
    const void *q, *k, *v;
    void* q_out;             // NULL: no queries
    const uint64_t* turns;   // NULL: no rotation (s.rot == 0)
    long long q_stride, kv_stride, q_out_stride;
    int heads, rows_per_cta;
    int ctas;                   // of a block of rows:
    int kv_per_cta, kv_ctas;    // 0 .. kv_ctas - 1 take its kv heads
    int heads_per_cta;          // and the others its query heads
    bool walk;                  // query heads by rotate_heads, a row after the other
    bool kv_wide;               // Q8: rows can be read eight elements at a time
    double mag;
    RopeShape s, plain;         // with rotation (keys, queries) and without (values)
};

// The Q8 row quantizer of the paged store (model_graph.cpp:1545-1573), as the
// decode kernel's: every step rounded to fp32.
__device__ __forceinline__ float q8_scale(float amax) {
    return amax > 0.0f ? __fdiv_rn(amax, 127.0f) : __fdiv_rn(1.0f, 127.0f);
}
// round() of the definition (halves away from zero), as a byte: to the nearest
// integer by adding 1.5 2^23, halves that went to the even side put right. NaN
// (also an infinity over its scale) is 0, as the conversion to an integer makes it.
__device__ __forceinline__ uint32_t q8_code(float x, float inv) {
    const float p = __fmul_rn(x, inv), y = p == p ? fminf(fmaxf(p, -127.0f), 127.0f) : 0.0f;
    const float t = __fadd_rn(y, 12582912.0f);
    const float rest = __fsub_rn(y, __fsub_rn(t, 12582912.0f));  // exact
    int c = __float_as_int(t);
    if (rest == 0.5f && y > 0.0f) ++c;
    if (rest == -0.5f && y < 0.0f) --c;
    return static_cast<uint32_t>(c) & 0xFFu;
}

// Position of batch row `row` and the sequence that holds it (-1: none), by a
// warp: the entries of cu_q not above the row are counted 32 at a time, one
// trip to memory instead of a search's log2(batch).
__device__ __forceinline__ int2 locate(const RaggedView& r, int row, int lane) {
    int count = 0;
    for (int b0 = 0; b0 <= r.batch; b0 += 32)
        count += __popc(__ballot_sync(0xffffffffu, b0 + lane <= r.batch && r.cu_q[min(b0 + lane, r.batch)] <= row));
    const int b = count - 1;
    if (b < 0 || b >= r.batch) return make_int2(0, -1);
    return make_int2(r.kv_len[b] - (seq_rows(r, b).y - row), b);
}

// CTAs: for each block of rows_per_cta rows its kv heads, then its query heads
// (side by side, so that the quantizer's long chains run under the query rows'
// traffic: all kv heads first measured 79 us for 6 x 1000 tokens into Q8 pages).
template <int V, typename T, bool Q8>
__global__ void __launch_bounds__(kRopeThreads) b200q_rope_append_kernel(const AppendArgs a) {
    __shared__ float2 cs[kMaxRows * kMaxRot / 2];
    __shared__ double2 cs64[Q8 ? kMaxRows * 64 : 1];  // head <= 128
    __shared__ int2 place[kMaxRows];  // position and sequence of each row
    __shared__ uint32_t pool_of[kMaxRows];  // pool row of kv head 0 at the position; kNoRow without a page
    // No early start for the kernels behind: the one-position attention reads the
    // cached rows before it waits for the kernel ahead, and a kernel in between
    // that passes its own start on would let it run beside this one's stores.
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int np = a.s.rot / 2, hd = a.s.hd;
    const int block = blockIdx.x / a.ctas, part = blockIdx.x - block * a.ctas;
    const int r0 = block * a.rows_per_cta, nr = min(a.rows_per_cta, a.r.n_tokens - r0);
    const bool keys = part < a.kv_ctas;
    for (int i = warp; i < nr; i += kRopeThreads / 32) {
        const int2 at = locate(a.r, r0 + i, lane);
        if (lane == 0) {
            place[i] = at;
            uint32_t row = kNoRow;
            if (keys && at.y >= 0) {
                const int pg = at.x >= 0 ? at.x / a.kv.page : -1;
                const int slot = page_slot(a.kv, at.y, pg);
                if (slot >= 0) row = static_cast<uint32_t>(pool_row(a.kv, slot, 0, at.x - pg * a.kv.page));
                else if (part == 0) flag_bad_page(a.kv);
            }
            pool_of[i] = row;
        }
    }
    __syncthreads();
    const bool wide = Q8 && keys;
    for (int i = threadIdx.x; i < nr * np; i += kRopeThreads) {
        const int r = i / np, p = i - r * np;
        if (wide) {
            if constexpr (Q8) cs64[r * 64 + p] = cos_sin64(place[r].x, a.turns[p], a.mag);
        } else {
            cs[i] = cos_sin(place[r].x, a.turns[p], static_cast<float>(a.mag));
        }
    }
    __syncthreads();
    if (!keys) {
        const int h0 = (part - a.kv_ctas) * a.heads_per_cta;
        if (!a.walk) {
            const int per_row = min(a.heads_per_cta, a.heads - h0) * a.s.units, total = nr * per_row;
            const T* x = static_cast<const T*>(a.q) + r0 * a.q_stride + h0 * hd;
            T* y = static_cast<T*>(a.q_out) + r0 * a.q_out_stride + h0 * hd;
            for (int i0 = threadIdx.x; i0 < total; i0 += kRopeThreads * kAppendInFlight) {
                RopeUnit<T, V> u[kAppendInFlight];
                int at[kAppendInFlight], row[kAppendInFlight];
#pragma unroll
                for (int k = 0; k < kAppendInFlight; ++k) {
                    int i = i0 + k * kRopeThreads;
                    row[k] = -1;
                    if (i >= total) continue;
                    int r = 0;
                    while (i >= per_row) i -= per_row, ++r;
                    if (place[r].y < 0) continue;
                    const int h = div_by(i, a.s.unit_mul, a.s.unit_shift);
                    row[k] = r;
                    at[k] = h * hd;
                    u[k].load(a.s, x + r * a.q_stride + at[k], i - h * a.s.units);
                }
#pragma unroll
                for (int k = 0; k < kAppendInFlight; ++k)
                    if (row[k] >= 0) u[k].store(a.s, cs + row[k] * np, y + row[k] * a.q_out_stride + at[k]);
            }
            return;
        }
        for (int r = 0; r < nr; ++r)
            if (place[r].y >= 0)
                rotate_heads<V, kAppendInFlight>(
                    a.s, cs + r * np, static_cast<const T*>(a.q) + (r0 + r) * a.q_stride + h0 * hd,
                    static_cast<T*>(a.q_out) + (r0 + r) * a.q_out_stride + h0 * hd, static_cast<long long>(hd),
                    min(a.heads_per_cta, a.heads - h0));
        return;
    }
    const int kh0 = part * a.kv_per_cta;
    const int nh = min(a.kv_per_cta, a.kv.n_kv - kh0);
    if constexpr (!Q8) {
        // Keys, then values (every unit a copy), of the rows' heads: too few per row
        // to walk them row by row.
        const int keys_of_row = nh * a.s.units, per_row = keys_of_row + nh * a.plain.units, total = nr * per_row;
        for (int i0 = threadIdx.x; i0 < total; i0 += kRopeThreads * kAppendInFlight) {
            RopeUnit<T, V> u[kAppendInFlight];
            __half* dst[kAppendInFlight];
            int row[kAppendInFlight];
#pragma unroll
            for (int k = 0; k < kAppendInFlight; ++k) {
                int i = i0 + k * kRopeThreads;
                dst[k] = nullptr;
                if (i >= total) continue;
                int r = 0;
                while (i >= per_row) i -= per_row, ++r;
                if (pool_of[r] == kNoRow) continue;
                const bool is_v = i >= keys_of_row;
                if (is_v) i -= keys_of_row;
                const RopeShape& s = is_v ? a.plain : a.s;
                const int h = div_by(i, s.unit_mul, s.unit_shift);
                dst[k] = static_cast<__half*>(is_v ? a.kv.v : a.kv.k) +
                         (pool_of[r] + static_cast<long long>(kh0 + h) * a.kv.page) * hd;
                row[k] = r;
                u[k].load(s, static_cast<const T*>(is_v ? a.v : a.k) + (r0 + r) * a.kv_stride + (kh0 + h) * hd,
                          i - h * s.units);
            }
#pragma unroll
            for (int k = 0; k < kAppendInFlight; ++k)
                if (dst[k]) u[k].store(a.s, cs + row[k] * np, dst[k]);
        }
    } else {
        // A row of a kv head's keys or values is E elements a lane, over hd / E
        // lanes of a warp (so a warp takes two rows of 128, four of 64, at once);
        // for the half layout a lane also reads its elements' mates.
        constexpr int E = 8;
        const int lanes = hd / E, sub = lane / lanes, e0 = lane % lanes * E;
        const int tasks = nr * nh * 2, step = 32 / lanes * (kRopeThreads / 32);
        for (int i0 = 0; i0 < tasks; i0 += step) {
            int i = i0 + warp * (32 / lanes) + sub;
            bool mine = i < tasks;
            i = mine ? i : 0;
            int r = 0;
            while (i >= 2 * nh) i -= 2 * nh, ++r;
            mine = mine && pool_of[r] != kNoRow;  // a row of no sequence, or without a page, is not read
            const bool is_v = i >= nh;
            const int h = kh0 + (is_v ? i - nh : i);
            const T* src = static_cast<const T*>(is_v ? a.v : a.k) + (r0 + r) * a.kv_stride + h * hd;
            float x[E] = {}, mate[E] = {};
            if (mine && a.kv_wide) {
                Vec<T, E> v, w;
                v.load(src + e0);
                const bool other = !is_v && a.s.half && e0 < a.s.rot;
                if (other) w.load(src + (e0 < np ? e0 + np : e0 - np));
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    x[e] = v.get(e);
                    mate[e] = other ? w.get(e) : v.get(e ^ 1);
                }
            } else if (mine) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int el = e0 + e;
                    x[e] = load1(src + el);
                    if (!is_v && el < a.s.rot)
                        mate[e] = load1(src + (a.s.half ? (el < np ? el + np : el - np) : el ^ 1));
                }
            }
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int el = e0 + e;
                if (!is_v && el < a.s.rot) {
                    const bool second = a.s.half ? el >= np : (el & 1);
                    const double2 t = cs64[r * 64 + (a.s.half ? (second ? el - np : el) : el >> 1)];
                    const double w = static_cast<double>(mate[e]) * t.y;
                    x[e] = static_cast<float>(fma(static_cast<double>(x[e]), t.x, second ? w : -w));
                }
                amax = fmaxf(amax, fabsf(x[e]));
            }
            for (int o = lanes / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float scale = q8_scale(amax), inv = __fdiv_rn(1.0f, scale);
            if (!mine) continue;
            const long long dst = pool_of[r] + static_cast<long long>(h) * a.kv.page;
            uint32_t lo = 0, up = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo |= q8_code(x[e], inv) << (8 * e);
                up |= q8_code(x[4 + e], inv) << (8 * e);
            }
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(is_v ? a.kv.v : a.kv.k) + dst * hd + e0) = make_uint2(lo, up);
            if (e0 == 0) (is_v ? a.kv.vs : a.kv.ks)[dst] = scale;
        }
    }
}

cudaLaunchConfig_t ragged_cfg(dim3 grid, dim3 block, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    if (pdl_enabled()) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    return cfg;
}

bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The units of one head: V elements wide (16 bytes, or 8 for fp16) when every
// vector of them stays aligned -- rows, heads and both halves of the pairs --,
// else one pair or element.
int rope_units(int hd, int rot, int half, int v, RopeShape& s) {
    while (v > 1 && (hd % v || rot % (half ? 2 * v : v))) v = v == 8 ? 4 : 1;
    s.hd = hd;
    s.rot = rot;
    s.half = half;
    s.pair_units = v == 1 ? rot / 2 : (half ? rot / 2 / v : rot / v);
    s.units = s.pair_units + (hd - rot) / v;
    divisor(s.units, s.unit_mul, s.unit_shift);
    return v;
}

// The widest vector that pointers and strides (in elements) allow.
int widest(size_t es, std::initializer_list<const void*> ptrs, std::initializer_list<long long> strides) {
    for (int v = es == 2 ? 8 : 4; v > 1; v = v == 8 ? 4 : 1) {
        bool ok = true;
        for (const void* p : ptrs) ok = ok && aligned_to(p, v * es);
        for (long long st : strides) ok = ok && st % v == 0;
        if (ok) return v;
    }
    return 1;
}

size_t elem_size(int dtype) { return dtype == B200Q_F32 ? 4 : 2; }

const long double kTwoPi = 6.283185307179586476925286766559L;

// The pair whose frequency makes `turns` turns over `context` positions.
double pair_of_turns(double turns, int context, int rot_dim, double theta) {
    return static_cast<double>(rot_dim * std::log(context / (turns * kTwoPi)) /
                               (2.0L * std::log(static_cast<long double>(theta))));
}

}  // namespace

int rope_table(int rot_dim, double theta, int scaling, double factor, double low, double high, int original_context,
               unsigned long long* turns, double* mag) {
    if (!turns || !mag) return B200Q_EINVAL;
    if (rot_dim <= 0 || rot_dim % 2 || rot_dim > kMaxRot || !(theta > 1.0) || !std::isfinite(theta)) return B200Q_ESHAPE;
    if (scaling < B200Q_ROPE_PLAIN || scaling > B200Q_ROPE_YARN) return B200Q_EINVAL;
    if (scaling != B200Q_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return B200Q_EINVAL;
    const bool bands = scaling == B200Q_ROPE_LLAMA3 || scaling == B200Q_ROPE_YARN;
    if (bands && (original_context <= 0 || !(low > 0.0) || !(high > low) || !std::isfinite(high))) return B200Q_EINVAL;
    double y_lo = 0.0, y_hi = 1.0;
    if (scaling == B200Q_ROPE_YARN) {
        y_lo = std::max(0.0, std::floor(pair_of_turns(high, original_context, rot_dim, theta)));
        y_hi = std::min(rot_dim - 1.0, std::ceil(pair_of_turns(low, original_context, rot_dim, theta)));
        if (!(y_hi > y_lo)) y_hi = y_lo + 0.001;
    }
    for (int p = 0; p < rot_dim / 2; ++p) {
        long double f = std::pow(static_cast<long double>(theta), -2.0L * p / rot_dim);
        if (scaling == B200Q_ROPE_LINEAR) {
            f /= factor;
        } else if (scaling == B200Q_ROPE_LLAMA3) {
            const long double n = original_context * f / kTwoPi;  // turns over the original context
            if (n < low) {
                f /= factor;
            } else if (n <= high) {
                const long double t = (n - low) / (static_cast<long double>(high) - low);
                f = (1.0L - t) * f / factor + t * f;
            }
        } else if (scaling == B200Q_ROPE_YARN) {
            const long double at_p = (p - y_lo) / (static_cast<long double>(y_hi) - y_lo);
            const long double t = at_p < 0.0L ? 0.0L : at_p > 1.0L ? 1.0L : at_p;
            f = f / factor * t + f * (1.0L - t);
        }
        turns[p] = static_cast<unsigned long long>(std::ldexp(f / kTwoPi, 64) + 0.5L);
    }
    *mag = scaling == B200Q_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return B200Q_OK;
}

int launch_rope_rows(const void* x, void* out, int dtype, int rows, int heads, int hd, long long x_stride,
                     long long out_stride, const int* positions, const unsigned long long* turns, int rot, int layout,
                     double mag, Device* dev, cudaStream_t st) {
    if (!turns || rows < 0 || heads <= 0 || hd <= 0 || !dev) return B200Q_EINVAL;
    if (rows > 0 && (!x || !out || !positions)) return B200Q_EINVAL;  // (rows of no memory have no address)
    if ((dtype != B200Q_F32 && dtype != B200Q_F16) || (layout != B200Q_ROPE_INTERLEAVED && layout != B200Q_ROPE_HALF))
        return B200Q_EINVAL;
    if (rot <= 0 || rot % 2 || rot > hd || rot > kMaxRot) return B200Q_ESHAPE;
    const long long width = static_cast<long long>(heads) * hd;
    if (width > (1 << 30)) return B200Q_ESHAPE;
    if (x_stride == 0) x_stride = width;
    if (out_stride == 0) out_stride = width;
    if (x_stride < width || out_stride < width) return B200Q_ESHAPE;
    const size_t es = elem_size(dtype);
    if (!aligned_to(x, es) || !aligned_to(out, es) || !aligned_to(positions, 4) || !aligned_to(turns, 8))
        return B200Q_EALIGN;
    if (rows == 0) return B200Q_OK;
    RopeRowsArgs a{};
    a.x = x;
    a.y = out;
    a.pos = positions;
    a.turns = reinterpret_cast<const uint64_t*>(turns);
    a.x_stride = x_stride;
    a.y_stride = out_stride;
    a.rows = rows;
    a.heads = heads;
    a.mag = static_cast<float>(mag);
    const int v = rope_units(hd, rot, layout == B200Q_ROPE_HALF, widest(es, {x, out}, {x_stride, out_stride}), a.s);
    // A CTA takes a few units a thread when there are many, one when the
    // units would not give every SM a few CTAs.
    const long long units = static_cast<long long>(rows) * heads * a.s.units;
    const int per_cta = units > 2048ll * kRopeThreads ? kRowsInFlight * kRopeThreads : kRopeThreads;
    a.heads_per_cta = std::max(1, std::min(heads, per_cta / a.s.units));
    a.rows_per_cta = a.heads_per_cta < heads ? 1 : std::max(1, std::min(kMaxRows, per_cta / (heads * a.s.units)));
    const int head_ctas = (heads + a.heads_per_cta - 1) / a.heads_per_cta;
    if (head_ctas > 65535) return B200Q_ESHAPE;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ragged_cfg(dim3((rows + a.rows_per_cta - 1) / a.rows_per_cta, head_ctas),
                                        dim3(kRopeThreads), st, attr);
    cudaError_t e;
    if (dtype == B200Q_F32)
        e = v == 4 ? cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<4, float>, a)
                   : cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<1, float>, a);
    else
        e = v == 8   ? cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<8, __half>, a)
            : v == 4 ? cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<4, __half>, a)
                     : cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<1, __half>, a);
    return e == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

int check_paged(const PagedKV& p, int hd) {
    const bool q8 = p.kv_mode == B200Q_KV_Q8;
    if ((p.kv_mode != B200Q_KV_F16 && !q8) || !p.k_pages || !p.v_pages || !p.page_table || p.n_slots <= 0 ||
        p.page_size <= 0 || p.pages_per_seq <= 0 || p.n_kv <= 0 || (q8 && (!p.k_scales || !p.v_scales)))
        return B200Q_EINVAL;
    if (hd != 64 && hd != 128) return B200Q_ESHAPE;
    // positions and pool rows are 32-bit numbers in the kernels
    if (static_cast<long long>(p.pages_per_seq) * p.page_size > (1 << 30)) return B200Q_ESHAPE;
    if (static_cast<long long>(p.n_slots) * p.n_kv > 0xFFFFFFFEll / p.page_size) return B200Q_ESHAPE;
    if (!aligned_to(p.k_pages, 16) || !aligned_to(p.v_pages, 16) || !aligned_to(p.page_table, 4) ||
        (q8 && (!aligned_to(p.k_scales, 4) || !aligned_to(p.v_scales, 4))))
        return B200Q_EALIGN;
    return B200Q_OK;
}

PagedView paged_view(const PagedKV& p, Device* dev) {
    PagedView v{};
    v.k = p.k_pages;
    v.v = p.v_pages;
    v.ks = p.k_scales;
    v.vs = p.v_scales;
    v.table = p.page_table;
    v.pages_per_seq = p.pages_per_seq;
    v.page = p.page_size;
    v.n_slots = p.n_slots;
    v.n_kv = p.n_kv;
    v.status = dev->status;
    return v;
}

int launch_rope_append(const void* q, const void* k, const void* v, int dtype, int n_tokens, int batch, const int* cu_q,
                       const int* kv_len, int heads, int hd, long long q_stride, long long kv_stride, void* q_out,
                       long long q_out_stride, const unsigned long long* turns, int rot, int layout, double mag,
                       const PagedKV& pkv, Device* dev, cudaStream_t st) {
    if (!cu_q || !kv_len || n_tokens < 0 || batch <= 0 || !dev) return B200Q_EINVAL;
    if (n_tokens > 0 && (!k || !v)) return B200Q_EINVAL;  // (rows of no memory have no address)
    if (q_out && (!q || heads <= 0)) return B200Q_EINVAL;
    if (dtype != B200Q_F32 && dtype != B200Q_F16) return B200Q_EINVAL;
    if (turns && layout != B200Q_ROPE_INTERLEAVED && layout != B200Q_ROPE_HALF) return B200Q_EINVAL;
    int rc = check_paged(pkv, hd);
    if (rc != B200Q_OK) return rc;
    if (turns ? (rot <= 0 || rot % 2 || rot > hd) : rot != 0) return B200Q_ESHAPE;
    const long long qw = static_cast<long long>(heads) * hd, kw = static_cast<long long>(pkv.n_kv) * hd;
    if (qw > (1 << 30) || kw > (1 << 30)) return B200Q_ESHAPE;
    if (q_stride == 0) q_stride = qw;
    if (q_out_stride == 0) q_out_stride = qw;
    if (kv_stride == 0) kv_stride = kw;
    if ((q_out && (q_stride < qw || q_out_stride < qw)) || kv_stride < kw) return B200Q_ESHAPE;
    const size_t es = elem_size(dtype);
    if (!aligned_to(k, es) || !aligned_to(v, es) || !aligned_to(cu_q, 4) || !aligned_to(kv_len, 4) ||
        (q_out && (!aligned_to(q, es) || !aligned_to(q_out, es))) || (turns && !aligned_to(turns, 8)))
        return B200Q_EALIGN;
    if (n_tokens == 0) return B200Q_OK;
    AppendArgs a{};
    a.r = RaggedView{cu_q, kv_len, batch, n_tokens};
    a.kv = paged_view(pkv, dev);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.turns = reinterpret_cast<const uint64_t*>(turns);
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.q_out_stride = q_out_stride;
    a.heads = heads;
    a.mag = mag;
    const bool q8 = pkv.kv_mode == B200Q_KV_Q8;
    int width = q_out ? widest(es, {q, q_out}, {q_stride, q_out_stride}) : 8;
    // (Q8 rows are read by the warp that quantizes them, in its own widths.)
    if (!q8) width = std::min(width, widest(es, {k, v}, {kv_stride}));
    const int vec = rope_units(hd, rot, layout == B200Q_ROPE_HALF, std::min(width, es == 2 ? 8 : 4), a.s);
    rope_units(hd, 0, 0, vec, a.plain);
    const long long units = static_cast<long long>(n_tokens) * (q_out ? heads : pkv.n_kv) * a.s.units;
    const bool many = units > 2048ll * kRopeThreads;
    // Rows of many heads are walked (fewer instructions a unit), rows of few taken
    // together (7 x 1200 rows of 144 units: 22 us against 33).
    a.walk = many && heads * a.s.units >= kHeadsPerThread / 2 * kRopeThreads;
    const int per_cta = (a.walk ? kHeadsPerThread : many ? kAppendInFlight : 1) * kRopeThreads;
    a.heads_per_cta = std::max(1, std::min(heads, per_cta / a.s.units));
    const int q_ctas = q_out ? (heads + a.heads_per_cta - 1) / a.heads_per_cta : 0;
    a.rows_per_cta = std::min<long long>(kMaxRows, std::max<long long>(1, n_tokens / 2048));
    a.kv_per_cta = std::max(1, std::min(pkv.n_kv, (many ? 2 : 1) * kRopeThreads / (2 * a.s.units)));
    a.kv_ctas = (pkv.n_kv + a.kv_per_cta - 1) / a.kv_per_cta;
    a.ctas = q_ctas + a.kv_ctas;
    const long long blocks = (n_tokens + a.rows_per_cta - 1ll) / a.rows_per_cta;
    if (blocks * a.ctas > 0x7fffffffll) return B200Q_ESHAPE;
    // A lane's eight elements stay aligned, are all rotated or none, and so are
    // their mates half the pairs away.
    a.kv_wide = aligned_to(k, 16) && aligned_to(v, 16) && kv_stride % 8 == 0 &&
                rot % (layout == B200Q_ROPE_HALF ? 16 : 8) == 0;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ragged_cfg(dim3(static_cast<unsigned>(blocks * a.ctas)), dim3(kRopeThreads), st, attr);
    cudaError_t e;
#define B200Q_APPEND(V, T)                                                       \
    e = q8 ? cudaLaunchKernelEx(&cfg, b200q_rope_append_kernel<V, T, true>, a)   \
           : cudaLaunchKernelEx(&cfg, b200q_rope_append_kernel<V, T, false>, a)
    if (dtype == B200Q_F32) {
        if (vec == 4) B200Q_APPEND(4, float);
        else B200Q_APPEND(1, float);
    } else {
        if (vec == 8) B200Q_APPEND(8, __half);
        else if (vec == 4) B200Q_APPEND(4, __half);
        else B200Q_APPEND(1, __half);
    }
#undef B200Q_APPEND
    return e == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

}  // namespace b200q
