// Rotary positions and paged-cache appends for batches of sequences of
// different lengths, and the host side of the ragged operators.
//
// Angles. Pair p of a row at position pos turns by pos * f_p radians. In fp32
// the product loses the phase of far positions (at pos = 1e6 its last bit is
// 0.06 rad), so the table holds f_p / (2 pi) as a 64-bit fraction of a turn
// and the kernels form pos * turn modulo 2^64: the whole turns drop out of
// the product exactly and what is left is off by at most pos * 2^-65 turns.
// The fraction's nearest quarter turn is taken out as an integer too, so that
// sincospi sees at most an eighth of a turn, with all 24 bits of it.
//
// Q8 keys are rotated in fp64: the page's quantizer rounds the fp32 row to
// codes, and a key that is off by an fp32 rounding would fall on the other
// side of a border of two codes now and then (2e-5 of all codes measured at
// 2^-24 relative).
#include <algorithm>
#include <cmath>

#include "internal.h"
#include "ragged.cuh"

namespace b200q {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 256;  // rotated elements of a head: one cos/sin pair per thread of two rows

// Rounded to the nearest fp16 / kept.
template <typename T>
__device__ __forceinline__ float load1(const T* p) {
    return static_cast<float>(*p);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }

// N consecutive elements as floats; N * sizeof(T) is 8 or 16 and p aligned to it.
template <int N>
__device__ __forceinline__ void load_n(const float* p, float (&v)[N]) {
    static_assert(N == 4, "one 16-byte load");
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
template <int N>
__device__ __forceinline__ void load_n(const __half* p, float (&v)[N]) {
    static_assert(N == 4, "one 8-byte load");
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
template <int N>
__device__ __forceinline__ void store_n(float* p, const float (&v)[N]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <int N>
__device__ __forceinline__ void store_n(__half* p, const float (&v)[N]) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
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
__device__ __forceinline__ double2 cos_sin64(int pos, uint64_t turn, double mag) {
    const uint64_t a = static_cast<uint64_t>(static_cast<uint32_t>(pos)) * turn;
    const uint64_t quarter = (a + (1ull << 61)) >> 62;
    const long long rest = static_cast<long long>(a - (quarter << 62));
    double s, c;
    sincospi(static_cast<double>(rest) * 1.0842021724855044e-19, &s, &c);  // 2^-63
    const double cc = (quarter & 1u) ? -s : c, ss = (quarter & 1u) ? c : s;
    return (quarter & 2u) ? make_double2(-cc * mag, -ss * mag) : make_double2(cc * mag, ss * mag);
}

// How one head's elements are cut into units that read and write the same
// elements: a pair unit is one rotated pair (V = 1) or four elements of each
// half of the pairs (V = 4, half layout) or four elements of two pairs (V = 4,
// interleaved); a copy unit is the V elements after the rotated part.
struct RopeShape {
    int hd;
    int rot;
    int half;        // layout: pairs (p, p + rot / 2) instead of (2p, 2p + 1)
    int units;       // per head
    int pair_units;  // the first of them
};

// y = R x for unit u of one head; cs: this row's [rot / 2] cos, sin.
template <int V, typename T>
__device__ __forceinline__ void rope_unit(const RopeShape& s, const float2* cs, const T* x, T* y, int u) {
    if constexpr (V == 1) {
        if (u < s.pair_units) {
            const int i = s.half ? u : 2 * u, j = s.half ? u + s.rot / 2 : 2 * u + 1;
            const float a = load1(x + i), b = load1(x + j);
            store1(y + i, a * cs[u].x - b * cs[u].y);
            store1(y + j, a * cs[u].y + b * cs[u].x);
        } else {
            const int i = s.rot + u - s.pair_units;
            y[i] = x[i];
        }
    } else {
        float a[V], o[V];
        if (u >= s.pair_units) {
            const int i = s.rot + (u - s.pair_units) * V;
            load_n<V>(x + i, a);
            store_n<V>(y + i, a);
        } else if (s.half) {
            float b[V], o2[V];
            const int i = u * V, j = i + s.rot / 2;
            load_n<V>(x + i, a);
            load_n<V>(x + j, b);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = cs[i + e];
                o[e] = a[e] * t.x - b[e] * t.y;
                o2[e] = a[e] * t.y + b[e] * t.x;
            }
            store_n<V>(y + i, o);
            store_n<V>(y + j, o2);
        } else {
            const int i = u * V;
            load_n<V>(x + i, a);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 t = cs[(i + e) / 2];
                o[e] = a[e] * t.x - a[e + 1] * t.y;
                o[e + 1] = a[e] * t.y + a[e + 1] * t.x;
            }
            store_n<V>(y + i, o);
        }
    }
}

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

template <int V, typename T>
__global__ void __launch_bounds__(kRopeThreads) b200q_rope_rows_kernel(const RopeRowsArgs a) {
    __shared__ float2 cs[kRopeThreads];  // rows_per_cta x rot / 2
    griddep_launch_dependents();
    griddep_wait();
    const int np = a.s.rot / 2;
    const int r0 = blockIdx.x * a.rows_per_cta;
    const int nr = min(a.rows_per_cta, a.rows - r0);
    for (int i = threadIdx.x; i < nr * np; i += kRopeThreads)
        cs[i] = cos_sin(a.pos[r0 + i / np], a.turns[i % np], a.mag);
    __syncthreads();
    const int h0 = blockIdx.y * a.heads_per_cta;
    const int per_row = min(a.heads_per_cta, a.heads - h0) * a.s.units;
    for (int r = 0; r < nr; ++r) {
        const T* x = static_cast<const T*>(a.x) + (r0 + r) * a.x_stride + h0 * a.s.hd;
        T* y = static_cast<T*>(a.y) + (r0 + r) * a.y_stride + h0 * a.s.hd;
#pragma unroll 4
        for (int i = threadIdx.x; i < per_row; i += kRopeThreads) {
            const int h = i / a.s.units, u = i - h * a.s.units;
            rope_unit<V>(a.s, cs + r * np, x + h * a.s.hd, y + h * a.s.hd, u);
        }
    }
}

struct AppendArgs {
    RaggedView r;
    PagedView kv;
    const void *q, *k, *v;
    void* q_out;             // NULL: no queries
    const uint64_t* turns;   // NULL: no rotation (s.rot == 0)
    long long q_stride, kv_stride, q_out_stride;
    int heads, heads_per_cta;
    double mag;
    RopeShape s;
};

// The Q8 row quantizer of the paged store (model_graph.cpp:1545-1573), as the
// decode kernel's: every step rounded to fp32.
__device__ __forceinline__ float q8_scale(float amax) {
    return amax > 0.0f ? __fdiv_rn(amax, 127.0f) : __fdiv_rn(1.0f, 127.0f);
}
__device__ __forceinline__ int8_t q8_code(float x, float inv) {
    const int c = static_cast<int>(roundf(__fmul_rn(x, inv)));
    return static_cast<int8_t>(max(-127, min(127, c)));
}

// One CTA per row of the batch and group of query heads; the first group also
// writes the row's keys and values. Bound by the bytes of q (read and
// written) for prompts and by latency for decode steps.
template <int V, typename T, bool Q8>
__global__ void __launch_bounds__(kRopeThreads) b200q_rope_append_kernel(const AppendArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    __shared__ double2 cs64[Q8 ? kMaxRot / 2 : 1];
    griddep_launch_dependents();
    griddep_wait();
    const int row = blockIdx.x;
    const int b = seq_of_row(a.r, row);
    if (b < 0) return;
    const int2 rr = seq_rows(a.r, b);
    const int pos = a.r.kv_len[b] - (rr.y - row);
    const int np = a.s.rot / 2;
    const bool keys = blockIdx.y == 0;
    for (int i = threadIdx.x; i < np; i += kRopeThreads) {
        cs[i] = cos_sin(pos, a.turns[i], static_cast<float>(a.mag));
        if constexpr (Q8) {
            if (keys) cs64[i] = cos_sin64(pos, a.turns[i], a.mag);
        }
    }
    __syncthreads();
    if (a.q_out) {
        const int h0 = blockIdx.y * a.heads_per_cta;
        const int n = min(a.heads_per_cta, a.heads - h0) * a.s.units;
        const T* x = static_cast<const T*>(a.q) + row * a.q_stride + h0 * a.s.hd;
        T* y = static_cast<T*>(a.q_out) + row * a.q_out_stride + h0 * a.s.hd;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += kRopeThreads) {
            const int h = i / a.s.units, u = i - h * a.s.units;
            rope_unit<V>(a.s, cs, x + h * a.s.hd, y + h * a.s.hd, u);
        }
    }
    if (!keys) return;
    const int pg = pos >= 0 ? pos / a.kv.page : -1;
    const int slot = page_slot(a.kv, b, pg);
    if (slot < 0) {
        if (threadIdx.x == 0) flag_bad_page(a.kv);
        return;
    }
    const int off = pos - pg * a.kv.page;
    const T* kin = static_cast<const T*>(a.k) + row * a.kv_stride;
    const T* vin = static_cast<const T*>(a.v) + row * a.kv_stride;
    const int hd = a.s.hd;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // One warp per kv head's key or value row, lane l the elements l, l + 32, ...
    for (int i = warp; i < 2 * a.kv.n_kv; i += kRopeThreads / 32) {
        const bool is_v = i >= a.kv.n_kv;
        const int h = is_v ? i - a.kv.n_kv : i;
        const T* x = (is_v ? vin : kin) + h * hd;
        const long long dst = pool_row(a.kv, slot, h, off);
        constexpr int kMaxPer = 4;  // hd <= 128
        float val[kMaxPer];
        float amax = 0.0f;
#pragma unroll
        for (int t = 0; t < kMaxPer; ++t) {
            const int e = lane + 32 * t;
            val[t] = 0.0f;
            if (e >= hd) continue;
            val[t] = load1(x + e);
            if (!is_v && e < a.s.rot) {
                const int p = a.s.half ? (e < np ? e : e - np) : e >> 1;
                const bool second = a.s.half ? e >= np : (e & 1);
                const int mate = a.s.half ? (second ? e - np : e + np) : e ^ 1;
                const float other = load1(x + mate);
                if constexpr (Q8) {
                    const double2 t2 = cs64[p];
                    const double w = second ? other * t2.y + val[t] * t2.x : val[t] * t2.x - other * t2.y;
                    val[t] = static_cast<float>(w);
                } else {
                    const float2 t2 = cs[p];
                    val[t] = second ? other * t2.y + val[t] * t2.x : val[t] * t2.x - other * t2.y;
                }
            }
            amax = fmaxf(amax, fabsf(val[t]));
        }
        if constexpr (Q8) {
#pragma unroll
            for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float scale = q8_scale(amax), inv = __fdiv_rn(1.0f, scale);
            int8_t* out = static_cast<int8_t*>(is_v ? a.kv.v : a.kv.k) + dst * hd;
#pragma unroll
            for (int t = 0; t < kMaxPer; ++t)
                if (lane + 32 * t < hd) out[lane + 32 * t] = q8_code(val[t], inv);
            if (lane == 0) (is_v ? a.kv.vs : a.kv.ks)[dst] = scale;
        } else {
            __half* out = static_cast<__half*>(is_v ? a.kv.v : a.kv.k) + dst * hd;
#pragma unroll
            for (int t = 0; t < kMaxPer; ++t)
                if (lane + 32 * t < hd) out[lane + 32 * t] = __float2half_rn(val[t]);
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

// The units of one head, four elements wide when every vector of them stays
// aligned (rows, heads and both halves of the pairs), else one pair.
int rope_units(int hd, int rot, int half, bool wide, RopeShape& s) {
    const int v = wide && hd % 4 == 0 && rot % (half ? 8 : 4) == 0 ? 4 : 1;
    s.hd = hd;
    s.rot = rot;
    s.half = half;
    s.pair_units = v == 1 ? rot / 2 : (half ? rot / 2 / v : rot / v);
    s.units = s.pair_units + (hd - rot) / v;
    return v;
}

size_t elem_size(int dtype) { return dtype == B200Q_F32 ? 4 : 2; }

}  // namespace

int rope_table(int rot_dim, double theta, int scaling, double factor, double low, double high, int original_context,
               unsigned long long* turns, double* mag) {
    if (!turns || !mag) return B200Q_EINVAL;
    if (rot_dim <= 0 || rot_dim % 2 || rot_dim > kMaxRot || !(theta > 1.0) || !std::isfinite(theta)) return B200Q_ESHAPE;
    if (scaling < B200Q_ROPE_PLAIN || scaling > B200Q_ROPE_YARN) return B200Q_EINVAL;
    if (scaling != B200Q_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return B200Q_EINVAL;
    const bool bands = scaling == B200Q_ROPE_LLAMA3 || scaling == B200Q_ROPE_YARN;
    if (bands && (original_context <= 0 || !(low > 0.0) || !(high > low) || !std::isfinite(high))) return B200Q_EINVAL;
    const double two_pi = 6.283185307179586476925286766559;
    double y_lo = 0.0, y_hi = 1.0;
    if (scaling == B200Q_ROPE_YARN) {
        // the pair whose frequency makes beta turns over the original context
        auto at = [&](double beta) {
            return rot_dim * std::log(original_context / (beta * two_pi)) / (2.0 * std::log(theta));
        };
        y_lo = std::max(0.0, std::floor(at(high)));
        y_hi = std::min(rot_dim - 1.0, std::ceil(at(low)));
        if (!(y_hi > y_lo)) y_hi = y_lo + 0.001;
    }
    for (int p = 0; p < rot_dim / 2; ++p) {
        double f = std::pow(theta, -2.0 * p / rot_dim);
        if (scaling == B200Q_ROPE_LINEAR) {
            f /= factor;
        } else if (scaling == B200Q_ROPE_LLAMA3) {
            const double n = original_context * f / two_pi;  // turns over the original context
            if (n < low) {
                f /= factor;
            } else if (n <= high) {
                const double t = (n - low) / (high - low);
                f = (1.0 - t) * f / factor + t * f;
            }
        } else if (scaling == B200Q_ROPE_YARN) {
            const double t = std::min(1.0, std::max(0.0, (p - y_lo) / (y_hi - y_lo)));
            f = f / factor * t + f * (1.0 - t);
        }
        turns[p] = static_cast<unsigned long long>(std::ldexp(static_cast<long double>(f) / two_pi, 64) + 0.5L);
    }
    *mag = scaling == B200Q_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return B200Q_OK;
}

int launch_rope_rows(const void* x, void* out, int dtype, int rows, int heads, int hd, long long x_stride,
                     long long out_stride, const int* positions, const unsigned long long* turns, int rot, int layout,
                     double mag, Device* dev, cudaStream_t st) {
    if (!x || !out || !positions || !turns || rows < 0 || heads <= 0 || hd <= 0 || !dev) return B200Q_EINVAL;
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
    const bool wide = aligned_to(x, 4 * es) && aligned_to(out, 4 * es) && x_stride % 4 == 0 && out_stride % 4 == 0;
    const int v = rope_units(hd, rot, layout == B200Q_ROPE_HALF, wide, a.s);
    a.rows_per_cta = 1;
    a.heads_per_cta = heads;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ragged_cfg(dim3(rows, 1), dim3(kRopeThreads), st, attr);
    cudaError_t e;
    if (dtype == B200Q_F32)
        e = v == 4 ? cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<4, float>, a)
                   : cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<1, float>, a);
    else
        e = v == 4 ? cudaLaunchKernelEx(&cfg, b200q_rope_rows_kernel<4, __half>, a)
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
    if (!k || !v || !cu_q || !kv_len || n_tokens < 0 || batch <= 0 || !dev) return B200Q_EINVAL;
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
    const bool wide = !q_out || (aligned_to(q, 4 * es) && aligned_to(q_out, 4 * es) && q_stride % 4 == 0 &&
                                 q_out_stride % 4 == 0);
    const int vec = rope_units(hd, rot, layout == B200Q_ROPE_HALF, wide, a.s);
    a.heads_per_cta = heads;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ragged_cfg(dim3(n_tokens, 1), dim3(kRopeThreads), st, attr);
    const bool q8 = pkv.kv_mode == B200Q_KV_Q8;
    cudaError_t e;
#define B200Q_APPEND(V, T)                                                       \
    e = q8 ? cudaLaunchKernelEx(&cfg, b200q_rope_append_kernel<V, T, true>, a)   \
           : cudaLaunchKernelEx(&cfg, b200q_rope_append_kernel<V, T, false>, a)
    if (dtype == B200Q_F32) {
        if (vec == 4) B200Q_APPEND(4, float);
        else B200Q_APPEND(1, float);
    } else {
        if (vec == 4) B200Q_APPEND(4, __half);
        else B200Q_APPEND(1, __half);
    }
#undef B200Q_APPEND
    return e == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

}  // namespace b200q
