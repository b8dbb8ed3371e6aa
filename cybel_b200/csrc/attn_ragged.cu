// Attention of a ragged batch of query tokens over a paged cache.
//
// For the token at position i of sequence b and query head h (kv head
// h / (n_heads / n_kv)), over the visible positions j:
//
//     s_j = scale * q . k_j;  s_j = cap * tanh(s_j / cap)  (cap > 0);
//     s_j -= slope_h * |i - j|;                     o = sum_j softmax(s)_j v_j
//
// j is visible when j < kv_len, its page is assigned, and j <= i with
// i - j < window (window > 0), or j < prefix_b. A row that sees nothing is 0.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_ragged.cuh"
#include "internal.h"

namespace b200q {

namespace {

__device__ __forceinline__ float4 kv_quad(const __half* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 kv_quad(const int8_t* p) {
    const char4 x = *reinterpret_cast<const char4*>(p);
    return make_float4(x.x, x.y, x.z, x.w);
}

// One warp per row and query head, D / 4 lanes per key: the plain running
// softmax, in fp32 throughout.
template <int D, typename T, bool Q8>
__global__ void __launch_bounds__(128) b200q_attn_rows_kernel(const AttnArgs a) {
    using KV = typename std::conditional<Q8, int8_t, __half>::type;
    griddep_launch_dependents();
    griddep_wait();
    constexpr int L = D / 4;       // lanes per key
    constexpr int KPW = 32 / L;    // keys a warp scores at once
    const int row = blockIdx.x;
    const int head = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, sub = lane / L, e = (lane % L) * 4;
    if (head >= a.heads) return;
    const int b = seq_of_row(a.r, row);
    if (b < 0) return;
    const int2 rr = seq_rows(a.r, b);
    if ((rr.y - rr.x) * a.group <= a.few_rows) return;
    const int n = a.r.kv_len[b];
    const int pos = n - (rr.y - row);
    const int kvh = head / (a.heads / a.kv.n_kv);
    const T* qp = static_cast<const T*>(a.q) + row * a.q_stride + head * D + e;
    float4 q;
    q.x = static_cast<float>(qp[0]), q.y = static_cast<float>(qp[1]);
    q.z = static_cast<float>(qp[2]), q.w = static_cast<float>(qp[3]);
    const int pre = a.prefix ? min(max(a.prefix[b], 0), n) : 0;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int part = 0; part < 2; ++part) {
        const int lo = part == 0 ? 0 : max(first, pre);
        const int hi = part == 0 ? pre : pos + 1;
        for (int j0 = lo; j0 < hi; j0 += KPW) {
            const int j = j0 + sub;
            int slot = -1;
            if (j < hi) {
                slot = page_slot(a.kv, b, j / a.kv.page);
                if (slot == -2) flag_bad_page(a.kv);
            }
            const bool see = slot >= 0;
            const long long r = see ? pool_row(a.kv, slot, kvh, j % a.kv.page) : 0;
            float s = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (see) {
                const float4 k = kv_quad(static_cast<const KV*>(a.kv.k) + r * D + e);
                v = kv_quad(static_cast<const KV*>(a.kv.v) + r * D + e);
                s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
                if constexpr (Q8) {
                    s *= a.kv.ks[r];
                    const float vs = a.kv.vs[r];
                    v.x *= vs, v.y *= vs, v.z *= vs, v.w *= vs;
                }
            }
#pragma unroll
            for (int w = L / 2; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
            s *= a.scale;
            if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
            s -= slope * fabsf(static_cast<float>(pos - j));
            if (see) {
                const float mn = fmaxf(m, s);
                const float f = mn == -INFINITY ? 1.0f : expf(m - mn), p = mn == -INFINITY ? 0.0f : expf(s - mn);
                m = mn;
                l = l * f + p;
                o.x = o.x * f + p * v.x, o.y = o.y * f + p * v.y;
                o.z = o.z * f + p * v.z, o.w = o.w * f + p * v.w;
            }
        }
    }
    if constexpr (KPW > 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m, L);
        const float mn = fmaxf(m, mo);
        const float f = m == -INFINITY ? 0.0f : expf(m - mn);
        l *= f;
        l += __shfl_xor_sync(0xffffffffu, l, L);
        float* c = &o.x;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            c[t] *= f;
            c[t] += __shfl_xor_sync(0xffffffffu, c[t], L);
        }
    }
    if (sub) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + head * D + e;
    out[0] = static_cast<T>(o.x * inv), out[1] = static_cast<T>(o.y * inv);
    out[2] = static_cast<T>(o.z * inv), out[3] = static_cast<T>(o.w * inv);
}

}  // namespace

// Sequences with at most this many rows (tokens x query heads per kv head)
// are the few-row kernel's.
constexpr int kFewRows = 64;

int launch_attention_paged(const void* q, int dtype, int n_tokens, int batch, const int* cu_q, const int* kv_len,
                           int max_q_len, int max_kv_len, int heads, int hd, long long q_stride, void* out,
                           long long out_stride, float scale, float softcap, const float* slopes, int window,
                           const int* prefix, const PagedKV& pkv, Device* dev, cudaStream_t st) {
    if (!q || !out || !cu_q || !kv_len || n_tokens < 0 || batch <= 0 || heads <= 0 || max_q_len < 0 || max_kv_len < 0 ||
        !dev)
        return B200Q_EINVAL;
    if (dtype != B200Q_F32 && dtype != B200Q_F16) return B200Q_EINVAL;
    if (!(scale > 0.0f) || !std::isfinite(scale) || !(softcap >= 0.0f) || !std::isfinite(softcap) || window < 0)
        return B200Q_EINVAL;
    int rc = check_paged(pkv, hd);
    if (rc != B200Q_OK) return rc;
    const long long qw = static_cast<long long>(heads) * hd;
    if (heads % pkv.n_kv || qw > (1 << 30)) return B200Q_ESHAPE;
    if (q_stride == 0) q_stride = qw;
    if (out_stride == 0) out_stride = qw;
    if (q_stride < qw || out_stride < qw) return B200Q_ESHAPE;
    const uintptr_t align = 15;
    const long long es = dtype == B200Q_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(q) & align) || (reinterpret_cast<uintptr_t>(out) & align) ||
        ((q_stride * es) & 15) || ((out_stride * es) & 15) || (reinterpret_cast<uintptr_t>(cu_q) & 3) ||
        (reinterpret_cast<uintptr_t>(kv_len) & 3) || (reinterpret_cast<uintptr_t>(slopes) & 3) ||
        (reinterpret_cast<uintptr_t>(prefix) & 3))
        return B200Q_EALIGN;
    if (n_tokens == 0 || max_q_len == 0) return B200Q_OK;
    AttnArgs a{};
    a.r = RaggedView{cu_q, kv_len, batch, n_tokens};
    a.kv = paged_view(pkv, dev);
    a.q = q;
    a.out = out;
    a.slopes = slopes;
    a.prefix = prefix;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.heads = heads;
    a.window = window;
    a.scale = scale;
    a.cap = softcap;
    a.group = heads / pkv.n_kv;
    while ((1ll << a.page_shift) < pkv.page_size) ++a.page_shift;
    a.page_mul = static_cast<uint32_t>(((1ull << (31 + a.page_shift)) + pkv.page_size - 1) / pkv.page_size);
    a.few_rows = kFewRows;
    const bool q8 = pkv.kv_mode == B200Q_KV_Q8;
    const long long most = static_cast<long long>(max_q_len < n_tokens ? max_q_len : n_tokens) * a.group;
    rc = launch_attn_few(a, hd, dtype == B200Q_F32, q8, static_cast<int>(std::min<long long>(most, kFewRows)), max_kv_len, st);
    if (rc != B200Q_OK || most <= kFewRows) return rc;
    const dim3 grid(n_tokens, (heads + 3) / 4);
    auto go = [&](auto kern) { kern<<<grid, 128, 0, st>>>(a); };
    if (hd == 128) {
        if (dtype == B200Q_F32) q8 ? go(b200q_attn_rows_kernel<128, float, true>) : go(b200q_attn_rows_kernel<128, float, false>);
        else q8 ? go(b200q_attn_rows_kernel<128, __half, true>) : go(b200q_attn_rows_kernel<128, __half, false>);
    } else {
        if (dtype == B200Q_F32) q8 ? go(b200q_attn_rows_kernel<64, float, true>) : go(b200q_attn_rows_kernel<64, float, false>);
        else q8 ? go(b200q_attn_rows_kernel<64, __half, true>) : go(b200q_attn_rows_kernel<64, __half, false>);
    }
    return cudaGetLastError() == cudaSuccess ? B200Q_OK : B200Q_ECUDA;
}

}  // namespace b200q
