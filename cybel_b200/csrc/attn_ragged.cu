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

#include "attn_ragged.cuh"
#include "internal.h"

namespace b200q {

namespace {

// Sequences with at most this many rows (tokens x query heads per kv head) are
// the few-row kernel's, the others the tile kernel's. Up to 32 rows the few-row
// kernel is as fast or faster at any batch (fp16, 8 tokens of 4 heads per kv
// head at 2000 positions: 12 against 24 us for 1 sequence, 79 against 78 for
// 32); at 64 rows only while its blocks of rows leave SMs idle (16 tokens: 14
// against 25 us for 1 sequence, 32 against 28 for 4, 135 against 78 for 32).
int few_rows(long long heads, bool fp32, int sms) {
    const int blocks = 64 / (fp32 ? 8 : 16);
    return heads * blocks <= sms ? 64 : 32;
}

}  // namespace

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
    if (static_cast<long long>(n_tokens) * (heads / pkv.n_kv) > (1 << 30)) return B200Q_ESHAPE;  // rows are ints
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
    divisor(pkv.page_size, a.page_mul, a.page_shift);
    divisor(a.group, a.group_mul, a.group_shift);
    a.few_rows = few_rows(static_cast<long long>(batch) * pkv.n_kv, dtype == B200Q_F32, dev->num_sms);
    const bool q8 = pkv.kv_mode == B200Q_KV_Q8;
    const long long most = static_cast<long long>(max_q_len < n_tokens ? max_q_len : n_tokens) * a.group;
    rc = launch_attn_few(a, hd, dtype == B200Q_F32, q8, static_cast<int>(std::min<long long>(most, a.few_rows)),
                         max_kv_len, dev->num_sms, st);
    if (rc != B200Q_OK || most <= a.few_rows) return rc;
    return launch_attn_tiles(a, hd, dtype == B200Q_F32, q8, static_cast<long long>(n_tokens) * a.group, max_kv_len,
                             dev->num_sms, st);
}

}  // namespace b200q
