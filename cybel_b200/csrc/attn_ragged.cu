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
// kernel is as fast or faster at any batch (8 tokens of 4 heads per kv head at
// 2000 positions, fp16: 12 against 19 us for 1 sequence, 80 against 79 for 32).
// Beyond, whichever comes out ahead by what their times follow, as measured at
// 8 kv heads, 1 to 4 sequences of 48 to 256 rows and 300 to 8000 positions, and
// at 1 to 8 kv heads with up to 4000 rows: the
// few-row kernel's the positions of a CTA and its waves, the tile kernel's the
// steps of a CTA, however full its tiles are. (24 tokens of 4 heads per kv head
// at 2000 positions: fp32 26 against 35 us for 2 sequences, 50 against 52 for 4;
// fp16 14 against 19 for 1, 29 against 25 for 4. Of 360 such batches two take
// the kernel that is slower by more than 8 percent, by 20 at most. A prompt of
// 600 tokens on one kv head, 4 heads, fp32: 21 against 34 us; of 128 tokens, 32/8
// heads, fp16: 9 against 12; of 256: 17 against 14, the tile kernel's.)
int few_rows(int batch, int n_kv, long long total_rows, int most, int max_kv, bool fp32, bool q8, int sms) {
    if (most <= 32) return 32;
    const long long fu = static_cast<long long>(batch) * n_kv * ((most + (fp32 ? 7 : 15)) / (fp32 ? 8 : 16));
    const int fc = few_split(fu, max_kv, sms);
    const long long fw = (fu * fc + few_slots(sms) - 1) / few_slots(sms);
    const double few_us = 3.0 + static_cast<double>(fw) * (6.0 + (fp32 ? 0.018 : 0.021) * max_kv / fc);
    const long long tu = tile_blocks(batch, total_rows, most, 32) * n_kv;
    const int tc = tile_split(tu, max_kv, sms);
    const long long steps = (max_kv + 128ll * tc - 1) / (128 * tc), tw = (tu * tc + sms - 1) / sms;
    const double step_us = fp32 ? (q8 ? 6.8 : 5.4) : (q8 ? 3.2 : 2.2);
    return few_us < (fp32 ? 16.0 : 11.0) + step_us * static_cast<double>(steps * tw) ? most : 32;
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
    const bool q8 = pkv.kv_mode == B200Q_KV_Q8, fp32 = dtype == B200Q_F32;
    const long long total_rows = static_cast<long long>(n_tokens) * a.group;  // at most 2^30
    const int tokens = std::min(max_q_len, n_tokens);                        // of a sequence
    a.most_rows = tokens * a.group;
    // Positions that a row block has to read, for the splits below.
    const int reach = window > 0 && !prefix ? static_cast<int>(std::min<long long>(max_kv_len, static_cast<long long>(window) + tokens))
                                            : max_kv_len;
    a.few_rows = few_rows(batch, pkv.n_kv, total_rows, a.most_rows, reach, fp32, q8, dev->num_sms);
    rc = launch_attn_few(a, hd, fp32, q8, std::min(a.most_rows, a.few_rows), reach, dev->num_sms, st);
    if (rc != B200Q_OK || a.most_rows <= a.few_rows) return rc;
    return launch_attn_tiles(a, hd, fp32, q8, total_rows, reach, dev->num_sms, st);
}

}  // namespace b200q
