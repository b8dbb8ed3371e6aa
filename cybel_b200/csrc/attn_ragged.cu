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
// heads, fp16: 9 against 12; of 256: 17 against 14, the tile kernel's.) All of it
// for heads of 128 with plain scores and sequences of like lengths: heads of 64,
// caps, biases and lengths that differ do not enter the estimate.
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

// What a call launches, from its arguments alone.
struct AttnPlan {
    long long total_rows;
    int most_rows;  // of a sequence
    int few_rows;   // sequences of at most this many rows are the few-row kernel's
    int reach;      // positions that a block of rows has to read, for the splits
};

AttnPlan attention_plan(bool fp32, bool q8, int n_tokens, int batch, int max_q_len, int max_kv_len, int heads, int n_kv,
                        int window, bool prefix, int sms) {
    AttnPlan p;
    const int group = heads / n_kv, tokens = std::min(max_q_len, n_tokens);  // of a sequence
    p.total_rows = static_cast<long long>(n_tokens) * group;                 // at most 2^30
    p.most_rows = tokens * group;
    p.reach = window > 0 && !prefix
                  ? static_cast<int>(std::min<long long>(max_kv_len, static_cast<long long>(window) + tokens))
                  : max_kv_len;
    p.few_rows = few_rows(batch, n_kv, p.total_rows, p.most_rows, p.reach, fp32, q8, sms);
    return p;
}

}  // namespace

int launch_attention_paged(const void* q, int dtype, int n_tokens, int batch, const int* cu_q, const int* kv_len,
                           int max_q_len, int max_kv_len, int heads, int hd, long long q_stride, void* out,
                           long long out_stride, float scale, float softcap, const float* slopes, int window,
                           const int* prefix, const PagedKV& pkv, Device* dev, cudaStream_t st) {
    if (!cu_q || !kv_len || n_tokens < 0 || batch <= 0 || heads <= 0 || max_q_len < 0 || max_kv_len < 0 || !dev)
        return B200Q_EINVAL;
    if (n_tokens > 0 && (!q || !out)) return B200Q_EINVAL;  // (rows of no memory have no address)
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
    const AttnPlan p = attention_plan(fp32, q8, n_tokens, batch, max_q_len, max_kv_len, heads, pkv.n_kv, window,
                                      prefix != nullptr, dev->num_sms);
    a.most_rows = p.most_rows;
    a.few_rows = p.few_rows;
    rc = launch_attn_few(a, hd, fp32, q8, std::min(a.most_rows, a.few_rows), p.reach, dev->num_sms, st);
    if (rc != B200Q_OK || a.most_rows <= a.few_rows) return rc;
    return launch_attn_tiles(a, hd, fp32, q8, p.total_rows, p.reach, dev->num_sms, st);
}

int attention_plan_info(int dtype, int n_tokens, int batch, int max_q_len, int max_kv_len, int heads, int n_kv,
                        int window, bool prefix, int kv_mode, int num_sms, long long* out, int out_len) {
    const bool q8 = kv_mode == B200Q_KV_Q8, fp32 = dtype == B200Q_F32;
    if (!out || out_len < kAttnPlanFields || n_tokens <= 0 || batch <= 0 || max_q_len <= 0 || max_kv_len < 0 ||
        heads <= 0 || n_kv <= 0 || window < 0 || num_sms <= 0 || (!fp32 && dtype != B200Q_F16) ||
        (!q8 && kv_mode != B200Q_KV_F16))
        return B200Q_EINVAL;
    if (heads % n_kv || static_cast<long long>(n_tokens) * (heads / n_kv) > (1 << 30)) return B200Q_ESHAPE;
    const AttnPlan p =
        attention_plan(fp32, q8, n_tokens, batch, max_q_len, max_kv_len, heads, n_kv, window, prefix, num_sms);
    const int few = std::min(p.most_rows, p.few_rows), rows = few_block_rows(fp32, few);
    out[0] = p.few_rows;
    out[1] = few_split(static_cast<long long>(batch) * n_kv * ((few + rows - 1) / rows), p.reach, num_sms);
    const long long blocks =
        p.most_rows > p.few_rows ? tile_blocks(batch, p.total_rows, p.most_rows, p.few_rows) * n_kv : 0;
    out[2] = blocks;
    out[3] = blocks > 0 ? tile_split(blocks, p.reach, num_sms) : 0;
    return B200Q_OK;
}

}  // namespace b200q
