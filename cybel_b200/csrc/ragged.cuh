// Shared by the ragged-batch kernels (rotary rows, paged append, paged
// attention): the views of a batch of sequences of different lengths and of
// a paged cache, and the lookups in them.
//
// Token t of sequence b (rows cu_q[b] .. cu_q[b + 1] of the batch's rows)
// sits at position kv_len[b] - q_len[b] + t: the batch's tokens are the last
// ones of their sequences. The arrays live on the device and are read by the
// kernels only, so a captured graph replays with new lengths.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr uint32_t kNoRow = 0xFFFFFFFFu;  // a pool row that is none

struct RaggedView {
    const int* cu_q;    // [batch + 1] first row of each sequence
    const int* kv_len;  // [batch] positions of the sequence, this batch's tokens included
    int batch;
    int n_tokens;       // rows that q, k, v and the outputs hold
};

struct PagedView {
    void* k;            // [n_slots][n_kv][page][hd] fp16 or int8 codes
    void* v;
    float* ks;          // [n_slots][n_kv][page] (Q8)
    float* vs;
    const int* table;   // [batch][pages_per_seq] slots, -1: no page
    int pages_per_seq;
    int page;
    int n_slots;
    int n_kv;
    volatile int* status;
};

// x / d for 0 <= x < 2^31: umulhi(2 x, mul) >> shift, shift = ceil(log2 d), mul
// = ceil(2^(31 + shift) / d) (its excess e < d adds less than x e / (d
// 2^(31 + shift)) < 1 / d to the quotient).
__device__ __forceinline__ int div_by(int x, uint32_t mul, int shift) {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(x), mul) >> shift);
}

inline void divisor(int d, uint32_t& mul, int& shift) {
    shift = 0;
    while ((1ll << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << (31 + shift)) + d - 1) / d);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Rows of sequence b, clamped to the rows that exist (cu_q is the caller's).
__device__ __forceinline__ int2 seq_rows(const RaggedView& r, int b) {
    const int lo = min(max(r.cu_q[b], 0), r.n_tokens);
    const int hi = min(max(r.cu_q[b + 1], lo), r.n_tokens);
    return make_int2(lo, hi);
}

// Pool slot of page `pg` of sequence b: -1 for a page not assigned, -2 for
// an entry that names none of the pool's slots or a page past the table.
__device__ __forceinline__ int page_slot(const PagedView& kv, int b, int pg) {
    if (pg < 0 || pg >= kv.pages_per_seq) return -2;
    const int s = kv.table[static_cast<long long>(b) * kv.pages_per_seq + pg];
    return s >= 0 && s < kv.n_slots ? s : (s == -1 ? -1 : -2);
}

__device__ __forceinline__ void flag_bad_page(const PagedView& kv) {
    kv.status[kBadPageWord] = STATUS_BAD_PAGE;
}

// Row index (of hd elements, or of one scale) of position `off` of a page.
__device__ __forceinline__ long long pool_row(const PagedView& kv, int slot, int head, int off) {
    return (static_cast<long long>(slot) * kv.n_kv + head) * kv.page + off;
}

}  // namespace b200q
