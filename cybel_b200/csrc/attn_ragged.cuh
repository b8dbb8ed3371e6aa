// Shared by the two kernels of b200q_attention_paged: the arguments, which
// positions a row sees, and how raw products become exponents.
#pragma once

#include "ragged.cuh"

namespace b200q {

struct AttnArgs {
    RaggedView r;
    PagedView kv;
    const void* q;
    void* out;
    const float* slopes;  // [heads] or NULL
    const int* prefix;    // [batch] or NULL
    long long q_stride, out_stride;
    int heads;
    int group;            // query heads per kv head
    int window;           // 0: none
    float scale, cap;     // cap 0: none
    uint32_t page_mul;    // position / page = div_by(position, page_mul, page_shift)
    int page_shift;
    uint32_t group_mul;   // the same of row / group
    int group_shift;
    int few_rows;         // sequences of at most this many rows (tokens x group) are the few-row kernel's
    int most_rows;        // of a sequence, as the caller says
    int row_blocks;       // few-row kernel: blocks of rows per sequence and kv head
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
// Codes + 128 (bytes of w ^ 0x80808080) as fp16 pairs: 0x64 above a byte u
// is 1024 + u exactly; less 1152 the code.
__device__ __forceinline__ uint32_t codes_fp16(uint32_t bytes, uint32_t sel) {
    const uint32_t h = __byte_perm(bytes, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// tanh(z) = z P(z^2) near 0, P minimax in the relative error by Remez's
// exchange: of degree 6 for |z| <= 1 (2^-24), or of degree 3 for |z| <= 1/2
// (2^-20.8: a score of 15 moves by 8e-6, a weight by as much relatively, which
// fp16 rounds by 2.4e-4).
template <bool PREC>
__device__ __forceinline__ float2 tanh_near(float2 z) {
    const float2 u = mul2(z, z);
    float2 p;
    if constexpr (PREC) {
        p = fma2(u, both(1.041022634e-03f), both(-6.203379105e-03f));
        p = fma2(p, u, both(2.028998042e-02f));
        p = fma2(p, u, both(-5.345702957e-02f));
        p = fma2(p, u, both(1.332520408e-01f));
        p = fma2(p, u, both(-3.333283915e-01f));
        p = fma2(p, u, both(9.999999502e-01f));
    } else {
        p = fma2(u, both(-4.440222613e-02f), both(1.319029660e-01f));
        p = fma2(p, u, both(-3.332631794e-01f));
        p = fma2(p, u, both(9.999994558e-01f));
    }
    return mul2(p, z);
}
// tanh(z) as 1 - 2 / (e^2z + 1) from two approximate instructions: off by 2^-22
// absolutely, which beyond 1 is as good as exact.
__device__ __forceinline__ float tanh_far(float z) {
    return 1.0f - 2.0f * rcp_fast(ex2(z * (2.0f * kLog2e)) + 1.0f);
}

// The smallest power of two above x (finite, >= 0), at least 2^-126.
__device__ __forceinline__ float pow2_above(float x) {
    const int e = min((__float_as_int(x) & 0x7f800000) + 0x00800000, 0x7f000000);
    return __int_as_float(e);
}

// What the rows of one tile of a sequence see: positions [0, pre) and, for
// the row at position i, [i - window + 1, i]; n positions in all.
struct Sight {
    int n, pre, window;
    int limit;  // positions that the page table reaches, n at most
    // First position of the range that the row at position i sees by itself.
    __device__ __forceinline__ int first(int i) const { return window > 0 ? max(0, i - window + 1) : 0; }
    // Last position that rows up to position hi see and the table reaches.
    __device__ __forceinline__ int last(int hi) const { return min(max(hi, pre - 1), limit - 1); }
    __device__ __forceinline__ bool sees(int i, int j) const { return j < pre || (j <= i && j >= first(i)); }
    // Whether every row at lo .. hi sees all of j0 .. j1.
    __device__ __forceinline__ bool all(int lo, int hi, int j0, int j1) const {
        return j1 < pre || (j1 <= lo && j0 >= first(hi));
    }
};

__device__ __forceinline__ Sight sight_of(const AttnArgs& a, int b) {
    Sight s;
    s.n = a.r.kv_len[b];
    s.limit = min(max(s.n, 0), a.kv.pages_per_seq * a.kv.page);
    s.pre = a.prefix ? min(max(a.prefix[b], 0), s.limit) : 0;
    s.window = a.window;
    return s;
}

// The tiles of T positions that rows at lo .. hi (lo <= hi, hi >= 0) need, in
// order: those of the prefix before the rows' own range, then that range.
template <int T>
struct TileList {
    int before, from, count;
    __device__ __forceinline__ TileList(const Sight& s, int lo, int hi) {
        from = s.first(max(lo, 0)) / T;
        before = min((s.pre + T - 1) / T, from);
        const int last = s.last(hi);
        count = before + max(0, last / T - from + (last >= 0));
    }
    __device__ __forceinline__ int at(int i) const { return (i < before ? i : from + i - before) * T; }
};

// Pool row of position j of sequence b, kv head h; kNoRow without one.
__device__ __forceinline__ uint32_t row_of(const AttnArgs& a, int b, int h, int j) {
    const int pg = div_by(j, a.page_mul, a.page_shift);
    const int slot = page_slot(a.kv, b, pg);
    if (slot < 0) {
        if (slot == -2) flag_bad_page(a.kv);
        return kNoRow;
    }
    return static_cast<uint32_t>(pool_row(a.kv, slot, h, j - pg * a.kv.page));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- clusters ----------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this CTA's shared address `a` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_peer2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ void store_out4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store_out4(__half* p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

int launch_attn_few(const AttnArgs& a, int hd, bool fp32, bool q8, int max_rows, int max_kv, int sms,
                    cudaStream_t st);

int launch_attn_tiles(const AttnArgs& a, int hd, bool fp32, bool q8, long long total_rows, int max_kv, int sms,
                      cudaStream_t st);
// Blocks of rows that the tile kernel is launched for, an upper bound of those
// there are (the lengths are on the device) ...
long long tile_blocks(int batch, long long total_rows, int most_rows, int few_rows);
// ... and the CTAs that split the positions of each.
int tile_split(long long units, int max_kv, int sms);
// The few-row kernel's split of `units` blocks, and the CTAs that run at once.
int few_split(long long units, int max_kv, int sms);
int few_slots(int sms);
// Rows of its blocks, where no sequence has more than max_rows of its rows.
int few_block_rows(bool fp32, int max_rows);

}  // namespace b200q
