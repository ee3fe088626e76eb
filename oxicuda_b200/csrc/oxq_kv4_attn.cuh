// What the kernels of attention over the 4-bit cache share: the call's parameters, a sequence's extent, the output row.
#pragma once
#include "oxq_kv4.cuh"

namespace oxq {
namespace kv4 {

struct AttnParams {
    Pool c;
    Batch s;
    const void* q; int64_t q_ts, q_hs; int q_vec;       // strides in elements; 16-byte loads allowed
    void* out; int64_t o_ts, o_hs;
    float* lse;                                         // [tokens][q_heads], or null
    int per, q_heads;                                   // query heads per kv head, all query heads
    FastDiv by_per;
    float scale_log2;                                   // scale * log2(e)
    int causal, window;                                 // window 0: none
    int row_limit, row_min;                             // sequences of at most row_limit rows (0: all) are the row kernel's, of more than row_min the tile kernel's
    int setup;                                          // row kernel: steps an item costs besides its tiles
    int parts, out_vec;                                 // tile kernel: CTAs that share an item's keys; 16-byte stores allowed
    float* ws;
    int32_t* status;
};

// An ordinary load that the compiler does not move or repeat (without it the few-rows kernel's main loop spills: 77 -> 80 us for
// 32 sequences of 50 to 16000 keys).
__device__ __forceinline__ int ld_word(const int32_t* at) {
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(at));
    return v;
}

// Sequence b: its first query token, how many of its tokens are in the call's rows, the position before its first one's, and
// how many keys the table can give.  Offsets and lengths come from the device and are held to their arrays here.
struct SeqInfo { int start, n, before, len; };
__device__ __forceinline__ SeqInfo seq_info(const AttnParams& p, int b) {
    SeqInfo q;
    const int a = ld_word(p.s.cu + b), e = ld_word(p.s.cu + b + 1), len = max(ld_word(p.s.lens + b), 0);
    const bool sound = a >= 0 && e >= a;
    q.start = a;
    q.n = sound && a < p.s.tokens ? (int)min((int64_t)(e - a), p.s.tokens - a) : 0;
    q.before = len - (sound ? e - a : 0);
    const int64_t most = p.s.width << p.c.page_shift;
    q.len = len > most ? (int)most : len;
    if (len > most && q.n > 0) *p.status = OXQ_ERR_INVALID_ARGUMENT;
    return q;
}

// The first position that the window of a query at `pos` holds (0 and less: all).  A query before position 0 sees nothing, wherever
// its window begins; it must only not wrap around.
__device__ __forceinline__ int window_start(const AttnParams& p, int pos) { return p.window > 0 ? max(pos + 1, 0) - p.window : 0; }

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two elements of an output row: row `row` of kv head `head` is query token row / per, query head head * per + row % per.
// o / sum, or zeros where nothing was seen; with the first two goes lse = ln(sum over keys of exp(score)).
template <typename T>
__device__ __forceinline__ void store_row(const AttnParams& p, const SeqInfo& q, int head, int row, int d, float2 o, float ref, float sum) {
    const int64_t t = q.start + p.by_per.div(row);
    const int qh = head * p.per + p.by_per.mod(row);
    const float inv = sum > 0.0f ? 1.0f / sum : sum != sum ? sum : 0.0f;
    struct alignas(4) Pair { T x, y; } v;
    v.x = Elem<T>::from_f32(o.x * inv);
    v.y = Elem<T>::from_f32(o.y * inv);
    *reinterpret_cast<Pair*>((T*)p.out + t * p.o_ts + (int64_t)qh * p.o_hs + d) = v;
    if (d == 0 && p.lse) p.lse[t * p.q_heads + qh] = sum > 0.0f || sum != sum ? (ref + log2f(sum)) * 0.693147180559945309417f : -INFINITY;
}

}  // namespace kv4
}  // namespace oxq

// Many query rows: oxq_kv4_tiles.cu.  `items` bounds the pairs of row blocks of all sequences.
int64_t oxq_kv4_tiles_slot_bytes(int dim);
int32_t oxq_kv4_tiles_launch(oxq_handle* h, const oxq_kv4_cache* cache, const oxq::kv4::AttnParams& p, int dtype, int64_t items);
