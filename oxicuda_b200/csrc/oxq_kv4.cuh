// The paged 4-bit key / value cache: layout, and what its kernels share.
//
// A pool holds `pages` pages of `page` tokens of every kv head, head-major, so that one head's tokens of a page are
// contiguous: codes [pages][heads][page][D / 2] bytes, params [pages][heads][page][D / G] pairs of f16 (s, m).  A group
// of G consecutive elements of a row (one head of one token) stands for c * s + m.  A row is D / 8 words of eight codes
// (element e of a word at bits [4 e, 4 e + 4)); the words are transposed inside the row:
//   keys    word 4 i + c lies at place c * (D / 32) + i: lane c of a quad finds its share of every 32-element block of
//           the score product in one 16-byte load, and a matrix instruction never mixes two scale groups;
//   values  word 8 i + r lies at place r * (D / 64) + i: lane row r finds its elements of every 64-element block of the
//           weighted sum in one load.
//
// None of the kernels reads through the read-only path: the pool, the queries and the batch's arrays are what earlier kernels of
// the stream write, and with programmatic launches a kernel is resident while they do.
#pragma once
#include "oxq_common.cuh"

namespace oxq {
namespace kv4 {

// n / d for 0 <= n < 2^31 by a product: mul = ceil(2^(32 + shift) / d) with 2^(shift + 1) >= d is exact in that range; d = 1 apart.
struct FastDiv {
    uint32_t mul; int shift, d;
    void set(int div) {
        d = div;
        shift = 0;
        while ((2ll << shift) < div) shift++;
        mul = div == 1 ? 0u : (uint32_t)((((unsigned long long)1 << (32 + shift)) + (unsigned)div - 1) / (unsigned)div);
    }
    __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
    __device__ __forceinline__ int mod(int n) const { return n - div(n) * d; }
};

struct Pool {
    uint8_t* kc; uint32_t* kp;          // params as packed pairs: s in the low half, m in the high half
    uint8_t* vc; uint32_t* vp;
    int64_t pages;
    int page_shift;                     // page size is a power of two
    int heads;
};

// The call's tokens: sequence b owns tokens cu[b] .. cu[b + 1], the last of them at position lens[b] - 1.
struct Batch {
    const int32_t* table; int64_t width;
    const int32_t* lens;
    const int32_t* cu;
    int seqs;
    int64_t tokens;
};

__device__ __forceinline__ int key_place(int word, int dim) { return (word & 3) * (dim >> 5) + (word >> 2); }
__device__ __forceinline__ int value_place(int word, int dim) { return (word & 7) * (dim >> 6) + (word >> 3); }

// Row index of (position, head) in a pool, or -1 where the table gives no page of the pool.
__device__ __forceinline__ int64_t pool_row(const Pool& c, const Batch& s, int b, int64_t pos, int head, int32_t* status) {
    const int64_t entry = pos >> c.page_shift;
    int64_t page = -1;
    if (pos >= 0 && entry < s.width) page = s.table[(int64_t)b * s.width + entry];
    if (page < 0 || page >= c.pages) {
        if (pos >= 0 && status) *status = OXQ_ERR_INVALID_ARGUMENT;
        return -1;
    }
    return ((page * c.heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

// Smallest b with cu[b + 1] > t (seqs if there is none), found by a whole warp: 32 probes a round.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int seqs, int64_t t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;
    while (hi > lo) {
        const int step = (hi - lo + 31) >> 5;
        const int i = lo + lane * step + step - 1;
        const bool before = i < hi && cu[i + 1] <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, before));
        const int nlo = min(hi, lo + c * step);
        hi = min(hi, nlo + step - 1);
        lo = nlo;
    }
    return lo;
}

}  // namespace kv4
}  // namespace oxq

// Host: checks a cache and a batch descriptor and fills the device forms.  Defined in oxq_kv4.cu.
int32_t oxq_kv4_check(oxq_handle* h, const oxq_kv4_cache* cache, const oxq_kv4_batch* batch, oxq::kv4::Pool* pool, oxq::kv4::Batch* b);
