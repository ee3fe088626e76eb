// Writing tokens into the paged 4-bit key / value cache, and reading them back (layout: oxq_kv4.cuh).
//
// Quantizer, per group of G elements of one head of one token:
//   s = f16((max - min) / 15), m = f16(min), c = clamp(rint((x - m) / s), 0, 15), and c = 0 where s is 0.
// The codes are computed from the rounded s and m, the numbers the reader uses, so rounding them costs no accuracy in the
// codes.  s and m stay f16 (4 bytes a group): the offset is a float, not a zero-point in code units, because a group whose
// values all lie on one side of zero must keep its four bits for its own range.
//
// What bounds them: appending, 8192 tokens of 8 heads, keys and values, takes 18 us where the bytes need 6.6.  No pipe is full
// (issue 0.67 of the cycles, logic 0.53): an instruction takes 9.9 cycles of a warp, 3.0 of them waits for rows, and 26 of 64
// warps are there; what is missing are rows on their way.  Reading: memory (131k tokens: 125 us = 5.6 TB/s, 0.86 of the copy
// rate).
#include "oxq_kv4.cuh"

namespace oxq {
namespace kv4 {

template <typename T> struct Packed;
template <> struct Packed<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Packed<__half> { using type = __half2; };

template <typename T>
struct Rows {
    const T* p[2];                      // keys, values
    int64_t token_stride[2], head_stride[2];
    int vec;                            // 16-byte loads are aligned
};

// How the warps walk the call.  A warp takes `each` (at most 32) tokens; lane j finds the place of token first + j, and the lanes
// ask it for that place.  A step is 32 words of one token, or the words of `beside` whole tokens where a token has fewer; a
// token has `rounds` of them.  `share` warps take turns at the steps of the same tokens.
struct Walk { int each, share, beside, rounds; };
// A lane's part of every step: which of the tokens beside each other, its word of the row (the same in every round, 32 being a
// multiple of a row's words) and the word's head and place in the token.
template <int D> struct Lane {
    int next_to, word, head, at;
    bool real;
    __device__ __forceinline__ Lane(const Walk& w, int words) {
        const int lane = threadIdx.x & 31;
        next_to = w.beside > 1 ? lane / words : 0;
        at = lane - next_to * words;
        word = at % (D / 8);
        head = at / (D / 8);
        real = next_to < w.beside;
    }
};

constexpr int64_t NO_PLACE = -1, NO_SEQUENCE = -2;
__device__ __forceinline__ int64_t place_of(const Pool& c, const Batch& s, int64_t first, int each, int32_t* status) {
    int b = sequence_of(s.cu, s.seqs, first);
    const int64_t t = first + (threadIdx.x & 31);
    if ((int)(threadIdx.x & 31) >= each || t >= s.tokens) return NO_SEQUENCE;
    while (b < s.seqs && s.cu[b + 1] <= t) b++;
    if (b >= s.seqs || t < s.cu[b]) return NO_SEQUENCE;
    return pool_row(c, s, b, (int64_t)s.lens[b] - s.cu[b + 1] + t, 0, status);
}

// Eight elements as they lie.
template <typename T> struct Eight { uint32_t w[sizeof(T) * 2]; };
template <typename T> __device__ __forceinline__ void load8(const T* p, int vec, Eight<T>& r) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const Vec16<uint32_t> v = ld16_written_stream(reinterpret_cast<const uint32_t*>(p) + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) r.w[4 * i + e] = v.v[e];
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 8; e++) r.w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) r.w[e] = (uint32_t)h[2 * e] | ((uint32_t)h[2 * e + 1] << 16);
    }
}
template <typename T> __device__ __forceinline__ float element(const Eight<T>& r, int e) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[e]);
    else if constexpr (Elem<T>::kDtype == OXQ_BF16) return __uint_as_float(e & 1 ? r.w[e / 2] & 0xFFFF0000u : r.w[e / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(r.w[e / 2] >> (16 * (e & 1)))));
}
// Whether an element is beyond f16's range (s and m are f16), infinite or NaN.
template <typename T> __device__ __forceinline__ bool beyond(const Eight<T>& r) {
    if constexpr (sizeof(T) == 4) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; e++) any |= !(fabsf(__uint_as_float(r.w[e])) <= 65504.0f);
        return any;
    } else {
        uint32_t m = r.w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int e = 1; e < 4; e++) m = __vmaxu2(m, r.w[e] & 0x7FFF7FFFu);
        const uint32_t top = max(m & 0xFFFFu, m >> 16);
        return top > (Elem<T>::kDtype == OXQ_BF16 ? 0x477Fu : 0x7BFFu);              // the largest bf16 below 65504, the largest f16
    }
}
// Smallest and largest of the group that W neighbouring lanes hold eight elements of each.  16-bit types stay packed: the pair
// (smallest, -largest) takes one shuffle and one packed minimum a step.
template <typename T, int W> __device__ __forceinline__ void group_range(const Eight<T>& r, float& lo, float& hi) {
    if constexpr (sizeof(T) == 4) {
        lo = hi = __uint_as_float(r.w[0]);
#pragma unroll
        for (int e = 1; e < 8; e++) { lo = fminf(lo, __uint_as_float(r.w[e])); hi = fmaxf(hi, __uint_as_float(r.w[e])); }
#pragma unroll
        for (int o = 1; o < W; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
    } else {
        using T2 = typename Packed<T>::type;
        const auto pack = [](uint32_t v) { return *reinterpret_cast<T2*>(&v); };
        const auto bits = [](T2 v) { return *reinterpret_cast<uint32_t*>(&v); };
        T2 l = __hmin2(__hmin2(pack(r.w[0]), pack(r.w[1])), __hmin2(pack(r.w[2]), pack(r.w[3])));
        T2 h = __hmax2(__hmax2(pack(r.w[0]), pack(r.w[1])), __hmax2(pack(r.w[2]), pack(r.w[3])));
        const uint32_t lb = bits(l), hb = bits(h) ^ 0x80008000u;
        uint32_t v = bits(__hmin2(pack(__byte_perm(lb, hb, 0x5410)), pack(__byte_perm(lb, hb, 0x7632))));
#pragma unroll
        for (int o = 1; o < W; o <<= 1) v = bits(__hmin2(pack(v), pack(__shfl_xor_sync(0xffffffffu, v, o))));
        Eight<T> e; e.w[0] = v;
        lo = element(e, 0);
        hi = -element(e, 1);
    }
}

// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ void split(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// Eight elements of a lane to a word of codes and, the same in all lanes of the group, its (s, m).
template <typename T, int G> __device__ __forceinline__ void quantize8(const Eight<T>& x, uint32_t& codes, uint32_t& params) {
    float lo, hi, f[8];
    if (__any_sync(0xffffffffu, beyond(x))) {            // NaN counts as 0, the rest is held to +-65504
#pragma unroll
        for (int e = 0; e < 8; e++) {
            f[e] = element(x, e);
            f[e] = f[e] != f[e] ? 0.0f : fminf(fmaxf(f[e], -65504.0f), 65504.0f);
            lo = e ? fminf(lo, f[e]) : f[e];
            hi = e ? fmaxf(hi, f[e]) : f[e];
        }
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = element(x, e);
        group_range<T, G / 8>(x, lo, hi);
    }
    // range / 15 and (x - m) / s, correctly rounded by a reciprocal and one correction (Markstein; see InvDiv; a range too
    // small for that to hold is one that f16 rounds to 0, and s is 0 or in [2^-24, 8736]); the quotients held to
    // [0, 15]; rounded half to even by adding 1.5 * 2^23; four codes make a number below 2^16, which f32 holds exactly.
    const float range = hi - lo, fifteenth = 1.0f / 15.0f, s0 = range * fifteenth;
    const __half sh = __float2half_rn(fmaf(fmaf(-15.0f, s0, range), fifteenth, s0)), mh = __float2half_rn(lo);
    const float sc = __half2float(sh), m = __half2float(mh), y = __frcp_rn(sc);
    constexpr float kMagic = 12582912.0f;
    const uint64_t m2 = pair(-m, -m), y2 = pair(y, y), s2 = pair(-sc, -sc), up = pair(kMagic, kMagic), down = pair(-kMagic, -kMagic);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint64_t d = add2(pair(f[e], f[e + 1]), m2), q0 = mul2(d, y2);
        float a, b;
        split(fma2(fma2(s2, q0, d), y2, q0), a, b);
        const uint64_t r = add2(add2(pair(fminf(fmaxf(a, 0.0f), 15.0f), fminf(fmaxf(b, 0.0f), 15.0f)), up), down);
        sum[e >> 2] = fma2(r, e & 2 ? pair(256.0f, 4096.0f) : pair(1.0f, 16.0f), sum[e >> 2]);
    }
    float half[2];
#pragma unroll
    for (int h = 0; h < 2; h++) { float a, b; split(sum[h], a, b); half[h] = a + b; }
    codes = (__float_as_uint(half[0] + 8388608.0f) & 0xFFFFu) | (__float_as_uint(half[1] + 8388608.0f) << 16);
    if (!(sc > 0.0f)) codes = 0;
    params = (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(mh) << 16);
}

template <typename T, int D, int G, int U, bool KEYS>
__device__ __forceinline__ void append_rows(const Pool& c, const Batch& s, const Rows<T>& in, const Walk& walk, int32_t* status) {
    const int words = c.heads * (D / 8), warp = blockIdx.x * 8 + (threadIdx.x >> 5);          // words of a token
    const int64_t first = (int64_t)(warp / walk.share) * walk.each;
    if (first >= s.tokens) return;                                  // whole warps
    const int64_t mine = place_of(c, s, first, walk.each, status);
    const Lane<D> lane(walk, words);
    const int64_t token_stride = in.token_stride[KEYS ? 0 : 1], round_stride = 256 / D * in.head_stride[KEYS ? 0 : 1];
    const int64_t round_rows = (int64_t)(256 / D) << c.page_shift;  // rows of the pool from one round to the next
    const T* base = in.p[KEYS ? 0 : 1] + (first + lane.next_to) * token_stride + lane.head * in.head_stride[KEYS ? 0 : 1] + lane.word * 8;
    uint32_t* codes_at = reinterpret_cast<uint32_t*>(KEYS ? c.kc : c.vc) + (KEYS ? key_place(lane.word, D) : value_place(lane.word, D));
    uint32_t* params_at = (KEYS ? c.kp : c.vp) + lane.word / (G / 8);
    const bool leads = lane.word % (G / 8) == 0;
    for (int j0 = 0, t0 = 0; t0 < walk.each; j0 += U, t0 += U * walk.beside) {
        int64_t at[U];                                              // row in the pool, below 0: none
        const T* from[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int tok = t0 + u * walk.beside + lane.next_to;
            at[u] = __shfl_sync(0xffffffffu, mine, tok & 31);
            if (!lane.real || tok >= walk.each) at[u] = NO_PLACE;
            if (at[u] >= 0) at[u] += (int64_t)lane.head << c.page_shift;
            from[u] = base + (t0 + u * walk.beside) * token_stride;
        }
        // the rounds of a token; where several warps share the tokens, every share-th step is this one's
        for (int k = 0; k < walk.rounds; k++) {
            if (U == 1 && walk.share > 1 && (j0 * walk.rounds + k) % walk.share != warp % walk.share) continue;
            const bool inside = lane.at + 32 * k < words;
            Eight<T> x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int e = 0; e < (int)sizeof(T) * 2; e++) x[u].w[e] = 0;
                if (inside && at[u] >= 0) load8(from[u] + k * round_stride, in.vec, x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint32_t codes, params;
                quantize8<T, G>(x[u], codes, params);
                if (inside && at[u] >= 0) {
                    const int64_t row = at[u] + k * round_rows;
                    codes_at[row * (D / 8)] = codes;
                    if (leads) params_at[row * (D / G)] = params;
                }
            }
        }
    }
}
template <typename T, int D, int G, int U>
__global__ void __launch_bounds__(256) kv4_append_kernel(Pool c, Batch s, Rows<T> in, Walk walk, int32_t* status) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.y == 0) append_rows<T, D, G, U, true>(c, s, in, walk, status);
    else append_rows<T, D, G, U, false>(c, s, in, walk, status);
}

// c * s + m in f32: c * s is exact (4 + 11 bits), so there is one rounding, and one more to T.  The words come out in the
// order of the output's elements.
template <typename T, int D, int G, int U, bool KEYS>
__device__ __forceinline__ void read_rows(const Pool& c, const Batch& s, T* rows_out, const Walk& walk, int32_t* status) {
    const int words = c.heads * (D / 8), warp = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t first = (int64_t)(warp / walk.share) * walk.each;
    if (first >= s.tokens) return;
    const int64_t mine = place_of(c, s, first, walk.each, status);
    const Lane<D> lane(walk, words);
    const int64_t round_rows = (int64_t)(256 / D) << c.page_shift;
    const uint32_t* codes_at = reinterpret_cast<const uint32_t*>(KEYS ? c.kc : c.vc) + (KEYS ? key_place(lane.word, D) : value_place(lane.word, D));
    const uint32_t* params_at = (KEYS ? c.kp : c.vp) + lane.word / (G / 8);
    T* out = rows_out + ((first + lane.next_to) * words + lane.at) * 8;
    for (int j0 = 0, t0 = 0; t0 < walk.each; j0 += U, t0 += U * walk.beside) {
        int64_t at[U];
        bool write[U];
        T* to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int tok = t0 + u * walk.beside + lane.next_to;
            at[u] = __shfl_sync(0xffffffffu, mine, tok & 31);
            write[u] = lane.real && tok < walk.each && at[u] != NO_SEQUENCE;
            if (at[u] >= 0) at[u] += (int64_t)lane.head << c.page_shift;
            to[u] = out + (t0 + u * walk.beside) * words * 8;
        }
        for (int k = 0; k < walk.rounds; k++) {
            if (U == 1 && walk.share > 1 && (j0 * walk.rounds + k) % walk.share != warp % walk.share) continue;
            const bool inside = lane.at + 32 * k < words;
            uint32_t codes[U], sm[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                codes[u] = 0; sm[u] = 0;                            // a token without a page of the pool reads as zeros
                if (inside && write[u] && at[u] >= 0) {
                    const int64_t row = at[u] + k * round_rows;
                    codes[u] = codes_at[row * (D / 8)];
                    sm[u] = params_at[row * (D / G)];
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (!inside || !write[u]) continue;
                const __half2 h = *reinterpret_cast<const __half2*>(&sm[u]);
                const float sc = __low2float(h), m = __high2float(h);
                // two codes at a time as f16: under the exponent of 1024 a nibble is 1024 + c, or 1024 + 16 c where it lies four bits up
                const auto half2_of = [](uint32_t v) { return *reinterpret_cast<const __half2*>(&v); };
                float f[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t w = e < 2 ? codes[u] : codes[u] >> 8;
                    const __half2 c2 = e & 1 ? __hfma2(half2_of((w & 0x00F000F0u) | 0x64006400u), half2_of(0x2C002C00u), half2_of(0xD400D400u))
                                             : __hsub2(half2_of((w & 0x000F000Fu) | 0x64006400u), half2_of(0x64006400u));
                    f[e] = fmaf(__low2float(c2), sc, m);
                    f[e + 4] = fmaf(__high2float(c2), sc, m);
                }
                constexpr int N = Vec16<T>::N;
#pragma unroll
                for (int i = 0; i < 8 / N; i++) {
                    Vec16<T> v;
#pragma unroll
                    for (int e = 0; e < N; e++) v.v[e] = Elem<T>::from_f32(f[i * N + e]);
                    *reinterpret_cast<uint4*>(to[u] + k * 256 + i * N) = *reinterpret_cast<const uint4*>(&v);
                }
            }
        }
    }
}
template <typename T, int D, int G, int U>
__global__ void __launch_bounds__(256) kv4_read_kernel(Pool c, Batch s, T* k_out, T* v_out, Walk walk, int32_t* status) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.y == 0) read_rows<T, D, G, U, true>(c, s, k_out, walk, status);
    else read_rows<T, D, G, U, false>(c, s, v_out, walk, status);
}

}  // namespace kv4
}  // namespace oxq

using namespace oxq;
using namespace oxq::kv4;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int32_t oxq_kv4_check(oxq_handle* h, const oxq_kv4_cache* c, const oxq_kv4_batch* s, Pool* pool, Batch* b) {
    if (!c || !s) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4: null cache or batch descriptor");
    if (c->dim != 64 && c->dim != 128) OXQ_FAIL(h, OXQ_ERR_UNSUPPORTED_OPERATION, "kv4: head dimension must be 64 or 128, got %d", c->dim);
    if ((c->group != 64 && c->group != 128) || c->group > c->dim)
        OXQ_FAIL(h, OXQ_ERR_GROUP_SIZE_MISMATCH, "kv4: group must be 64 or 128 and divide the head dimension %d, got %d", c->dim, c->group);
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4: page size must be a power of two from 16 to 4096, got %d", c->page_size);
    if (c->pages <= 0 || c->heads <= 0 || c->pages > INT32_MAX || c->heads > 65535)
        OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4: a pool of %lld pages and %d heads", (long long)c->pages, c->heads);
    if (!c->k_codes || !c->k_params || !c->v_codes || !c->v_params || !aligned16(c->k_codes) || !aligned16(c->k_params) || !aligned16(c->v_codes) || !aligned16(c->v_params))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4: null pool pointer, or one that is not 16-byte aligned");
    if (s->seqs < 0 || s->tokens < 0 || s->table_width < 0 || s->seqs > (1 << 24) || s->table_width > (1 << 27) || s->tokens > INT32_MAX)
        OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4: %lld sequences, %lld tokens, a table of %lld columns", (long long)s->seqs, (long long)s->tokens, (long long)s->table_width);
    if (s->table_width * c->page_size > (1 << 30))
        OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4: a table row covers %lld tokens", (long long)(s->table_width * c->page_size));
    if (s->seqs > 0 && s->tokens > 0 && ((!s->block_table && s->table_width > 0) || !s->seq_lens || !s->cu_tokens))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4: null block table, lengths or token offsets");
    int shift = 0;
    while ((1 << shift) < c->page_size) shift++;
    pool->kc = (uint8_t*)c->k_codes; pool->kp = (uint32_t*)c->k_params;
    pool->vc = (uint8_t*)c->v_codes; pool->vp = (uint32_t*)c->v_params;
    pool->pages = c->pages; pool->page_shift = shift; pool->heads = c->heads;
    b->table = s->block_table; b->width = s->table_width; b->lens = s->seq_lens; b->cu = s->cu_tokens; b->seqs = (int)s->seqs; b->tokens = s->tokens;
    return OXQ_OK;
}

// Tokens per warp: what leaves about `warps` warps on every SM for keys and for values, at least a word for every lane, at most
// eight (a read of 131k tokens: 125 us; with 32 a warp 150 us, for the last wave of CTAs is then long); a multiple of the tokens
// whose loads are in flight at once.  Where even a token a warp leaves SMs without work -- a decode step -- up to eight warps
// share the token's words.  Reading streams: 16 warps, four tokens at once.  Appending computes: 32 warps and two (8192 tokens
// of 8 heads: 18.1 us; 16 and four 22.8, 64 and one 23.7).
static Walk walk_of(const oxq_handle* h, const Pool& c, const Batch& s, int dim, int warps, int at_once, dim3* grid) {
    Walk w;
    const int words = c.heads * (dim / 8), least = (32 + words - 1) / words;
    const int64_t each = s.tokens / ((int64_t)h->sm_count * warps);
    w.each = (int)(each < least ? least : each > 8 && least <= 8 ? 8 : each > 32 ? 32 : each);
    w.beside = words < 32 ? 32 / words : 1;
    w.rounds = (words + 31) / 32;
    const int share = s.tokens < 8ll * h->sm_count ? (w.each + w.beside - 1) / w.beside * w.rounds : 1;
    w.share = share > 8 ? 8 : share;
    if (w.share == 1) {
        const int whole = at_once * w.beside;
        w.each = w.each + whole - 1 < 32 ? (w.each + whole - 1) / whole * whole : 32;
    }
    *grid = dim3((unsigned)(((s.tokens + w.each - 1) / w.each * w.share + 7) / 8), 2);
    return w;
}

template <typename T, int D, int G>
static cudaError_t launch_append(oxq_handle* h, const Pool& c, const Batch& s, const Rows<T>& in) {
    dim3 grid;
    const Walk w = walk_of(h, c, s, D, 32, 2, &grid);
    if (w.share > 1) return oxq_launch(kv4_append_kernel<T, D, G, 1>, grid, 256, 0, h->stream, c, s, in, w, h->dev_status);
    return oxq_launch(kv4_append_kernel<T, D, G, 2>, grid, 256, 0, h->stream, c, s, in, w, h->dev_status);
}

template <typename T, int D, int G>
static cudaError_t launch_read(oxq_handle* h, const Pool& c, const Batch& s, void* k, void* v) {
    dim3 grid;
    const Walk w = walk_of(h, c, s, D, 16, 4, &grid);
    if (w.share > 1) return oxq_launch(kv4_read_kernel<T, D, G, 1>, grid, 256, 0, h->stream, c, s, (T*)k, (T*)v, w, h->dev_status);
    return oxq_launch(kv4_read_kernel<T, D, G, 4>, grid, 256, 0, h->stream, c, s, (T*)k, (T*)v, w, h->dev_status);
}

template <typename T>
static int32_t append_t(oxq_handle* h, const oxq_kv4_cache* cc, const Pool& c, const Batch& s, const void* k, const void* v, int64_t kt, int64_t kh, int64_t vt, int64_t vh) {
    Rows<T> in;
    in.p[0] = (const T*)k; in.p[1] = (const T*)v;
    in.token_stride[0] = kt; in.token_stride[1] = vt; in.head_stride[0] = kh; in.head_stride[1] = vh;
    const int64_t all = kt | kh | vt | vh;
    in.vec = aligned16(k) && aligned16(v) && (all * (int64_t)sizeof(T)) % 16 == 0;
    if (cc->dim == 64) OXQ_CUDA(h, (launch_append<T, 64, 64>(h, c, s, in)));
    else if (cc->group == 64) OXQ_CUDA(h, (launch_append<T, 128, 64>(h, c, s, in)));
    else OXQ_CUDA(h, (launch_append<T, 128, 128>(h, c, s, in)));
    return OXQ_OK;
}

template <typename T>
static int32_t read_t(oxq_handle* h, const oxq_kv4_cache* cc, const Pool& c, const Batch& s, void* k, void* v) {
    if (cc->dim == 64) OXQ_CUDA(h, (launch_read<T, 64, 64>(h, c, s, k, v)));
    else if (cc->group == 64) OXQ_CUDA(h, (launch_read<T, 128, 64>(h, c, s, k, v)));
    else OXQ_CUDA(h, (launch_read<T, 128, 128>(h, c, s, k, v)));
    return OXQ_OK;
}

extern "C" {

int32_t oxq_kv4_append(oxq_handle* h, const oxq_kv4_cache* cache, const oxq_kv4_batch* batch, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                       const void* v, int64_t v_token_stride, int64_t v_head_stride, int dtype) {
    OXQ_CHECK_HANDLE(h);
    Pool c; Batch s;
    if (int32_t rc = oxq_kv4_check(h, cache, batch, &c, &s)) return rc;
    if (dtype != OXQ_F32 && dtype != OXQ_BF16 && dtype != OXQ_F16) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (s.tokens == 0 || s.seqs == 0) return OXQ_OK;
    if (!k || !v) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 append: null keys or values");
    if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 append: negative stride");
    if (s.tokens * c.heads > INT32_MAX) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 append: %lld tokens of %d heads", (long long)s.tokens, c.heads);
    if (int32_t rc = oxq_require_sm100(h)) return rc;
    OxqDeviceGuard guard(h->device);
    switch (dtype) {
        case OXQ_F32: return append_t<float>(h, cache, c, s, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride);
        case OXQ_BF16: return append_t<__nv_bfloat16>(h, cache, c, s, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride);
        default: return append_t<__half>(h, cache, c, s, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride);
    }
}

int32_t oxq_kv4_read(oxq_handle* h, const oxq_kv4_cache* cache, const oxq_kv4_batch* batch, void* k_out, void* v_out, int dtype) {
    OXQ_CHECK_HANDLE(h);
    Pool c; Batch s;
    if (int32_t rc = oxq_kv4_check(h, cache, batch, &c, &s)) return rc;
    if (dtype != OXQ_F32 && dtype != OXQ_BF16 && dtype != OXQ_F16) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (s.tokens == 0 || s.seqs == 0) return OXQ_OK;
    if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 read: null output, or one that is not 16-byte aligned");
    if (s.tokens * c.heads > INT32_MAX) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "kv4 read: %lld tokens of %d heads", (long long)s.tokens, c.heads);
    const uint64_t bytes = (uint64_t)s.tokens * c.heads * cache->dim * (dtype == OXQ_F32 ? 4 : 2), ka = (uintptr_t)k_out, va = (uintptr_t)v_out;
    if ((ka < va ? va - ka : ka - va) < bytes) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "kv4 read: the outputs overlap");
    if (int32_t rc = oxq_require_sm100(h)) return rc;
    OxqDeviceGuard guard(h->device);
    switch (dtype) {
        case OXQ_F32: return read_t<float>(h, cache, c, s, k_out, v_out);
        case OXQ_BF16: return read_t<__nv_bfloat16>(h, cache, c, s, k_out, v_out);
        default: return read_t<__half>(h, cache, c, s, k_out, v_out);
    }
}

}  // extern "C"
