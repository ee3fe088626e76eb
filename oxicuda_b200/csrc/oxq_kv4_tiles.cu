// Attention over the paged 4-bit cache for many query rows per kv head (layout: oxq_kv4.cuh): prompts and chunks of them.
//
// The mathematics is the usual one: S = Q K^T, a running reference M per row (moved only when a score exceeds it by 2^8, as
// all exponents are taken in base 2), P = 2^(S - M), O += P V, l += row sums of P, o = O / l at the end.  Keys and values
// become f16 numbers rounded once from c s + m (a number below 2^-13 is a multiple of 2^-24 and not rounded at all; one that
// the rounding of s has lifted above 65504, by 64 at most, counts as 65504), P is f16, everything else f32.  f16 rather than bf16 operands, for either type of the queries: their rounding is eight times
// finer.  A query row enters scaled by a power of two so that its largest element lies in [2^11, 2^12): exact, but for
// elements below 2^-25 of it, which are off by at most 2^-36 of it; the row's factor goes into the softmax.  l is summed from
// the unrounded p.
//
// The shape: a CTA takes two blocks of 128 query rows (tokens and the query heads of one kv head, packed) and walks the keys
// in tiles of 128.  tcgen05.mma: S from shared memory (Q and the tile's keys), O from P in tensor memory, written over the
// scores, and the tile's values.  Roles: two warpgroups of softmax (one row a thread), two that turn codes into f16 tiles
// (two stages each of keys and values), one warp that issues the products; registers go from the others to the softmax.
// While one block's scores are in softmax the tensor core works on the other block's.  Inside every eight elements of a head
// the order is 0 4 1 5 2 6 3 7, which is the order in which a word's nibbles come out in pairs; it is undone where O is stored.
//
// What bounds it: a block's softmax and its products take turns (of 4300 cycles a tile and block: 1900 waiting for products,
// 1650 exponentials, 450 fetching scores, 400 finding their maximum, before P was handed over in halves) and the two blocks
// fill each other's gaps in part only; a prompt of 8192 tokens with 32 query heads on 8 takes 558 us = 985 TFLOP/s, 0.58 of
// cuBLAS's rate (0.52 in a long run under the power cap), the products alone 401.  A CTA's set-up is 10 us.  At 96 registers a
// thread before the split the compiler spills 70 to 86 bytes.
#include "oxq_kv4_attn.cuh"
#include "oxq_tc.cuh"

namespace oxq {
namespace kv4 {

using namespace tc;

constexpr int BLOCK = 128;                      // rows of a block, and keys of a tile
constexpr int ATOM = BLOCK * 128;               // bytes of 128 rows of 128 bytes (64 f16), the swizzle's unit

template <int D> struct TileSmem {
    static constexpr int OPERAND = ATOM * (D / 64);
    static constexpr int Q = 0, K = Q + 2 * OPERAND, V = K + 2 * OPERAND, BARS = V + 2 * OPERAND, VALID = BARS + 128, SLOT = VALID + 32, BYTES = SLOT + 16 + 1024;
};
enum { BAR_Q = 0, BAR_KFULL = 1, BAR_KEMPTY = 3, BAR_VFULL = 5, BAR_VEMPTY = 7, BAR_S = 9, BAR_P = 11, BAR_END = 13, BAR_P2 = 14 };      // P in halves of 64 keys

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// two f32 operations in one instruction, and the largest of three
__device__ __forceinline__ uint64_t two(float x, float y) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ void apart(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Eight codes of a word to f16 c s + m, one rounding each, in the order 0 4 1 5 2 6 3 7.  A nibble under the exponent of 1024
// is the number 1024 + c (or 1024 + 16 c where it is left four bits up), from which c is exact in one operation.  s is not
// negative and m finite, so that overflow has one side only; a NaN stays one.
__device__ __forceinline__ uint4 expand(uint32_t w, __half2 s, __half2 m) {
    const __half2 k1024 = as_half2(0x64006400u), k16 = as_half2(0x2C002C00u), k64 = as_half2(0xD400D400u);    // 1024, 1 / 16, -64
    const auto value = [&](__half2 c) { return as_u32(__hmin2_nan(__hfma2(c, s, m), as_half2(0x7BFF7BFFu))); };
    uint4 o;
    o.x = value(__hsub2(as_half2((w & 0x000F000Fu) | 0x64006400u), k1024));
    o.y = value(__hfma2(as_half2((w & 0x00F000F0u) | 0x64006400u), k16, k64));
    w >>= 8;
    o.z = value(__hsub2(as_half2((w & 0x000F000Fu) | 0x64006400u), k1024));
    o.w = value(__hfma2(as_half2((w & 0x00F000F0u) | 0x64006400u), k16, k64));
    return o;
}

// Threads: warpgroups 0, 1 softmax, 2, 3 producers, 4 (its first warp) products.  Registers a thread after the split: launched with
// 96 x 640 = 61440 in all, 2 x 128 x 168 + 2 x 128 x 56 + 128 x 32 = 61440.
constexpr int THREADS = 640, PRODUCERS = 256, MMA_WARP = 16;
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The CTA's item: sequence and pair of row blocks.  Items of a sequence come last rows first: they see the most keys.
struct TileItem { int b, pair; SeqInfo q; };
__device__ __forceinline__ int pairs_of(const AttnParams& p, int b) {
    const SeqInfo q = seq_info(p, b);
    const int64_t rows = (int64_t)q.n * p.per;
    return rows <= p.row_min ? 0 : (int)((rows + 2 * BLOCK - 1) / (2 * BLOCK));
}
// Whole warp; false: there is no such item.
__device__ __forceinline__ bool find_pair(const AttnParams& p, int want, TileItem& it) {
    const int lane = threadIdx.x & 31;
    int base = 0;
    for (int b0 = 0; b0 < p.s.seqs; b0 += 32) {
        const int n = b0 + lane < p.s.seqs ? pairs_of(p, b0 + lane) : 0;
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want >= base + x - n && want < base + x);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.b = b0 + src;
            it.pair = __shfl_sync(0xffffffffu, x, src) + base - 1 - want;
            it.q = seq_info(p, it.b);
            return true;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    return false;
}

// What the rows row0 .. of an item see together: positions [lo, hi), and this CTA's part of the tiles that hold them,
// [first, first + n).  Places outside [lo, hi) are not looked at: pages in front of a window may have been given back.
struct Walk { int first, n, lo, hi; };
__device__ __forceinline__ Walk walk_of(const AttnParams& p, const SeqInfo& q, int pair, int part) {
    const int row0 = pair * 2 * BLOCK;
    const int j0 = p.by_per.div(row0), j1 = p.by_per.div(min(row0 + 2 * BLOCK, q.n * p.per) - 1);
    const int hi = max(0, p.causal ? min(q.len, q.before + j1 + 1) : q.len);
    const int lo = min(hi, max(0, window_start(p, q.before + j0)));
    const int first = lo / BLOCK, all = (hi + BLOCK - 1) / BLOCK - first;
    const int a = (int)((int64_t)all * part / p.parts), e = (int)((int64_t)all * (part + 1) / p.parts);
    return {first + a, e - a, lo, hi};
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(THREADS, 1) kv4_attn_tiles_kernel(AttnParams p) {
    using L = TileSmem<D>;
    constexpr int NA = D / 64;
    extern __shared__ unsigned char smem_dyn[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();

    TileItem it;
    const int head = blockIdx.x % p.c.heads, part = blockIdx.y;
    if (!find_pair(p, blockIdx.x / p.c.heads, it)) { pdl_trigger(); return; }      // the grid is an upper bound
    const SeqInfo q = it.q;
    const Walk walk = walk_of(p, q, it.pair, part);
    const int n = walk.n;

    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* smem = smem_dyn + (base - smem_u32(smem_dyn));
    const auto bar = [&](int i) { return base + L::BARS + 8 * i; };
    // Each role asks for its first data, then meets the others: barriers and tensor memory are set up by the last one.
    uint32_t tmem = 0;
    const auto ready = [&]() {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        pdl_trigger();                          // only now: a kernel that starts early must not find tensor memory before this one
        tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::SLOT);
    };
    const auto fail = [&]() { *p.status = OXQ_ERR_DEVICE_TIMEOUT; };

    if (warp < 8) {
        // ------------------------------------------------------------------------------------ softmax: one row a thread
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;
        const int row = it.pair * 2 * BLOCK + t * BLOCK + r;
        const bool real = row < q.n * p.per;
        const int tok = p.by_per.div(row), qh = head * p.per + p.by_per.mod(row);
        const int pos = q.before + tok;
        const int vhi = !real ? 0 : p.causal ? min(q.len, pos + 1) : q.len, vlo = window_start(p, pos);
        float a;                                // scores to units of log2
        {
            const T* src = (const T*)p.q + (int64_t)(q.start + tok) * p.q_ts + (int64_t)qh * p.q_hs;
            uint32_t raw[D / 2];
            if (real && p.q_vec) {
#pragma unroll
                for (int i = 0; i < D / 8; i++) {
                    const uint4 v = reinterpret_cast<const uint4*>(src)[i];
                    raw[4 * i] = v.x; raw[4 * i + 1] = v.y; raw[4 * i + 2] = v.z; raw[4 * i + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < D / 2; i++)
                    raw[i] = real ? (uint32_t)reinterpret_cast<const unsigned short*>(src)[2 * i] |
                                        ((uint32_t)reinterpret_cast<const unsigned short*>(src)[2 * i + 1] << 16) : 0u;
            }
            ready();
            more_registers<168>();
            const auto value = [&](int e) {
                const unsigned short h = (unsigned short)(raw[e >> 1] >> (16 * (e & 1)));
                if constexpr (Elem<T>::kDtype == OXQ_BF16) return __uint_as_float((uint32_t)h << 16);
                else return __half2float(__ushort_as_half(h));
            };
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < D; e++) top = fmaxf(top, fabsf(value(e)));
            const int ex = max((int)(__float_as_uint(top) >> 23) - 127, -116);                      // 2^(11 - ex) has to be a number
            // a negative scale goes into the sign of the queries, a zero one into their magnitude, so that a > 0 below
            const float up = p.scale_log2 == 0.0f ? 0.0f : copysignf(pow2_of(max(11 - ex, -126)), p.scale_log2);
            a = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2) * pow2_of(ex - 11);
            unsigned char* dst = smem + L::Q + t * L::OPERAND + r * 128;
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                uint4 o;
                o.x = pack2(value(8 * i) * up, value(8 * i + 4) * up); o.y = pack2(value(8 * i + 1) * up, value(8 * i + 5) * up);
                o.z = pack2(value(8 * i + 2) * up, value(8 * i + 6) * up); o.w = pack2(value(8 * i + 3) * up, value(8 * i + 7) * up);
                *reinterpret_cast<uint4*>(dst + (i >> 3) * ATOM + (((i & 7) ^ (r & 7)) << 4)) = o;
            }
            fence_proxy_async();
            mbar_arrive(bar(BAR_Q));
        }
        // keys that every row of this warp sees need no mask
        const int all_hi = __reduce_min_sync(0xffffffffu, real ? vhi : INT32_MAX), all_lo = __reduce_max_sync(0xffffffffu, real ? vlo : 0);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + t * BLOCK + lanes, o_col = tmem + 256 + t * BLOCK + lanes;
        float M = -1e30f;
        uint64_t l2[2] = {0, 0};                // the sum in four parts
        const uint64_t a2 = two(a, a);
        bool ok = true;
        for (int i = 0; i < n; i++) {
            ok = mbar_wait_warp(bar(BAR_S + t), i & 1);
            if (!ok) { if (lane == 0) fail(); break; }
            tc_fence_after();
            const int t0 = (walk.first + i) * BLOCK;
            const uint32_t* valid = reinterpret_cast<const uint32_t*>(smem + L::VALID + (i & 3) * 8);
            const uint32_t v0 = valid[0], v1 = valid[1];
            const bool masked = t0 < all_lo || t0 + BLOCK > all_hi || (v0 & v1) != 0x01010101u;
            uint32_t s[4][32];                  // loaded below, in two halves
            const auto at = [&](int e) { return __uint_as_float(s[e >> 5][e & 31]); };
            float top[8];
            // the second half is on its way while the first one's largest is found
            tmem_ld_32x32b_x32(s_col, s[0]);
            tmem_ld_32x32b_x32(s_col + 32, s[1]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (h == 0) {
                    tmem_ld_32x32b_x32(s_col + 64, s[2]);
                    tmem_ld_32x32b_x32(s_col + 96, s[3]);
                } else {
                    tmem_ld_wait();
                }
                if (masked) {
#pragma unroll
                    for (int e = 64 * h; e < 64 * h + 64; e++) {
                        const int key = t0 + e;
                        const bool have = ((h ? v1 : v0) >> (8 * ((e >> 4) & 3))) & 1u;
                        if (key < vlo || key >= vhi || !have) s[e >> 5][e & 31] = 0xFF800000u;
                    }
                }
#pragma unroll
                for (int f = 0; f < 8; f++) {
                    float x = h ? max3(top[f], at(64 + f), at(72 + f)) : fmaxf(at(f), at(8 + f));
#pragma unroll
                    for (int e = 16; e < 64; e += 16) x = max3(x, at(64 * h + e + f), at(64 * h + e + 8 + f));
                    top[f] = x;
                }
            }
            const float most = fmaxf(max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]), top[6]), top[7]) * a;
            const bool over = most > M + 8.0f;
            if (__any_sync(0xffffffffu, over)) {
                // the reference moves: what was summed so far shrinks with it -- l, and O (the last product into it is
                // complete: it was issued before these scores)
                const float to = over ? most : M, f = exp2_approx(M - to);
                M = to;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x, y;
                    apart(l2[h], x, y);
                    l2[h] = two(x * f, y * f);
                }
                if (i > 0) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_col + c0, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_32x32b_x16(o_col + c0, o);
                    }
                }
            }
            const uint64_t m2 = two(-M, -M);
#pragma unroll
            for (int ch = 0; ch < 4; ch++) {
                uint32_t o[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float x, y;
                    apart(fma2(two(at(32 * ch + 2 * e), at(32 * ch + 2 * e + 1)), a2, m2), x, y);
                    x = exp2_approx(x);
                    y = exp2_approx(y);
                    l2[e & 1] = add2(l2[e & 1], two(x, y));
                    o[e] = pack2(x, y);
                }
                tmem_st_32x32b_x16(s_col + 16 * ch, o);
                if (ch & 1) {                       // the product with the first half need not wait for the second
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(bar((ch == 1 ? BAR_P : BAR_P2) + t));
                }
            }
        }
        if (ok && n > 0) {
            ok = mbar_wait_warp(bar(BAR_S + t), n & 1);         // the last product into O
            if (!ok && lane == 0) fail();
            tc_fence_after();
        }
        float l, l_odd;
        apart(add2(l2[0], l2[1]), l, l_odd);
        l += l_odd;
        if (ok) {
            float* slot = p.parts > 1 ? p.ws + ((int64_t)blockIdx.x * p.parts + part) * (2 * BLOCK * (D + 2)) : nullptr;
            const float inv = l > 0.0f ? 1.0f / l : l != l ? l : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld_32x32b_x32(o_col + c0, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0;
                }
                constexpr int kAt[8] = {0, 2, 4, 6, 1, 3, 5, 7};                                          // column of element e
                if (real) {
                    if (slot) {
                        float* dst = slot + (t * BLOCK + r) * D + c0;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(dst + e) = make_float4(
                                __uint_as_float(o[(e & ~7) + kAt[e & 7]]), __uint_as_float(o[(e & ~7) + kAt[(e & 7) + 1]]),
                                __uint_as_float(o[(e & ~7) + kAt[(e & 7) + 2]]), __uint_as_float(o[(e & ~7) + kAt[(e & 7) + 3]]));
                        if (c0 == 0) { slot[2 * BLOCK * D + t * BLOCK + r] = M; slot[2 * BLOCK * (D + 1) + t * BLOCK + r] = l; }
                    } else {
                        T* dst = (T*)p.out + (int64_t)(q.start + tok) * p.o_ts + (int64_t)qh * p.o_hs + c0;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            struct alignas(16) Eight { T v[8]; } w;
#pragma unroll
                            for (int k = 0; k < 8; k++) w.v[k] = Elem<T>::from_f32(l > 0.0f || l != l ? __uint_as_float(o[e + kAt[k]]) * inv : 0.0f);
                            const uint4 u = *reinterpret_cast<const uint4*>(&w);
                            if (p.out_vec) *reinterpret_cast<uint4*>(dst + e) = u;
                            else {
                                uint32_t* d4 = reinterpret_cast<uint32_t*>(dst + e);
                                d4[0] = u.x; d4[1] = u.y; d4[2] = u.z; d4[3] = u.w;
                            }
                        }
                        if (c0 == 0 && p.lse)
                            p.lse[(int64_t)(q.start + tok) * p.q_heads + qh] = l > 0.0f || l != l ? (M + log2f(l)) * 0.693147180559945309417f : -INFINITY;
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------------------------------------------ codes to f16 tiles
        constexpr int Q16 = D / 32;                                 // 16-byte pieces of a row
        constexpr int ROUNDS = BLOCK * Q16 / PRODUCERS, PER_ROUND = PRODUCERS / Q16;
        const int pt = tid - 256, piece = pt % Q16, tok0 = pt / Q16;
        const int32_t* table = p.s.table + (int64_t)it.b * p.s.width;
        // One tile's codes wait in registers, keys and values apart: the next tile's keys are requested when this one's have
        // been turned into f16, and are there when its values have; the table's entries are fetched a tile before that.
        uint4 kraw[ROUNDS], vraw[ROUNDS];
        uint32_t kpar[ROUNDS][NG], vpar[ROUNDS][NG];
        int page[ROUNDS];
        bool gone[ROUNDS];                                          // a key without a page of the pool; those that no row sees are masked by their positions
        const auto wanted = [&](int i, int key) { return i < n && key >= walk.lo && key < walk.hi; };
        const auto get_pages = [&](int i) {
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) {
                const int key = (walk.first + i) * BLOCK + tok0 + u * PER_ROUND;
                page[u] = wanted(i, key) ? table[key >> p.c.page_shift] : -1;
            }
        };
        const auto load = [&](int i, const uint8_t* codes, const uint32_t* params, uint4 (&raw)[ROUNDS], uint32_t (&par)[ROUNDS][NG], bool keys) {
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) {
                const int key = (walk.first + i) * BLOCK + tok0 + u * PER_ROUND;
                raw[u] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int g = 0; g < NG; g++) par[u][g] = 0;
                const bool inside = wanted(i, key), good = inside && page[u] >= 0 && page[u] < p.c.pages;
                if (keys) {
                    gone[u] = inside && !good;
                    if (gone[u] && piece == 0) *p.status = OXQ_ERR_INVALID_ARGUMENT;
                }
                if (good) {
                    const int64_t row = (((int64_t)page[u] * p.c.heads + head) << p.c.page_shift) + (key & ((1 << p.c.page_shift) - 1));
                    raw[u] = reinterpret_cast<const uint4*>(codes + row * (D / 2))[piece];
                    if constexpr (NG == 2) {
                        const uint2 v = *reinterpret_cast<const uint2*>(params + row * 2);
                        par[u][0] = v.x; par[u][1] = v.y;
                    } else par[u][0] = params[row];
                }
            }
        };
        const auto put = [&](uint32_t tile, const uint4 (&raw)[ROUNDS], const uint32_t (&par)[ROUNDS][NG], bool keys) {
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) {
                const int tok = tok0 + u * PER_ROUND;
                const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                __half2 s[NG], m[NG];
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    s[g] = __low2half2(as_half2(par[u][g])); m[g] = __high2half2(as_half2(par[u][g]));
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    constexpr int KI = D / 32, VI = D / 64;
                    // place 4 * piece + i of the row -> its word; with 16 bytes a piece, i alone decides which group it is in
                    const int c = keys ? (4 * piece + i) / KI : (4 * piece + i) / VI, b = keys ? (4 * piece + i) % KI : (4 * piece + i) % VI;
                    const int word = keys ? 4 * b + c : 8 * b + c;
                    const int g = NG == 1 ? 0 : keys ? (i % KI) / (KI / NG) : i % VI;
                    const uint32_t at = tile + (word >> 3) * ATOM + tok * 128 + (((word & 7) ^ (tok & 7)) << 4);
                    const uint4 o = expand(w[i], s[g], m[g]);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w) : "memory");
                }
            }
        };
        get_pages(0);
        load(0, p.c.kc, p.c.kp, kraw, kpar, true);
        load(0, p.c.vc, p.c.vp, vraw, vpar, false);
        get_pages(1);
        ready();
        fewer_registers<56>();
        for (int i = 0; i < n; i++) {
            const int st = i & 1;
            const uint32_t ph = (i >> 1) & 1;
            if (!mbar_wait_warp(bar(BAR_KEMPTY + st), ph ^ 1)) { if (lane == 0) fail(); break; }
            put(base + L::K + st * L::OPERAND, kraw, kpar, true);
#pragma unroll
            for (int u = 0; u < ROUNDS; u++) {
                const int tok = tok0 + u * PER_ROUND;
                if (piece == 0 && (tok & 15) == 0) smem[L::VALID + (i & 3) * 8 + (tok >> 4)] = gone[u] ? 0 : 1;
            }
            fence_proxy_async();
            mbar_arrive(bar(BAR_KFULL + st));
            load(i + 1, p.c.kc, p.c.kp, kraw, kpar, true);
            if (!mbar_wait_warp(bar(BAR_VEMPTY + st), ph ^ 1)) { if (lane == 0) fail(); break; }
            put(base + L::V + st * L::OPERAND, vraw, vpar, false);
            fence_proxy_async();
            mbar_arrive(bar(BAR_VFULL + st));
            load(i + 1, p.c.vc, p.c.vp, vraw, vpar, false);
            get_pages(i + 2);
        }
    } else {
        if (warp == MMA_WARP) {
            if (lane == 0) {
                mbar_init(bar(BAR_Q), 256);
                mbar_init(bar(BAR_END), 1);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mbar_init(bar(BAR_KFULL + i), PRODUCERS); mbar_init(bar(BAR_KEMPTY + i), 1);
                    mbar_init(bar(BAR_VFULL + i), PRODUCERS); mbar_init(bar(BAR_VEMPTY + i), 1);
                    mbar_init(bar(BAR_S + i), 1); mbar_init(bar(BAR_P + i), 128); mbar_init(bar(BAR_P2 + i), 128);
                }
                fence_barrier_init();
            }
            __syncwarp();
            tmem_alloc(base + L::SLOT, 512);
            tmem_relinquish();
        }
        ready();
        fewer_registers<32>();
        if (warp == MMA_WARP) {
        // ------------------------------------------------------------------------------------ products (whole warp, one lane issues)
        constexpr uint32_t id_s = idesc_dense(1, 0, 0, BLOCK, BLOCK), id_o = idesc_dense(1, 0, 0, BLOCK, D) | idesc_majors(0, 1);
        const auto scores = [&](int t, int st) {
            const uint32_t qa = base + L::Q + t * L::OPERAND, ka = base + L::K + st * L::OPERAND;
#pragma unroll
            for (int at = 0; at < NA; at++) {
                const uint64_t ad = smem_desc_sw128(qa + at * ATOM), bd = smem_desc_sw128(ka + at * ATOM);
#pragma unroll
                for (int kk = 0; kk < 4; kk++) mma_f16(tmem + t * BLOCK, ad + kk * 2, bd + kk * 2, id_s, (at | kk) != 0);
            }
        };
        const auto sums = [&](int t, int st, bool more, int half) {
            const uint64_t bd = smem_desc_mn_sw128(base + L::V + st * L::OPERAND, ATOM);
#pragma unroll
            for (int kk = half * (BLOCK / 32); kk < (half + 1) * (BLOCK / 32); kk++) mma_f16_ts(tmem + 256 + t * BLOCK, tmem + t * BLOCK + kk * 8, bd + kk * 128, id_o, more || kk != 0);
        };
        bool ok = true;
        if (n > 0) {
            ok = mbar_wait_warp(bar(BAR_Q), 0) && mbar_wait_warp(bar(BAR_KFULL), 0);
            if (!ok && lane == 0) fail();
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    scores(0, 0); tc_commit(bar(BAR_S));
                    scores(1, 0); tc_commit(bar(BAR_S + 1));
                    tc_commit(bar(BAR_KEMPTY));
                }
                __syncwarp();
            }
        }
        for (int i = 0; i < n && ok; i++) {
            const int st = i & 1, nx = (i + 1) & 1;
            ok = mbar_wait_warp(bar(BAR_VFULL + st), (i >> 1) & 1);
            for (int t = 0; t < 2 && ok; t++) {
                ok = mbar_wait_warp(bar(BAR_P + t), i & 1);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) sums(t, st, i > 0, 0);
                __syncwarp();
                if (t == 0 && i + 1 < n) ok = mbar_wait_warp(bar(BAR_KFULL + nx), ((i + 1) >> 1) & 1);
                ok = ok && mbar_wait_warp(bar(BAR_P2 + t), i & 1);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    sums(t, st, true, 1);
                    if (i + 1 < n) scores(t, nx);
                    tc_commit(bar(BAR_S + t));
                    if (t == 1) {
                        tc_commit(bar(BAR_VEMPTY + st));
                        if (i + 1 < n) tc_commit(bar(BAR_KEMPTY + nx));
                    }
                }
                __syncwarp();
            }
            if (!ok) { if (lane == 0) fail(); break; }
        }
        if (!ok) {
            // Something did not arrive.  What was issued still has to end, with a limit, before tensor memory is given back.
            if (elect_one()) tc_commit(bar(BAR_END));
            __syncwarp();
            mbar_wait_warp(bar(BAR_END), 0);
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of an item: block (item and head, eight or sixteen rows), D / 4 threads a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_tiles_join_kernel(AttnParams p) {
    pdl_trigger();
    pdl_wait();
    TileItem it;
    const int head = blockIdx.x % p.c.heads;
    if (!find_pair(p, blockIdx.x / p.c.heads, it)) return;
    const int r = blockIdx.y * (256 / (D / 4)) + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int row = it.pair * 2 * BLOCK + r;
    if (row >= it.q.n * p.per) return;
    const float* slot = p.ws + (int64_t)blockIdx.x * p.parts * (2 * BLOCK * (D + 2));
    float top = -1e30f, sum = 0.0f;
    for (int k = 0; k < p.parts; k++) top = fmaxf(top, slot[(int64_t)k * (2 * BLOCK * (D + 2)) + 2 * BLOCK * D + r]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int k = 0; k < p.parts; k++) {
        const float* s = slot + (int64_t)k * (2 * BLOCK * (D + 2));
        const float f = exp2_approx(s[2 * BLOCK * D + r] - top);
        const float4 v = *reinterpret_cast<const float4*>(s + r * D + d);
        sum = fmaf(s[2 * BLOCK * (D + 1) + r], f, sum);
        o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    store_row<T>(p, it.q, head, row, d, make_float2(o.x, o.y), top, sum);
    store_row<T>(p, it.q, head, row, d + 2, make_float2(o.z, o.w), top, sum);
}

}  // namespace kv4
}  // namespace oxq

using namespace oxq;
using namespace oxq::kv4;

template <typename T, int D, int NG>
static int32_t launch_tiles(oxq_handle* h, const AttnParams& p, int64_t items) {
    auto kernel = kv4_attn_tiles_kernel<T, D, NG>;
    constexpr int bytes = TileSmem<D>::BYTES < 120 * 1024 ? 120 * 1024 : TileSmem<D>::BYTES;      // one CTA per SM: each takes all of tensor memory
    static OxqPerDevice ready;
    if (!ready.get(h->device)) {
        OXQ_CUDA(h, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        ready.set(h->device, 1);
    }
    const dim3 grid((unsigned)(items * p.c.heads), (unsigned)p.parts);
    OXQ_CUDA(h, oxq_launch(kernel, grid, THREADS, bytes, h->stream, p));
    if (p.parts > 1) OXQ_CUDA(h, oxq_launch(kv4_tiles_join_kernel<T, D>, dim3(grid.x, 2 * BLOCK / (256 / (D / 4))), 256, 0, h->stream, p));
    return OXQ_OK;
}

int64_t oxq_kv4_tiles_slot_bytes(int dim) { return (int64_t)2 * BLOCK * (dim + 2) * (int64_t)sizeof(float); }

int32_t oxq_kv4_tiles_launch(oxq_handle* h, const oxq_kv4_cache* cc, const AttnParams& p, int dtype, int64_t items) {
    if (dtype == OXQ_BF16) {
        if (cc->dim == 64) return launch_tiles<__nv_bfloat16, 64, 1>(h, p, items);
        if (cc->group == 64) return launch_tiles<__nv_bfloat16, 128, 2>(h, p, items);
        return launch_tiles<__nv_bfloat16, 128, 1>(h, p, items);
    }
    if (cc->dim == 64) return launch_tiles<__half, 64, 1>(h, p, items);
    if (cc->group == 64) return launch_tiles<__half, 128, 2>(h, p, items);
    return launch_tiles<__half, 128, 1>(h, p, items);
}
