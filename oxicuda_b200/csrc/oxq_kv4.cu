// Writing tokens into the paged 4-bit key / value cache, and reading them back (layout: oxq_kv4.cuh).
//
// Quantizer, per group of G elements of one head of one token:
//   s = f16((max - min) / 15), m = f16(min), c = clamp(rint((x - m) / s), 0, 15), and c = 0 where s is 0.
// The codes are computed from the rounded s and m, the numbers the reader uses, so rounding them costs no accuracy in the
// codes.  s and m stay f16 (4 bytes a group): the offset is a float, not a zero-point in code units, because a group whose
// values all lie on one side of zero must keep its four bits for its own range.
#include "oxq_kv4.cuh"

namespace oxq {
namespace kv4 {

template <typename T>
struct Rows {
    const T* p[2];                      // keys, values
    int64_t token_stride[2], head_stride[2];
    int vec;                            // 16-byte loads are aligned
};

// Eight elements as f32, NaN as 0, held to the range of f16 (s and m are f16).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int vec, float (&f)[8]) {
    if (vec) {
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; i++) {
            const Vec16<T> v = ld16_stream(p + i * N);
#pragma unroll
            for (int e = 0; e < N; e++) f[i * N + e] = Elem<T>::to_f32(v.v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = Elem<T>::to_f32(p[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = f[e] != f[e] ? 0.0f : fminf(fmaxf(f[e], -65504.0f), 65504.0f);
}

// A thread takes one word (eight elements) of U rows; D / 8 neighbouring lanes make a row.
template <typename T, int D, int G, int U>
__global__ void __launch_bounds__(256) kv4_append_kernel(Pool c, Batch s, Rows<T> in, int32_t* status) {
    pdl_trigger();
    pdl_wait();
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    const int lane = threadIdx.x & 31, word = lane % LANES;
    const int which = blockIdx.y;
    const int64_t rows = s.tokens * c.heads;
    const int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (PER_WARP * U);
    if (first >= rows) return;                                      // whole warps
    int b = sequence_of(s.cu, s.seqs, first / c.heads);
    float f[U][8];
    int64_t at[U];                                                  // row in the pool, -1: none
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = first + u * PER_WARP + lane / LANES;
        const int64_t t = row / c.heads;
        const int head = (int)(row - t * c.heads);
        at[u] = -1;
#pragma unroll
        for (int e = 0; e < 8; e++) f[u][e] = 0.0f;
        if (row < rows) {
            while (b < s.seqs && __ldg(s.cu + b + 1) <= t) b++;
            if (b < s.seqs && t >= __ldg(s.cu + b)) {
                at[u] = pool_row(c, s, b, (int64_t)__ldg(s.lens + b) - __ldg(s.cu + b + 1) + t, head, status);
                if (at[u] >= 0) load8(in.p[which] + t * in.token_stride[which] + head * in.head_stride[which] + word * 8, in.vec, f[u]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float lo = f[u][0], hi = f[u][0];
#pragma unroll
        for (int e = 1; e < 8; e++) { lo = fminf(lo, f[u][e]); hi = fmaxf(hi, f[u][e]); }
#pragma unroll
        for (int o = 1; o < G / 8; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f)), mh = __float2half_rn(lo);
        const float sc = __half2float(sh), m = __half2float(mh);
        uint32_t codes = 0;
        if (sc > 0.0f) {
            const InvDiv d = make_invdiv(sc);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float q = fminf(fmaxf(rintf(div_exact_bounded(f[u][e] - m, d)), 0.0f), 15.0f);
                codes |= (uint32_t)(int)q << (4 * e);
            }
        }
        if (at[u] >= 0) {
            uint8_t* row = (which ? c.vc : c.kc) + at[u] * (D / 2);
            reinterpret_cast<uint32_t*>(row)[which ? value_place(word, D) : key_place(word, D)] = codes;
            if (word % (G / 8) == 0)
                (which ? c.vp : c.kp)[at[u] * (D / G) + word / (G / 8)] = (uint32_t)__half_as_ushort(sh) | ((uint32_t)__half_as_ushort(mh) << 16);
        }
    }
}

// c * s + m in f32: c * s is exact (4 + 11 bits), so there is one rounding, and one more to T.
template <typename T, int D, int G, int U>
__global__ void __launch_bounds__(256) kv4_read_kernel(Pool c, Batch s, T* k_out, T* v_out, int32_t* status) {
    pdl_trigger();
    pdl_wait();
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    const int lane = threadIdx.x & 31, word = lane % LANES;
    const int which = blockIdx.y;
    const int64_t rows = s.tokens * c.heads;
    const int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (PER_WARP * U);
    if (first >= rows) return;
    int b = sequence_of(s.cu, s.seqs, first / c.heads);
    const int place = which ? value_place(word, D) : key_place(word, D);
    uint32_t codes[U], sm[U];
    bool have[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = first + u * PER_WARP + lane / LANES;
        const int64_t t = row / c.heads;
        const int head = (int)(row - t * c.heads);
        have[u] = false;
        codes[u] = 0; sm[u] = 0;
        if (row < rows) {
            while (b < s.seqs && __ldg(s.cu + b + 1) <= t) b++;
            if (b < s.seqs && t >= __ldg(s.cu + b)) {
                have[u] = true;                                     // a token without a page of the pool reads as zeros
                const int64_t at = pool_row(c, s, b, (int64_t)__ldg(s.lens + b) - __ldg(s.cu + b + 1) + t, head, status);
                if (at >= 0) {
                    codes[u] = __ldg(reinterpret_cast<const uint32_t*>((which ? c.vc : c.kc) + at * (D / 2)) + place);
                    sm[u] = __ldg((which ? c.vp : c.kp) + at * (D / G) + word / (G / 8));
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (!have[u]) continue;
        const float sc = __half2float(__ushort_as_half((unsigned short)(sm[u] & 0xFFFFu))), m = __half2float(__ushort_as_half((unsigned short)(sm[u] >> 16)));
        T* out = (which ? v_out : k_out) + (first + u * PER_WARP + lane / LANES) * D + word * 8;
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < 8 / N; i++) {
            Vec16<T> v;
#pragma unroll
            for (int e = 0; e < N; e++) v.v[e] = Elem<T>::from_f32(fmaf((float)((codes[u] >> (4 * (i * N + e))) & 15u), sc, m));
            *reinterpret_cast<uint4*>(out + i * N) = *reinterpret_cast<const uint4*>(&v);
        }
    }
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
    if (s->table_width * c->page_size > INT32_MAX)
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

// Rows per thread: four keep enough loads in flight to stream; one where there are too few rows to fill the machine with
// four (a decode step), so that more SMs take part.
static int rows_per_thread(const oxq_handle* h, int64_t rows, int per_cta) { return rows >= (int64_t)h->sm_count * per_cta * 4 ? 4 : 1; }

template <typename T, int D, int G>
static cudaError_t launch_append(oxq_handle* h, const Pool& c, const Batch& s, const Rows<T>& in) {
    const int64_t rows = s.tokens * c.heads;
    constexpr int CTA = 8 * (32 / (D / 8));
    if (rows_per_thread(h, rows, CTA) == 4)
        return oxq_launch(kv4_append_kernel<T, D, G, 4>, dim3((unsigned)((rows + CTA * 4 - 1) / (CTA * 4)), 2), 256, 0, h->stream, c, s, in, h->dev_status);
    return oxq_launch(kv4_append_kernel<T, D, G, 1>, dim3((unsigned)((rows + CTA - 1) / CTA), 2), 256, 0, h->stream, c, s, in, h->dev_status);
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

template <typename T, int D, int G>
static cudaError_t launch_read(oxq_handle* h, const Pool& c, const Batch& s, void* k, void* v) {
    const int64_t rows = s.tokens * c.heads;
    constexpr int CTA = 8 * (32 / (D / 8));
    if (rows_per_thread(h, rows, CTA) == 4)
        return oxq_launch(kv4_read_kernel<T, D, G, 4>, dim3((unsigned)((rows + CTA * 4 - 1) / (CTA * 4)), 2), 256, 0, h->stream, c, s, (T*)k, (T*)v, h->dev_status);
    return oxq_launch(kv4_read_kernel<T, D, G, 1>, dim3((unsigned)((rows + CTA - 1) / CTA), 2), 256, 0, h->stream, c, s, (T*)k, (T*)v, h->dev_status);
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
    if (int32_t rc = oxq_require_sm100(h)) return rc;
    OxqDeviceGuard guard(h->device);
    switch (dtype) {
        case OXQ_F32: return read_t<float>(h, cache, c, s, k_out, v_out);
        case OXQ_BF16: return read_t<__nv_bfloat16>(h, cache, c, s, k_out, v_out);
        default: return read_t<__half>(h, cache, c, s, k_out, v_out);
    }
}

}  // extern "C"
