// The seam between two blocks of a decoder layer as one pass over its rows:
//   t  = y, or rms(y; post_weight) where the block has a norm behind it;  t *= gate where it has one
//   r' = residual + alpha t
//   h  = rms(r'; weight), stored as it is, as E4M3 at a calibrated scale, or as INT8 with a scale per row
// with rms(x; w) = x / sqrt(mean(x^2) + eps) * w.  All of it is f32; r' is normed before it is rounded to its own type.
// A row is held in registers by TPR threads (NV items of eight elements each, in their own type), so every input is read once and every
// output written once; the sums of squares meet in shared memory, in a fixed order.  Bound by memory: 8190 x 8192 bf16 with all
// parts 123 us = 5.5 TB/s, 0.83 of the copy rate.
// The weights alone are read through the read-only path: the rest is what earlier kernels write, or this one in place.
#include "oxq_common.cuh"

namespace oxq {
namespace resnorm {

enum { OUT_SAME = 0, OUT_FP8 = 1, OUT_INT8 = 2 };

struct Params {
    const void* y; int64_t y_ld;
    const void* residual; int64_t r_ld;
    const void* gate; int64_t g_ld;             // null: none; leading dimension 0: the same for every row
    const float* post; const float* weight;
    float alpha, eps;
    void* residual_out; int64_t ro_ld;
    void* out;                                  // h, its E4M3 bytes or its INT8 codes: [rows x cols]
    float* row_scales;                          // INT8
    const float* scale;                         // E4M3
    int64_t rows, cols;
    int mode;
};

// Eight elements as they lie: a row waits in registers in its own type, not in f32.
template <typename T> struct Eight { uint4 v[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Eight<T> load8(const T* p) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) {
        const Vec16<uint32_t> v = ld16_written_stream(reinterpret_cast<const uint32_t*>(p) + 4 * i);
        r.v[i] = make_uint4(v.v[0], v.v[1], v.v[2], v.v[3]);
    }
    return r;
}
template <typename T> __device__ __forceinline__ Eight<T> zero8() {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.v[i] = make_uint4(0, 0, 0, 0);
    return r;
}
template <typename T> __device__ __forceinline__ float element(const Eight<T>& r, int e) {
    const uint4 v = r.v[sizeof(T) == 4 ? e >> 2 : 0];
    const int i = sizeof(T) == 4 ? e & 3 : e >> 1;
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (Elem<T>::kDtype == OXQ_BF16) return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
    else return __half2float(__ushort_as_half((unsigned short)(w >> (16 * (e & 1)))));
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8 / N; i++) {
        Vec16<T> v;
#pragma unroll
        for (int e = 0; e < N; e++) v.v[e] = Elem<T>::from_f32(f[i * N + e]);
        *reinterpret_cast<uint4*>(p + i * N) = *reinterpret_cast<const uint4*>(&v);
    }
}
__device__ __forceinline__ void weight8(const float* p, float (&f)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// the larger one, or NaN where one is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Over the TPR threads of a row; `red` holds a word per warp of the CTA.
template <int TPR, bool MAX> __device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = threadIdx.x >> 5, first = warp / W * W;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[warp] = v;
        __syncthreads();
        v = red[first];
#pragma unroll
        for (int i = 1; i < W; i++) v = MAX ? max_nan(v, red[first + i]) : v + red[first + i];
    }
    return v;
}

template <typename T, typename R, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) residual_rmsnorm_kernel(Params p) {
    pdl_trigger();
    pdl_wait();
    __shared__ float red[32];
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    const int64_t row0 = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    const bool live = row0 < p.rows;
    const int64_t row = live ? row0 : p.rows - 1;                   // idle threads of the last CTA meet the barriers
    const int64_t items = p.cols >> 3;
    const int lane = threadIdx.x % TPR;
    Eight<T> y[NV], gate[NV];
    Eight<R> res[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t it = lane + i * TPR;
        y[i] = zero8<T>(); gate[i] = zero8<T>(); res[i] = zero8<R>();
        if (it < items) {
            y[i] = load8((const T*)p.y + row * p.y_ld + it * 8);
            res[i] = load8((const R*)p.residual + row * p.r_ld + it * 8);
            if (p.gate) gate[i] = load8((const T*)p.gate + row * p.g_ld + it * 8);
        }
    }
    float k = p.alpha;
    if (p.post) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(element(y[i], e), element(y[i], e), ss);
        ss = row_reduce<TPR, false>(ss, red);
        k *= __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)p.cols) + p.eps));
    }
    float ss = 0.0f, r[NV][8];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t it = lane + i * TPR;
#pragma unroll
        for (int e = 0; e < 8; e++) r[i][e] = 0.0f;
        if (it < items) {
            float t[8], w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) t[e] = element(y[i], e);
            if (p.post) {
                weight8(p.post + it * 8, w);
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] *= w[e];
            }
            if (p.gate) {
#pragma unroll
                for (int e = 0; e < 8; e++) t[e] *= element(gate[i], e);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                r[i][e] = fmaf(k, t[e], element(res[i], e));
                ss = fmaf(r[i][e], r[i][e], ss);
            }
            if (live) store8((R*)p.residual_out + row * p.ro_ld + it * 8, r[i]);
        }
    }
    ss = row_reduce<TPR, false>(ss, red);
    const float inv = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)p.cols) + p.eps));
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t it = lane + i * TPR;
        if (it < items) {
            float w[8];
            weight8(p.weight + it * 8, w);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                r[i][e] = r[i][e] * inv * w[e];
                top = max_nan(top, fabsf(r[i][e]));
            }
        }
    }
    InvDiv d;
    if (p.mode == OUT_INT8) {
        top = row_reduce<TPR, true>(top, red);
        const float sc = __fdiv_rn(max_nan(top, 1e-8f), 127.0f);        // a NaN or an infinity in the row has made an h NaN: so is then the scale, codes have no NaN
        if (live && lane == 0) p.row_scales[row] = sc;
        d = make_invdiv(sc);
    } else if (p.mode == OUT_FP8) {
        d = make_invdiv(*p.scale);
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t it = lane + i * TPR;
        if (it >= items || !live) continue;
        if (p.mode == OUT_SAME) {
            store8((T*)p.out + row * p.cols + it * 8, r[i]);
        } else {
            uint2 o;
            if (p.mode == OUT_FP8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = div_exact(r[i][e], d);
                o.x = (uint32_t)cvt_e4m3x2(v[0], v[1]) | ((uint32_t)cvt_e4m3x2(v[2], v[3]) << 16);
                o.y = (uint32_t)cvt_e4m3x2(v[4], v[5]) | ((uint32_t)cvt_e4m3x2(v[6], v[7]) << 16);
            } else {
                uint32_t q[8];
#pragma unroll
                for (int e = 0; e < 8; e++) q[e] = (uint32_t)(int)fminf(fmaxf(rintf(div_exact_bounded(r[i][e], d)), -127.0f), 127.0f) & 0xFFu;
                o.x = q[0] | (q[1] << 8) | (q[2] << 16) | (q[3] << 24);
                o.y = q[4] | (q[5] << 8) | (q[6] << 16) | (q[7] << 24);
            }
            *reinterpret_cast<uint2*>((uint8_t*)p.out + row * p.cols + it * 8) = o;
        }
    }
}

// Threads per row.  With rows enough to fill the machine, what holds the row at two items each: y, residual and gate of a row
// are then all in flight at 64 registers a thread, 32 warps on an SM (8190 x 8192 bf16 with all parts: 173 us with half the
// threads and four items).  With fewer rows than that, one item a thread, for the latency.
template <typename T, typename R>
static cudaError_t launch(oxq_handle* h, const Params& p) {
    const int64_t items = p.cols >> 3;
#define OXQ_RN(TPR, NV) \
    oxq_launch(residual_rmsnorm_kernel<T, R, TPR, NV>, (unsigned)((p.rows + (TPR < 256 ? 256 / TPR : 1) - 1) / (TPR < 256 ? 256 / TPR : 1)), TPR < 256 ? 256 : TPR, 0, h->stream, p)
    if (p.rows >= 2 * (int64_t)h->sm_count) {
        if (items <= 64) return OXQ_RN(32, 2);
        if (items <= 128) return OXQ_RN(64, 2);
        if (items <= 256) return OXQ_RN(128, 2);
        if (items <= 512) return OXQ_RN(256, 2);
        if (items <= 1024) return OXQ_RN(512, 2);
        return OXQ_RN(1024, 2);
    }
    if (items <= 128) return OXQ_RN(128, 1);
    if (items <= 512) return OXQ_RN(512, 1);
    if (items <= 1024) return OXQ_RN(1024, 1);
    return OXQ_RN(1024, 2);
#undef OXQ_RN
}

}  // namespace resnorm
}  // namespace oxq

using namespace oxq;
using namespace oxq::resnorm;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static int32_t residual_rmsnorm(oxq_handle* h, const oxq_residual_norm* a, int64_t rows, int64_t cols, int mode, void* out, const float* scale, float* row_scales) {
    OXQ_CHECK_HANDLE(h);
    if (!a) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "residual rmsnorm: null arguments");
    if (rows <= 0 || cols <= 0) OXQ_FAIL(h, OXQ_ERR_EMPTY_INPUT, "residual rmsnorm: empty input");
    if (cols % 8 != 0 || cols > 16384) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "residual rmsnorm: cols must be a multiple of 8 and at most 16384, got %lld", (long long)cols);
    if (rows > INT32_MAX) OXQ_FAIL(h, OXQ_ERR_INVALID_DIMENSION, "residual rmsnorm: %lld rows", (long long)rows);
    if (!a->y || !a->residual || !a->weight || !a->residual_out || !out || (mode == OUT_FP8 && !scale) || (mode == OUT_INT8 && !row_scales))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "residual rmsnorm: null pointer");
    if (!aligned16(a->y) || !aligned16(a->residual) || !aligned16(a->weight) || !aligned16(a->residual_out) || (a->gate && !aligned16(a->gate)) ||
        (a->post_weight && !aligned16(a->post_weight)) || ((uintptr_t)out & (mode == OUT_SAME ? 15u : 7u)))
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "residual rmsnorm: misaligned pointer");
    if (a->y_ld < cols || a->residual_ld < cols || a->residual_out_ld < cols || (a->gate && a->gate_ld != 0 && a->gate_ld < cols) ||
        (a->y_ld | a->residual_ld | a->residual_out_ld | (a->gate ? a->gate_ld : 0)) % 8 != 0)
        OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "residual rmsnorm: leading dimensions are multiples of 8 and not below cols");
    if (a->dtype != OXQ_F32 && a->dtype != OXQ_BF16 && a->dtype != OXQ_F16) OXQ_FAIL(h, OXQ_ERR_INVALID_ARGUMENT, "unknown dtype %d", a->dtype);
    if (a->residual_dtype != a->dtype && a->residual_dtype != OXQ_F32)
        OXQ_FAIL(h, OXQ_ERR_UNSUPPORTED_OPERATION, "residual rmsnorm: the residual has the type of y or is f32");
    if (int32_t rc = oxq_require_sm100(h)) return rc;
    OxqDeviceGuard guard(h->device);
    Params p;
    p.y = a->y; p.y_ld = a->y_ld; p.residual = a->residual; p.r_ld = a->residual_ld; p.gate = a->gate; p.g_ld = a->gate_ld;
    p.post = a->post_weight; p.weight = a->weight; p.alpha = a->alpha; p.eps = a->eps; p.residual_out = a->residual_out; p.ro_ld = a->residual_out_ld;
    p.out = out; p.row_scales = row_scales; p.scale = scale; p.rows = rows; p.cols = cols; p.mode = mode;
    const bool wide = a->residual_dtype == OXQ_F32;
    switch (a->dtype) {
        case OXQ_F32: OXQ_CUDA(h, (launch<float, float>(h, p))); break;
        case OXQ_BF16: if (wide) OXQ_CUDA(h, (launch<__nv_bfloat16, float>(h, p))); else OXQ_CUDA(h, (launch<__nv_bfloat16, __nv_bfloat16>(h, p))); break;
        default: if (wide) OXQ_CUDA(h, (launch<__half, float>(h, p))); else OXQ_CUDA(h, (launch<__half, __half>(h, p))); break;
    }
    return OXQ_OK;
}

extern "C" {

int32_t oxq_residual_rmsnorm(oxq_handle* h, const oxq_residual_norm* args, int64_t rows, int64_t cols, void* out) {
    return residual_rmsnorm(h, args, rows, cols, OUT_SAME, out, nullptr, nullptr);
}
int32_t oxq_residual_rmsnorm_fp8(oxq_handle* h, const oxq_residual_norm* args, int64_t rows, int64_t cols, const float* scale, uint8_t* q) {
    return residual_rmsnorm(h, args, rows, cols, OUT_FP8, q, scale, nullptr);
}
int32_t oxq_residual_rmsnorm_int8_rows(oxq_handle* h, const oxq_residual_norm* args, int64_t rows, int64_t cols, int8_t* q, float* scales) {
    return residual_rmsnorm(h, args, rows, cols, OUT_INT8, q, nullptr, scales);
}

}  // extern "C"
