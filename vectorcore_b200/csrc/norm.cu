// norm.cu -- root-mean-square norm with the residual's addition, forward and
// backward, and its 8-bit output with a scale for each row.
//
//   h = x + residual          s = 1 / sqrt(mean(h^2) + eps)
//   y = (h * s) * w
//   dh = s * (t - h * (s^2 * mean(t * h))) + gh,  t = gy * w
//   dw = sum over rows of gy * (h * s)
//   8 bits: u = h * w, M = max |u|, q = rint(u * (127 / M)), scale = (M * s) / 127
//
// In the 8-bit form s is common to the whole row, so q does not depend on it
// and one pass over the row yields both reductions (the sum of squares and M).
#include "vc_internal.cuh"

#include <cmath>

namespace vc {
namespace {

// What a row's pass computes.
enum NormMode { NORM_F32 = 0, NORM_Q8 = 1, QUANT_Q8 = 2 };

struct NormArgs {
    const float* x;
    unsigned long long xs;  // elements between rows of x
    const float* r;         // residual or null
    unsigned long long rs;
    const float* w;
    unsigned long long rows;
    unsigned cols;
    float eps;
    float* h;  // x + residual, or null
    float* y;
    float* rstd;  // or null
    signed char* q;
    unsigned long long pitch;  // bytes between rows of q
    float* scale;
};

// Rows whose largest |u| is below this quantise to zeros with scale 0: 127 / M
// stays finite above it.
constexpr float kQ8Tiny = 0x1p-100f;

struct RowStats {
    double sq;
    float amax;
};

__device__ __forceinline__ float warp_amax(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// The row's sum of squares and largest |u|, in every thread of its T threads.
// fmaxf drops NaN; a NaN (or infinity) shows in the sum, or in `bad` for
// QUANT_Q8, and poisons the row's scale.
template <int MODE>
__device__ __forceinline__ RowStats reduce_row(double sq, float amax, double* ssq, float* smax) {
    const unsigned nw = blockDim.x >> 5;
    if (MODE != QUANT_Q8) sq = warp_sum(sq);
    if (MODE != NORM_F32) amax = warp_amax(amax);
    if (nw > 1) {
        const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) {
            ssq[warp] = sq;
            smax[warp] = amax;
        }
        __syncthreads();
        sq = lane < nw ? ssq[lane] : 0.0;
        amax = lane < nw ? smax[lane] : 0.0f;
        if (MODE != QUANT_Q8) sq = warp_sum(sq);
        if (MODE != NORM_F32) amax = warp_amax(amax);
    }
    return RowStats{sq, amax};
}

template <int VEC>
struct Group {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Group<VEC> load_group(const float* p, unsigned long long g) {
    Group<VEC> o;
    if constexpr (VEC == 4) {
        const float4 f = reinterpret_cast<const float4*>(p)[g];
        o.v[0] = f.x, o.v[1] = f.y, o.v[2] = f.z, o.v[3] = f.w;
    } else {
        o.v[0] = p[g];
    }
    return o;
}

template <int VEC>
__device__ __forceinline__ void store_group(float* p, unsigned long long g, const Group<VEC>& o) {
    if constexpr (VEC == 4)
        reinterpret_cast<float4*>(p)[g] = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
    else
        p[g] = o.v[0];
}

// max |u| as fmaxf, but a NaN stays: NaN compares false, so it is kept by the
// second select and never replaced.
__device__ __forceinline__ float amax_nan(float m, float a) { return m >= a ? m : (m != m ? m : a); }

struct Q8Row {
    float inv;    // 127 / M, or 0 for a zero or non-finite row
    float scale;  // what one step stands for
};
__device__ __forceinline__ Q8Row q8_row(float amax, float rstd) {
    Q8Row o;
    if (!(amax < INFINITY)) {  // NaN or infinity somewhere in the row
        o.inv = 0.0f;
        o.scale = NAN;
    } else if (amax < kQ8Tiny) {
        o.inv = 0.0f;
        o.scale = 0.0f;
    } else {
        o.inv = 127.0f / amax;
        o.scale = amax * (1.0f / 127.0f) * rstd;
    }
    return o;
}
// u * inv rounds to at most 127: M * (127 / M) is below 127.00002.
__device__ __forceinline__ int q8_value(float u, float inv) { return inv == 0.0f ? 0 : __float2int_rn(u * inv); }

// One row a CTA (or a row a warp, blockDim.y of them, for short rows): the row
// is read once and stays in registers, NV groups of VEC floats a thread.
template <int MODE, int VEC, int NV>
__global__ void __launch_bounds__(1024)
norm_kernel(const NormArgs a) {
    __shared__ double ssq[32];
    __shared__ float smax[32];
    const unsigned long long row = static_cast<unsigned long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // whole warps: blockDim.y > 1 only with one warp a row
    const unsigned T = blockDim.x, t = threadIdx.x;
    const unsigned G = a.cols / VEC;  // VEC divides cols
    const float* x = a.x + row * a.xs;
    const float* r = a.r ? a.r + row * a.rs : nullptr;
    Group<VEC> h[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned g = t + i * T;
        if (g < G) h[i] = load_group<VEC>(x, g);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[i].v[e] = 0.0f;
    }
    if (r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned g = t + i * T;
            if (g < G) {
                const Group<VEC> o = load_group<VEC>(r, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i].v[e] += o.v[e];
            }
        }
    }
    double sq = 0.0;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned g = t + i * T;
        if (g < G) {
            if (a.h) store_group<VEC>(a.h + row * a.cols, g, h[i]);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) part = fmaf(h[i].v[e], h[i].v[e], part);
            if (MODE != QUANT_Q8) sq += part;
            if (MODE == NORM_Q8) {
                const Group<VEC> w = load_group<VEC>(a.w, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i].v[e] *= w.v[e];
            }
            if (MODE != NORM_F32)
#pragma unroll
                for (int e = 0; e < VEC; ++e) amax = amax_nan(amax, fabsf(h[i].v[e]));
        }
    }
    // a NaN maximum survives the fmaxf tree as infinity (both poison the row)
    if (MODE != NORM_F32 && amax != amax) amax = INFINITY;
    const RowStats st = reduce_row<MODE>(sq, amax, ssq, smax);
    const float rstd = MODE == QUANT_Q8 ? 1.0f : 1.0f / sqrtf(static_cast<float>(st.sq / a.cols) + a.eps);
    if (MODE != QUANT_Q8 && a.rstd && t == 0) a.rstd[row] = rstd;
    if (MODE == NORM_F32) {
        float* y = a.y + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned g = t + i * T;
            if (g < G) {
                const Group<VEC> w = load_group<VEC>(a.w, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i].v[e] = h[i].v[e] * rstd * w.v[e];
                store_group<VEC>(y, g, h[i]);
            }
        }
    } else {
        const Q8Row o = q8_row(st.amax, rstd);
        if (t == 0) a.scale[row] = o.scale;
        signed char* q = a.q + row * a.pitch;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned g = t + i * T;
            if (g < G) {
                if constexpr (VEC == 4)
                    reinterpret_cast<char4*>(q)[g] =
                        make_char4(q8_value(h[i].v[0], o.inv), q8_value(h[i].v[1], o.inv), q8_value(h[i].v[2], o.inv),
                                   q8_value(h[i].v[3], o.inv));
                else
                    q[g] = static_cast<signed char>(q8_value(h[i].v[0], o.inv));
            }
        }
        for (unsigned long long j = a.cols + t; j < a.pitch; j += T) q[j] = 0;
    }
}

// Rows too long for the registers of one CTA: the same in two passes, the
// second reading h back (or x and the residual again where h is not wanted).
template <int MODE>
__global__ void __launch_bounds__(1024)
norm_long_kernel(const NormArgs a) {
    __shared__ double ssq[32];
    __shared__ float smax[32];
    const unsigned long long row = blockIdx.x;
    const float* x = a.x + row * a.xs;
    const float* r = a.r ? a.r + row * a.rs : nullptr;
    float* h = a.h ? a.h + row * a.cols : nullptr;
    double sq = 0.0;
    float amax = 0.0f;
    for (unsigned j = threadIdx.x; j < a.cols; j += blockDim.x) {
        const float v = r ? x[j] + r[j] : x[j];
        if (h) h[j] = v;
        if (MODE != QUANT_Q8) sq += static_cast<double>(v) * v;
        if (MODE == NORM_Q8) amax = amax_nan(amax, fabsf(v * a.w[j]));
        if (MODE == QUANT_Q8) amax = amax_nan(amax, fabsf(v));
    }
    if (MODE != NORM_F32 && amax != amax) amax = INFINITY;
    const RowStats st = reduce_row<MODE>(sq, amax, ssq, smax);
    const float rstd = MODE == QUANT_Q8 ? 1.0f : 1.0f / sqrtf(static_cast<float>(st.sq / a.cols) + a.eps);
    if (MODE != QUANT_Q8 && a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    Q8Row o{};
    if (MODE != NORM_F32) {
        o = q8_row(st.amax, rstd);
        if (threadIdx.x == 0) a.scale[row] = o.scale;
    }
    for (unsigned j = threadIdx.x; j < a.cols; j += blockDim.x) {
        const float v = h ? h[j] : (r ? x[j] + r[j] : x[j]);
        if (MODE == NORM_F32) a.y[row * a.cols + j] = v * rstd * a.w[j];
        else
            a.q[row * a.pitch + j] = static_cast<signed char>(q8_value(MODE == NORM_Q8 ? v * a.w[j] : v, o.inv));
    }
    if (MODE != NORM_F32)
        for (unsigned long long j = a.cols + threadIdx.x; j < a.pitch; j += blockDim.x) a.q[row * a.pitch + j] = 0;
}

// Floats a CTA of 1024 threads keeps in registers (32 a thread).
constexpr unsigned kNormRegCols = 32768;

template <int MODE, int VEC, int NV>
void launch_norm_nv(const NormArgs& a, unsigned T, unsigned R) {
    const unsigned long long ctas = (a.rows + R - 1) / R;
    if (ctas > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm: too many rows");
    norm_kernel<MODE, VEC, NV><<<static_cast<unsigned>(ctas), dim3(T, R), 0, stream()>>>(a);
    check_launch("norm_kernel");
}

template <int MODE>
void launch_norm(const NormArgs& a) {
    if (a.cols > kNormRegCols) {
        if (a.rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm: too many rows");
        norm_long_kernel<MODE><<<static_cast<unsigned>(a.rows), 1024, 0, stream()>>>(a);
        check_launch("norm_long_kernel");
        return;
    }
    const bool vec = a.cols % 4 == 0 && aligned16(a.x) && (a.rows == 1 || a.xs % 4 == 0) &&
                     (!a.r || (aligned16(a.r) && (a.rows == 1 || a.rs % 4 == 0))) && (!a.w || aligned16(a.w)) &&
                     (!a.h || aligned16(a.h)) && (!a.y || aligned16(a.y));
    const unsigned groups = vec ? a.cols / 4 : a.cols;
    const unsigned per = vec ? 4 : 8;  // groups a thread, while 1024 threads are enough
    unsigned T = std::min(1024u, ((groups + per - 1) / per + 31) / 32 * 32);
    const unsigned R = T == 32 ? 8 : 1;
    const unsigned nv = (groups + T - 1) / T;
    if (vec) {
        if (nv <= 4) launch_norm_nv<MODE, 4, 4>(a, T, R);
        else launch_norm_nv<MODE, 4, 8>(a, T, R);
    } else {
        if (nv <= 8) launch_norm_nv<MODE, 1, 8>(a, T, R);
        else launch_norm_nv<MODE, 1, 32>(a, T, R);
    }
}

// ---- backward -----------------------------------------------------------------

struct NormBwdArgs {
    const float* h;
    const float* w;
    const float* rstd;
    const float* gy;
    const float* gh;  // or null
    unsigned long long rows;
    unsigned cols;
    float* dh;
};

__global__ void __launch_bounds__(256)
norm_bwd_dh(const NormBwdArgs a) {
    __shared__ double scratch[32];
    const unsigned long long at = static_cast<unsigned long long>(blockIdx.x) * a.cols;
    double dot = 0.0;
    for (unsigned j = threadIdx.x; j < a.cols; j += blockDim.x)
        dot += static_cast<double>(a.gy[at + j] * a.w[j]) * a.h[at + j];
    dot = block_sum(dot, scratch);
    const float s = a.rstd[blockIdx.x];
    const float c = static_cast<float>(dot / a.cols) * (s * s);
    for (unsigned j = threadIdx.x; j < a.cols; j += blockDim.x) {
        const float v = s * (a.gy[at + j] * a.w[j] - a.h[at + j] * c);
        a.dh[at + j] = a.gh ? v + a.gh[at + j] : v;
    }
}

__global__ void __launch_bounds__(256)
norm_bwd_dw(const NormBwdArgs a, float* __restrict__ dw) {
    const unsigned j = blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= a.cols) return;
    double s = 0.0;
    for (unsigned long long i = 0; i < a.rows; ++i) s += a.gy[i * a.cols + j] * (a.h[i * a.cols + j] * a.rstd[i]);
    dw[j] = static_cast<float>(s);
}

void check_rows_cols(const char* what, std::size_t rows, std::size_t cols) {
    if (cols == 0) fail(VC_ERR_INVALID, std::string(what) + ": a row needs at least one column");
    if (cols > 0x7fffffffu) fail(VC_ERR_OVERFLOW, std::string(what) + ": row too long");
    if (rows > (1ull << 62) / cols / sizeof(float)) fail(VC_ERR_OVERFLOW, std::string(what) + ": tensor too large");
}

void check_q8_out(const char* what, const void* q, const float* scale, std::size_t cols, std::size_t pitch) {
    if (!q || !scale) fail(VC_ERR_INVALID, std::string(what) + ": null pointer");
    if (pitch < cols || pitch % 16 != 0 || !aligned16(q))
        fail(VC_ERR_INVALID, std::string(what) + ": 8-bit rows need a pitch of at least the row's length, and a "
                                                 "multiple of 16 bytes, on a 16-byte aligned base");
}

void check_eps(const char* what, float eps) {
    if (!(eps >= 0.0f) || !std::isfinite(eps)) fail(VC_ERR_INVALID, std::string(what) + ": eps must be finite and not negative");
}

}  // namespace
}  // namespace vc

using namespace vc;

extern "C" {

vc_status vc_cuda_rms_norm(const float* x, size_t x_stride, const float* residual, size_t residual_stride,
                           const float* weight, size_t rows, size_t cols, float eps, float* h, float* y,
                           float* rstd) {
    VC_API_BEGIN
    ensure_init();
    check_rows_cols("rms_norm", rows, cols);
    check_eps("rms_norm", eps);
    if (rows == 0) return VC_OK;
    if (!x || !weight || !y) fail(VC_ERR_INVALID, "rms_norm: null pointer");
    NormArgs a{};
    a.x = x, a.xs = x_stride, a.r = residual, a.rs = residual_stride, a.w = weight;
    a.rows = rows, a.cols = static_cast<unsigned>(cols), a.eps = eps;
    a.h = h, a.y = y, a.rstd = rstd;
    launch_norm<NORM_F32>(a);
    VC_API_END
}

vc_status vc_cuda_rms_norm_q8(const float* x, size_t x_stride, const float* residual, size_t residual_stride,
                              const float* weight, size_t rows, size_t cols, float eps, float* h, int8_t* q,
                              size_t q_pitch, float* scale) {
    VC_API_BEGIN
    ensure_init();
    check_rows_cols("rms_norm_q8", rows, cols);
    check_eps("rms_norm_q8", eps);
    if (rows == 0) return VC_OK;
    if (!x || !weight) fail(VC_ERR_INVALID, "rms_norm_q8: null pointer");
    check_q8_out("rms_norm_q8", q, scale, cols, q_pitch);
    NormArgs a{};
    a.x = x, a.xs = x_stride, a.r = residual, a.rs = residual_stride, a.w = weight;
    a.rows = rows, a.cols = static_cast<unsigned>(cols), a.eps = eps;
    a.h = h, a.q = q, a.pitch = q_pitch, a.scale = scale;
    launch_norm<NORM_Q8>(a);
    VC_API_END
}

vc_status vc_cuda_quantize_q8(const float* x, size_t x_stride, size_t rows, size_t cols, int8_t* q, size_t q_pitch,
                              float* scale) {
    VC_API_BEGIN
    ensure_init();
    check_rows_cols("quantize_q8", rows, cols);
    if (rows == 0) return VC_OK;
    if (!x) fail(VC_ERR_INVALID, "quantize_q8: null pointer");
    check_q8_out("quantize_q8", q, scale, cols, q_pitch);
    NormArgs a{};
    a.x = x, a.xs = x_stride;
    a.rows = rows, a.cols = static_cast<unsigned>(cols);
    a.q = q, a.pitch = q_pitch, a.scale = scale;
    launch_norm<QUANT_Q8>(a);
    VC_API_END
}

vc_status vc_cuda_rms_norm_backward(const float* h, const float* weight, const float* rstd, const float* gy,
                                    const float* gh, size_t rows, size_t cols, float* dh, float* dw) {
    VC_API_BEGIN
    ensure_init();
    check_rows_cols("rms_norm_backward", rows, cols);
    if (rows == 0) {  // the sum over no rows
        if (dw) VC_CUDA(cudaMemsetAsync(dw, 0, cols * sizeof(float), stream()));
        return VC_OK;
    }
    if (!h || !weight || !rstd || !gy) fail(VC_ERR_INVALID, "rms_norm_backward: null pointer");
    if (!dh && !dw) return VC_OK;
    if (rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm_backward: too many rows");
    NormBwdArgs a{h, weight, rstd, gy, gh, rows, static_cast<unsigned>(cols), dh};
    if (dw) {
        norm_bwd_dw<<<static_cast<unsigned>((cols + 255) / 256), 256, 0, stream()>>>(a, dw);
        check_launch("norm_bwd_dw");
    }
    if (dh) {
        norm_bwd_dh<<<static_cast<unsigned>(rows), 256, 0, stream()>>>(a);
        check_launch("norm_bwd_dh");
    }
    VC_API_END
}

}  // extern "C"
