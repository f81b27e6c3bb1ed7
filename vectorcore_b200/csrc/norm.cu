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

// The row's sum of squares and largest |u| (no NaN: the callers make it infinity),
// in every thread of its T threads.
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

// A row in groups of four floats on the 16-byte grid of its address. Rows whose
// length is no multiple of four start anywhere on it: with `skew` floats between
// the grid and the row's start, group g holds the elements 4g - skew ..
// 4g - skew + 3, and the first and last group may hold fewer.
struct Span {
    unsigned skew, cols;
    __device__ __forceinline__ unsigned groups() const { return (skew + cols + 3) >> 2; }
    __device__ __forceinline__ bool whole(unsigned g) const { return 4 * g >= skew && 4 * g + 4 <= skew + cols; }
    __device__ __forceinline__ bool has(unsigned g, unsigned e) const {
        return 4 * g + e >= skew && 4 * g + e < skew + cols;
    }
};
struct Group {
    float v[4];
};
__device__ __forceinline__ Group group_of(float4 f) { return Group{{f.x, f.y, f.z, f.w}}; }

// p: the row's start. SKEWED false: every row starts on the grid and ends on it.
template <bool SKEWED>
__device__ __forceinline__ Group load_group(const float* p, unsigned g, const Span& r) {
    if constexpr (!SKEWED) {
        return group_of(reinterpret_cast<const float4*>(p)[g]);
    } else {
        if (r.whole(g)) return group_of(*reinterpret_cast<const float4*>(p - r.skew + 4ull * g));
        Group o;
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) o.v[e] = r.has(g, e) ? p[4 * g + e - r.skew] : 0.0f;
        return o;
    }
}
// The norm's weight, which no output overlaps: read-only loads can be issued
// ahead of the stores (without that the forward ran at 45% of its speed). It
// starts on the grid, so a skewed group is four loads (the ends of two of the
// grid's groups, put together by selects, took as long).
template <bool SKEWED>
__device__ __forceinline__ Group load_weight(const float* w, unsigned g, const Span& r) {
    if constexpr (!SKEWED) {
        return group_of(__ldg(reinterpret_cast<const float4*>(w) + g));
    } else {
        Group o;
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) o.v[e] = r.has(g, e) ? __ldg(w + (4 * g + e - r.skew)) : 0.0f;
        return o;
    }
}
template <bool SKEWED>
__device__ __forceinline__ void store_group(float* p, unsigned g, const Group& o, const Span& r) {
    const float4 f = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
    if constexpr (!SKEWED) {
        reinterpret_cast<float4*>(p)[g] = f;
    } else if (r.whole(g)) {
        *reinterpret_cast<float4*>(p - r.skew + 4ull * g) = f;
    } else {
#pragma unroll
        for (unsigned e = 0; e < 4; ++e)
            if (r.has(g, e)) p[4 * g + e - r.skew] = o.v[e];
    }
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

__device__ __forceinline__ unsigned skew_of(const float* p) {
    return static_cast<unsigned>(reinterpret_cast<std::uintptr_t>(p) >> 2) & 3;
}

// A row of int8 values up to the next 16 bytes.
__host__ __device__ __forceinline__ unsigned q8_bytes(unsigned cols) { return (cols + 15) & ~15u; }

// One row a CTA (or a row a warp, blockDim.y of them, for short rows): the row
// is read once and stays in registers, NV groups a thread; HBM bounds it. 8192 x
// 8192: 158 us for the norm (6.8 TB/s), 129 in 8 bits (6.8), 57 for the 8 bits
// alone; rows off the 16-byte grid run at 5.4 TB/s (8000 x 5003: 118 us), their 8 bits
// at 4.3, bound by instructions.
template <int MODE, bool SKEWED, int NV>
__global__ void __launch_bounds__(1024)
norm_kernel(const NormArgs a) {
    __shared__ double ssq[32];
    __shared__ float smax[32];
    const unsigned long long row = static_cast<unsigned long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // whole warps: blockDim.y > 1 only with one warp a row
    const unsigned T = blockDim.x, t = threadIdx.x;
    const float* x = a.x + row * a.xs;
    const float* r = a.r ? a.r + row * a.rs : nullptr;
    const Span span{SKEWED ? skew_of(x) : 0, a.cols};
    const unsigned G = span.groups();
    Group h[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned g = t + i * T;
        h[i] = g < G ? load_group<SKEWED>(x, g, span) : Group{};
    }
    if (r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned g = t + i * T;
            if (g < G) {
                const Group o = load_group<SKEWED>(r, g, span);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[i].v[e] += o.v[e];
            }
        }
    }
    double sq = 0.0;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned g = t + i * T;
        if (g < G) {
            if (a.h) store_group<SKEWED>(a.h + row * a.cols, g, h[i], span);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) part = fmaf(h[i].v[e], h[i].v[e], part);
            if (MODE != QUANT_Q8) sq += part;
            if (MODE == NORM_Q8) {
                const Group w = load_weight<SKEWED>(a.w, g, span);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[i].v[e] *= w.v[e];
            }
            if (MODE != NORM_F32)
#pragma unroll
                for (int e = 0; e < 4; ++e) amax = amax_nan(amax, fabsf(h[i].v[e]));
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
                const Group w = load_weight<SKEWED>(a.w, g, span);
#pragma unroll
                for (int e = 0; e < 4; ++e) h[i].v[e] = h[i].v[e] * rstd * w.v[e];
                store_group<SKEWED>(y, g, h[i], span);
            }
        }
    } else {
        const Q8Row o = q8_row(st.amax, rstd);
        if (t == 0) a.scale[row] = o.scale;
        signed char* q = a.q + row * a.pitch;
        if constexpr (!SKEWED) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const unsigned g = t + i * T;
                int v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = q8_value(h[i].v[e], o.inv);
                if (g < G) reinterpret_cast<char4*>(q)[g] = make_char4(v[0], v[1], v[2], v[3]);
            }
            for (unsigned long long j = a.cols + t; j < a.pitch; j += T) q[j] = 0;
        } else {
            // The row of q starts on the grid, the groups do not: their bytes meet in
            // shared memory, those ahead of the row in 16 of its own. (Joined by
            // shuffles, the ends of warps by bytes, 30000 x 2047 took 127 us without
            // the norm, now 78.)
            extern __shared__ __align__(16) signed char rows[];
            const unsigned bytes = q8_bytes(a.cols);
            signed char* out = rows + threadIdx.y * (16 + bytes) + 16;
            if (t < bytes - a.cols) out[a.cols + t] = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const unsigned g = t + i * T;
                if (g >= G) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out[static_cast<int>(4 * g + e) - static_cast<int>(span.skew)] =
                        static_cast<signed char>(q8_value(h[i].v[e], o.inv));
            }
            if (T > 32) __syncthreads();
            else __syncwarp();
            for (unsigned c = t; c < bytes / 16; c += T)
                reinterpret_cast<int4*>(q)[c] = reinterpret_cast<const int4*>(out)[c];
            for (unsigned long long j = bytes + t; j < a.pitch; j += T) q[j] = 0;
        }
    }
}

// Rows too long for the registers of one CTA, or tensors of unlike alignment: the
// same in two passes by single floats, the second reading h back (or x and the
// residual again where h is not wanted). 8192 x 8192 of unlike ones: 269 us, 4.0 TB/s.
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

// Row lengths that a CTA of 1024 threads keeps in registers: eight groups a
// thread forward, four of two tensors backward.
constexpr unsigned kNormRegCols = 32768, kNormBwdRegCols = 16384;
bool fits(unsigned cols, unsigned most, bool skewed) { return cols <= (skewed ? most - 3 : most); }

// Threads a row: four groups each, so that a thread has enough loads in flight,
// or one each where the rows are fewer than the SMs and latency counts.
struct RowShape {
    unsigned threads, rows, per;  // threads a row, rows a CTA, groups a thread
};
RowShape row_shape(unsigned cols, bool skewed, std::size_t rows) {
    const unsigned groups = skewed ? (cols + 3 + 3) / 4 : cols / 4;
    const unsigned want = rows <= static_cast<unsigned>(sm_count()) ? 1 : 4;
    RowShape s{};
    s.threads = std::min(1024u, ((groups + want - 1) / want + 31) / 32 * 32);
    s.rows = s.threads == 32 ? 8 : 1;
    s.per = (groups + s.threads - 1) / s.threads;
    return s;
}

// Whether rows `stride` floats apart from p lie on the 16-byte grid.
bool on_grid(const float* p, std::size_t stride, std::size_t rows) {
    return !p || (aligned16(p) && (rows == 1 || stride % 4 == 0));
}
// Whether both tensors' rows have the same skew, row by row.
bool same_skew(const float* p, std::size_t ps, const float* q, std::size_t qs, std::size_t rows) {
    return !q || ((reinterpret_cast<std::uintptr_t>(p) & 15) == (reinterpret_cast<std::uintptr_t>(q) & 15) &&
                  (rows == 1 || ps % 4 == qs % 4));
}

template <int MODE, bool SKEWED, int NV>
void launch_norm_nv(const NormArgs& a, const RowShape& s) {
    const unsigned long long ctas = (a.rows + s.rows - 1) / s.rows;
    if (ctas > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm: too many rows");
    // trailing zeros of the last group may reach past the row's 16-byte pieces
    const unsigned smem = MODE != NORM_F32 && SKEWED ? s.rows * (16 + q8_bytes(a.cols)) + 16 : 0;
    norm_kernel<MODE, SKEWED, NV><<<static_cast<unsigned>(ctas), dim3(s.threads, s.rows), smem, stream()>>>(a);
    check_launch("norm_kernel");
}
template <int MODE, bool SKEWED>
void launch_norm_skew(const NormArgs& a) {
    const RowShape s = row_shape(a.cols, SKEWED, a.rows);
    if (s.per <= 1) launch_norm_nv<MODE, SKEWED, 1>(a, s);
    else if (s.per <= 4) launch_norm_nv<MODE, SKEWED, 4>(a, s);
    else launch_norm_nv<MODE, SKEWED, 8>(a, s);
}

template <int MODE>
void launch_norm(const NormArgs& a) {
    const bool alike = same_skew(a.x, a.xs, a.r, a.rs, a.rows) && same_skew(a.x, a.xs, a.h, a.cols, a.rows) &&
                       same_skew(a.x, a.xs, a.y, a.cols, a.rows);
    const bool skewed = a.cols % 4 != 0 || !on_grid(a.x, a.xs, a.rows) || (a.w && !aligned16(a.w));
    if (!fits(a.cols, kNormRegCols, skewed) || !alike) {
        if (a.rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm: too many rows");
        norm_long_kernel<MODE><<<static_cast<unsigned>(a.rows), std::min(1024u, (a.cols + 31) / 32 * 32), 0, stream()>>>(a);
        check_launch("norm_long_kernel");
        return;
    }
    if (skewed) launch_norm_skew<MODE, true>(a);
    else launch_norm_skew<MODE, false>(a);
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

// dh and dw in one launch, for what the ring below does not take: few rows, lengths
// beyond its own, one of the two alone (8192 x 8192: dh 187 us, 5.7 TB/s, dw 92, 5.9).
// The first CTAs write dh: groups of T threads, 1024 / T of them a CTA, have a row
// each, h and t = gy * w in registers. The others add up dw: 32 columns a CTA, a slice
// of at most kDwRows of its rows a warp in float, the slices in double and in order.
// Rows beyond 32 slices go to further CTAs whose sums norm_dw_finish adds.
constexpr unsigned kDwRows = 64;          // float additions in a row of a sum
constexpr unsigned kDwSpan = 32 * kDwRows;  // rows a CTA adds up

struct BothArgs {
    NormBwdArgs n;
    unsigned T, dh_ctas, column_ctas;
    float* dw;  // or partial rows, one for each kDwSpan rows
};

template <bool SKEWED, int NV>
__device__ __forceinline__ void dh_of_rows(const BothArgs& b, double* slots) {
    const NormBwdArgs& a = b.n;
    const unsigned T = b.T, R = 1024 / T, group = threadIdx.x / T, t = threadIdx.x - group * T;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned long long row = static_cast<unsigned long long>(blockIdx.x) * R + group;
    if (row >= a.rows) return;  // a whole group
    const float* hp = a.h + row * a.cols;
    const float* gp = a.gy + row * a.cols;
    const Span span{SKEWED ? skew_of(hp) : 0, a.cols};
    const unsigned G = span.groups();
    const float s = __ldg(a.rstd + row);
    Group h[NV], g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned at = t + i * T;
        h[i] = at < G ? load_group<SKEWED>(hp, at, span) : Group{};
        g[i] = at < G ? load_group<SKEWED>(gp, at, span) : Group{};
    }
    double dot = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned at = t + i * T;
        if (at < G) {
            const Group w = load_weight<SKEWED>(a.w, at, span);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g[i].v[e] *= w.v[e];
                part = fmaf(g[i].v[e], h[i].v[e], part);
            }
            dot += part;
        }
    }
    dot = warp_sum(dot);
    if (T > 32) {  // the group's warps, in order
        if (lane == 0) slots[warp] = dot;
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
        dot = warp_sum(lane < T >> 5 ? slots[group * (T >> 5) + lane] : 0.0);
    }
    const float c = static_cast<float>(dot / a.cols) * (s * s);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned at = t + i * T;
        if (at < G) {
            const Group up = a.gh ? load_group<SKEWED>(a.gh + row * a.cols, at, span) : Group{};
#pragma unroll
            for (int e = 0; e < 4; ++e) g[i].v[e] = fmaf(s, fmaf(-h[i].v[e], c, g[i].v[e]), up.v[e]);
            store_group<SKEWED>(a.dh + row * a.cols, at, g[i], span);
        }
    }
}

__device__ __forceinline__ void dw_of_columns(const BothArgs& b, double (*part)[33]) {
    const NormBwdArgs& a = b.n;
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned at = blockIdx.x - b.dh_ctas, segment = at / b.column_ctas, j = (at - segment * b.column_ctas) * 32 + lane;
    const unsigned long long base = static_cast<unsigned long long>(segment) * kDwSpan;
    const unsigned rows = static_cast<unsigned>(min(static_cast<unsigned long long>(kDwSpan), a.rows - base));
    const unsigned per = (rows + 31) / 32, first = min(rows, warp * per), last = min(rows, first + per);
    float sum = 0.0f;
    if (j < a.cols) {
        const float* gy = a.gy + (base + first) * a.cols + j;
        const float* h = a.h + (base + first) * a.cols + j;
#pragma unroll 8
        for (unsigned i = first; i < last; ++i, gy += a.cols, h += a.cols)
            sum = fmaf(*gy, *h * __ldg(a.rstd + base + i), sum);
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && j < a.cols) {
        double all = 0.0;
        for (unsigned v = 0; v < 32; ++v) all += part[v][lane];
        b.dw[static_cast<unsigned long long>(segment) * a.cols + j] = static_cast<float>(all);
    }
}

template <bool SKEWED, int NV>
__global__ void __launch_bounds__(1024)
norm_bwd_both(const BothArgs b) {
    __shared__ double part[32][33];
    if (blockIdx.x < b.dh_ctas) dh_of_rows<SKEWED, NV>(b, part[0]);
    else dw_of_columns(b, part);
}

// dh for rows too long for registers, or tensors of unlike alignment (8192 x 8192 with
// dw in a launch before it: 409 us).
__global__ void __launch_bounds__(1024)
norm_bwd_dh_long(const NormBwdArgs a) {
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

// dw from `count` partial rows, added in double: 32 columns a CTA, a slice of the
// rows a warp, the slices added in order. Launched while the kernel that writes
// the partial rows still runs (the two-launch axis reduction took 15 us here,
// this takes 4).
__global__ void __launch_bounds__(1024)
norm_dw_finish(const float* __restrict__ partial, unsigned long long count, unsigned cols, float* __restrict__ dw) {
    __shared__ double part[32][33];
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    const unsigned long long per = (count + 31) / 32, first = warp * per, last = min(count, first + per);
    pdl_wait();
    double sum = 0.0;
    if (j < cols) {
#pragma unroll 8
        for (unsigned long long i = first; i < last; ++i) sum += partial[i * cols + j];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && j < cols) {
        sum = 0.0;
        for (unsigned v = 0; v < 32; ++v) sum += part[v][lane];
        dw[j] = static_cast<float>(sum);
    }
}

void launch_dw_finish(const float* partial, unsigned long long count, unsigned cols, float* dw) {
    launch_pdl(norm_dw_finish, dim3((cols + 31) / 32), dim3(1024), 0, stream(), partial, count, cols, dw);
    check_launch("norm_dw_finish");
}

// dh and dw from one pass over h, gy and gh, for rows of up to kRingCols floats, or
// twice as many by pairs of CTAs (below):
// 16 B an element is all that moves. One CTA an SM walks blocks of R rows (R
// groups of T threads). A producer warp bulk-copies the blocks of h and gy into a
// ring of shared-memory stages; gh is loaded a block ahead into registers. A group
// adds up the dot product of its next row before it writes dh of its current one,
// so that the one barrier a row and the sums' latency lie behind work that does
// not depend on them (8192 x 8192 a row at a time: 232 us, so: 189). A thread owns
// the same columns in every row, so dw adds up in its registers; the groups' dw
// meet in shared memory and leave as one partial row a CTA, and the partial rows
// are added in double.
//
// Rows whose length is no multiple of four start off the 16-byte grid, every
// second or fourth of them alike: a CTA takes rows of one such class (`classes`
// apart), copies each from the grid to the grid, and its threads' columns are
// still the same in every row. A warp of its own zeroes the neighbours' columns
// that come with a copy (with every thread looking for them 30000 x 2047 took 347
// us, now 253; with columns by single floats 458, with dh and dw by themselves 327).
//
// HBM bounds the even lengths (8192 x 8192: 5.84 TB/s, 30000 x 2048 in 157 us: 6.3
// TB/s), instructions the odd ones, those at the rows' ends above all.
constexpr unsigned kRingThreads = 512;
constexpr unsigned kRingWarps = kRingThreads / 32;
constexpr unsigned kRingCols = 8192;  // three stages of two rows fit an SM
constexpr unsigned kRingSmem = 3 * 2 * (kRingCols + 4) * sizeof(float);
constexpr unsigned kRingMaxStages = 8;

struct RingArgs {
    NormBwdArgs n;
    unsigned T, R;          // threads a row, rows a block
    unsigned stages;
    unsigned classes;       // 1, 2 or 4; the grid is a multiple of it
    unsigned pitch;         // floats between rows in a stage
    unsigned long long blocks;  // of the largest class
    unsigned segments;      // of kDwRows blocks, the CTA with the most
    float* partial;         // [grid][segments - 1][R][cols], then [grid][cols]
    unsigned* err;
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_addr(dst)),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// Rows of up to twice kRingCols floats: a pair of CTAs has a row, each one half of
// its columns, and every warp tells both CTAs its part of the dot product. Four
// places for them go round: before a warp writes to one again, both CTAs have
// used it. 4000 x 16384 takes 196 us, 5.3 TB/s (dh and dw by themselves 286); 11008
// columns, 2.7 groups a thread, 4.3 TB/s.
struct PairSlots {
    double dot[4][2 * kRingWarps];
    unsigned long long told[4];
};
__device__ __forceinline__ unsigned in_pair(const void* p, unsigned rank) {
    unsigned a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void pair_tell(PairSlots& s, unsigned place, unsigned warp, double v) {
    for (unsigned r = 0; r < 2; ++r) {
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_pair(&s.dot[place][warp], r)), "d"(v) : "memory");
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_pair(&s.told[place], r))
                     : "memory");
    }
}
__device__ __forceinline__ bool pair_wait(unsigned long long* bar, unsigned parity, unsigned* err) {
    for (long long i = 0; i < kWaitPolls / 8; ++i) {
        unsigned ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, "
            "1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(smem_addr(bar)), "r"(parity), "r"(kWaitHintNs)
            : "memory");
        if (ok) return true;
    }
    atomicOr(err, kErrWaitTimeout);
    return false;
}
__device__ __forceinline__ void pair_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool SKEWED, bool PAIRED, int NV>
__global__ void __launch_bounds__(kRingThreads + (SKEWED ? 64 : 32), 1)
norm_bwd_ring(const RingArgs a) {
    static_assert(!(SKEWED && PAIRED), "pairs have whole groups");
    extern __shared__ __align__(128) float ring[];
    __shared__ unsigned long long full[kRingMaxStages], empty[kRingMaxStages], clean[SKEWED ? kRingMaxStages : 1];
    __shared__ double slots[3][kRingWarps];
    __shared__ unsigned dead_flag;
    volatile unsigned* dead = &dead_flag;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ PairSlots pair;  // not in the kernels of single CTAs
    // this CTA's columns of a row, c0 on, and its place among the CTAs or pairs
    const unsigned length = a.n.cols, half = PAIRED ? blockIdx.x & 1 : 0, c0 = half * a.pitch;
    const unsigned cols = PAIRED ? (half ? length - a.pitch : a.pitch) : length;
    const unsigned place = PAIRED ? blockIdx.x >> 1 : blockIdx.x, places = PAIRED ? gridDim.x >> 1 : gridDim.x;
    const unsigned block_floats = a.R * a.pitch;
    const unsigned stage_floats = 2 * block_floats;
    // this CTA's class and its rows' skew, its first block and the step to the next
    const unsigned classes = SKEWED ? a.classes : 1, kind = SKEWED ? place % classes : 0;
    const Span span{SKEWED ? (kind * cols) & 3 : 0, cols};
    const unsigned long long begin = place / classes;
    const unsigned step = places / classes;
    const auto row_at = [&](unsigned long long b, unsigned r) { return (b * a.R + r) * classes + kind; };
    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (unsigned s = 0; s < a.stages; ++s) {
            mbar_init(full + s, 1);
            if (SKEWED) mbar_init(clean + s, 1);
            mbar_init(empty + s, a.R * a.T / 32);
        }
        if (PAIRED)
            for (unsigned s = 0; s < 4; ++s) mbar_init(pair.told + s, 2 * kRingWarps);
        mbar_fence_init();
    }
    __syncthreads();
    if (PAIRED) pair_barrier();

    if (warp == kRingWarps) {  // producer
        unsigned issued = 0;
        for (unsigned long long b = begin; b < a.blocks; b += step, ++issued) {
            const unsigned slot = issued % a.stages, turn = issued / a.stages;
            bool go = true;
            if (turn && lane == 0)
                go = !*dead && mbar_wait_bounded(empty + slot, (turn - 1) & 1, a.err, kWaitPolls / 8);
            if (!__shfl_sync(0xffffffffu, go, 0)) {
                *dead = 1;
                break;
            }
            float* at = ring + slot * stage_floats;
            if constexpr (!SKEWED) {
                const unsigned long long row = b * a.R;
                const unsigned rows = static_cast<unsigned>(min(static_cast<unsigned long long>(a.R), a.n.rows - row));
                const unsigned bytes = rows * cols * sizeof(float);
                if (lane == 0) {
                    mbar_expect_tx(full + slot, 2 * bytes);
                    bulk_copy(at, a.n.h + row * length + c0, bytes, full + slot);
                    bulk_copy(at + block_floats, a.n.gy + row * length + c0, bytes, full + slot);
                }
            } else {  // a row a lane
                const unsigned long long row = row_at(b, lane), first = row * cols;
                const bool have = lane < a.R && row < a.n.rows;
                unsigned floats = have ? 4 * span.groups() : 0;
                float* to = at + lane * a.pitch;
                if (have && row + 1 == a.n.rows) {  // the tensors end with the row
                    floats = (span.skew + cols) & ~3u;
                    for (unsigned i = floats; i < span.skew + cols; ++i) {
                        to[i] = a.n.h[first + i - span.skew];
                        to[block_floats + i] = a.n.gy[first + i - span.skew];
                    }
                }
                const unsigned all = __reduce_add_sync(0xffffffffu, floats);
                __syncwarp();  // lane 0 arrives for the other lanes' stores too
                if (lane == 0) mbar_expect_tx(full + slot, 2 * all * sizeof(float));
                __syncwarp();
                if (have) {
                    bulk_copy(to, a.n.h + (first - span.skew), floats * sizeof(float), full + slot);
                    bulk_copy(to + block_floats, a.n.gy + (first - span.skew), floats * sizeof(float), full + slot);
                }
            }
        }
        // the copies still in flight land before the CTA may finish
        if (lane == 0)
            for (unsigned s = issued > a.stages ? issued - a.stages : 0; s < issued; ++s)
                mbar_wait_bounded(full + s % a.stages, (s / a.stages) & 1, a.err, kWaitPolls / 16);
    } else if (SKEWED && warp > kRingWarps) {
        // Zeros in the place of the neighbours' columns, a row a lane: the others
        // then need no look at where a row begins and ends.
        unsigned i_th = 0;
        for (unsigned long long b = begin; b < a.blocks; b += step, ++i_th) {
            const unsigned slot = i_th % a.stages;
            bool go = true;
            if (lane == 0) go = !*dead && mbar_wait_bounded(full + slot, (i_th / a.stages) & 1, a.err, kWaitPolls / 8);
            if (!__shfl_sync(0xffffffffu, go, 0)) {
                *dead = 1;
                break;
            }
            if (lane < a.R && row_at(b, lane) < a.n.rows) {
                float* row = ring + slot * stage_floats + lane * a.pitch;
                for (unsigned e = 0; e < span.skew; ++e) row[e] = row[block_floats + e] = 0.0f;
                for (unsigned e = span.skew + cols; e < 4 * span.groups(); ++e) row[e] = row[block_floats + e] = 0.0f;
            }
            fence_proxy_async_smem();  // before the slot's next copy
            __syncwarp();
            if (lane == 0) mbar_arrive(clean + slot);
        }
    } else {
        const unsigned group = threadIdx.x / a.T, t = threadIdx.x - group * a.T;
        const unsigned G = span.groups();
        // the weight stays in registers: the ring leaves L1 too little to hold it
        Group dw[NV], w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            dw[i] = Group{};
            w[i] = t + i * a.T < G ? load_weight<SKEWED>(a.n.w + c0, t + i * a.T, span) : Group{};
        }
        // A thread's columns of a partial row, whose own rows are off the grid too.
        const auto put = [&](float* out, unsigned at_c, const Group& v) {
            if (at_c >= G) return;
            if constexpr (!SKEWED) {
                reinterpret_cast<float4*>(out)[at_c] = make_float4(v.v[0], v.v[1], v.v[2], v.v[3]);
            } else {
#pragma unroll
                for (unsigned e = 0; e < 4; ++e)
                    if (span.has(at_c, e)) out[4 * at_c + e - span.skew] = v.v[e];
            }
        };
        unsigned segment = 0;
        const double by_cols = 1.0 / length;
        const auto row_of = [&](unsigned long long b) { return row_at(b, group); };
        Group up[NV];  // gh of the row whose dot product was added up last
        float s_of = 0.0f;  // and its rstd
        // The dot product of block b's row, the i-th of this CTA; dw.
        const auto take = [&](unsigned long long b, unsigned i_th) {
            const unsigned slot = i_th % a.stages;
            const unsigned long long row = row_of(b);
            const bool mine = row < a.n.rows;
            s_of = mine ? __ldg(a.n.rstd + row) : 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const unsigned c = t + i * a.T;
                up[i] = Group{};
                if (mine && a.n.gh && c < G) {
                    const float* gh = a.n.gh + row * length + c0;
                    if (SKEWED && row + 1 == a.n.rows) up[i] = load_group<SKEWED>(gh, c, span);
                    else up[i] = group_of(reinterpret_cast<const float4*>(gh - span.skew)[c]);
                }
            }
            if (!*dead && !mbar_wait_bounded((SKEWED ? clean : full) + slot, (i_th / a.stages) & 1, a.err, kWaitPolls / 8)) *dead = 1;
            const float* at = ring + slot * stage_floats + group * a.pitch;
            double dot = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const unsigned c = t + i * a.T;
                if (mine && c < G) {
                    const Group h = group_of(reinterpret_cast<const float4*>(at)[c]), g = group_of(reinterpret_cast<const float4*>(at + block_floats)[c]);
                    float part = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        dw[i].v[e] = fmaf(g.v[e], h.v[e] * s_of, dw[i].v[e]);
                        part = fmaf(g.v[e] * w[i].v[e], h.v[e], part);
                    }
                    dot += part;
                }
            }
            dot = warp_sum(dot);
            if (lane == 0) {
                if constexpr (PAIRED) pair_tell(pair, i_th & 3, half * kRingWarps + warp, dot);
                else slots[i_th % 3][warp] = dot;
            }
        };
        // dh of block b's row, whose gh and rstd are given.
        const auto give = [&](unsigned long long b, unsigned i_th, const Group (&gh)[NV], float s) {
            const unsigned slot = i_th % a.stages;
            const unsigned long long row = row_of(b);
            double dot;
            if constexpr (PAIRED) {
                if (!*dead && !pair_wait(pair.told + (i_th & 3), (i_th >> 2) & 1, a.err)) *dead = 1;
                dot = warp_sum(pair.dot[i_th & 3][lane]);
            } else {
                dot = warp_sum(lane < a.T >> 5 ? slots[i_th % 3][group * (a.T >> 5) + lane] : 0.0);
            }
            const float c = static_cast<float>(dot * by_cols) * (s * s);
            if (row < a.n.rows) {
                const float* at = ring + slot * stage_floats + group * a.pitch;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const unsigned at_c = t + i * a.T;
                    if (at_c >= G) continue;
                    const Group h = group_of(reinterpret_cast<const float4*>(at)[at_c]), g = group_of(reinterpret_cast<const float4*>(at + block_floats)[at_c]);
                    Group o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.v[e] = fmaf(s, fmaf(-h.v[e], c, g.v[e] * w[i].v[e]), gh[i].v[e]);
                    float* dh = a.n.dh + row * length + c0;
                    if (!SKEWED || (at_c > 0 && at_c < G - 1))
                        __stcs(reinterpret_cast<float4*>(dh - span.skew) + at_c, make_float4(o.v[0], o.v[1], o.v[2], o.v[3]));
                    else
                        put(dh, at_c, o);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + slot);
        };
        unsigned used = 0;
        const bool works = !SKEWED || group < a.R;  // some threads may be over
        if (works && begin < a.blocks) take(begin, 0);
        for (unsigned long long b = begin; works && b < a.blocks; b += step, ++used) {
            Group gh[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) gh[i] = up[i];
            const float s = s_of;
            if ((used + 1) % kDwRows == 0 && segment + 1 < a.segments) {  // enough float additions
                float* out = a.partial + ((static_cast<unsigned long long>(place) * (a.segments - 1) + segment) * a.R + group) * length + c0;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    put(out, t + i * a.T, dw[i]);
                    dw[i] = Group{};
                }
                ++segment;
            }
            if (b + step < a.blocks) take(b + step, used + 1);
            if (PAIRED || a.T == 32) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(a.T) : "memory");
            give(b, used, gh, s);
        }
        for (; works && segment + 1 < a.segments; ++segment) {  // CTAs with fewer blocks
            float* out = a.partial + ((static_cast<unsigned long long>(place) * (a.segments - 1) + segment) * a.R + group) * length + c0;
#pragma unroll
            for (int i = 0; i < NV; ++i) put(out, t + i * a.T, Group{});
        }
        // the groups' rows meet in the ring, which nothing reads any more
        asm volatile("bar.sync 15, %0;" ::"n"(kRingThreads) : "memory");
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (works) put(ring + group * cols, t + i * a.T, dw[i]);
        asm volatile("bar.sync 15, %0;" ::"n"(kRingThreads) : "memory");
        float* out = a.partial + (static_cast<unsigned long long>(places) * (a.segments - 1) * a.R + place) * length + c0;
        for (unsigned c = threadIdx.x; c < cols; c += kRingThreads) {
            float sum = ring[c];
            for (unsigned r = 1; r < a.R; ++r) sum += ring[r * cols + c];
            out[c] = sum;
        }
    }
    if (PAIRED) {
        __syncwarp();
        pair_barrier();  // nobody leaves while its shared memory may be written
    }
}

template <bool SKEWED, bool PAIRED, int NV>
void launch_ring_nv(const RingArgs& a, unsigned ctas, unsigned smem) {
    allow_smem<norm_bwd_ring<SKEWED, PAIRED, NV>, kRingSmem>();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kRingThreads + (SKEWED ? 64 : 32));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIRED ? 2 : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VC_CUDA(cudaLaunchKernelEx(&cfg, norm_bwd_ring<SKEWED, PAIRED, NV>, a));
}
template <bool SKEWED>
void launch_ring(const RingArgs& a, unsigned groups, unsigned ctas, unsigned smem) {
    const unsigned per = (groups + a.T - 1) / a.T;
    if (per <= 1) launch_ring_nv<SKEWED, false, 1>(a, ctas, smem);
    else if (per <= 2) launch_ring_nv<SKEWED, false, 2>(a, ctas, smem);
    else launch_ring_nv<SKEWED, false, 4>(a, ctas, smem);
}

// The fused pass, where it applies; false, having launched nothing, otherwise.
bool try_bwd_ring(const NormBwdArgs& n, float* dw) {
    if (!aligned16(n.h) || !aligned16(n.gy) || !aligned16(n.dh) || (n.gh && !aligned16(n.gh))) return false;
    const bool skewed = n.cols % 4 != 0 || !aligned16(n.w), paired = !skewed && n.cols > kRingCols;
    // groups of a row, or of a CTA's half of it, at most
    const unsigned groups = skewed ? (n.cols + 3 + 3) / 4 : paired ? (n.cols / 4 + 1) / 2 : n.cols / 4;
    // (a row's copy may reach three floats into the next row)
    if (groups > kRingCols / 4 || n.cols < 4) return false;
    RingArgs a{};
    a.n = n;
    // up to four groups a thread; rows of 2^n floats and their neighbours off the
    // grid need one group more, and 3 or 5 rows a block instead of half of 4 or 8
    for (a.R = paired ? 1 : 16; a.R > 1 && 4 * (kRingThreads / a.R / 32 * 32) < groups;) a.R = skewed ? a.R - 1 : a.R / 2;
    a.T = kRingThreads / a.R / 32 * 32;
    a.classes = n.cols % 4 == 0 ? 1 : n.cols % 2 == 0 ? 2 : 4;
    a.pitch = skewed || paired ? 4 * groups : n.cols;
    const unsigned share = a.classes * (paired ? 2 : 1);
    const unsigned step = static_cast<unsigned>(sm_count()) / share, ctas = step * share, places = step * a.classes;
    a.blocks = ((n.rows + a.classes - 1) / a.classes + a.R - 1) / a.R;
    if (a.blocks < 3ull * step) return false;
    const unsigned stage = 2 * a.R * a.pitch * sizeof(float);
    a.stages = std::min(kRingMaxStages, kRingSmem / stage);
    const unsigned long long most = (a.blocks + step - 1) / step;
    a.segments = static_cast<unsigned>((most + kDwRows - 1) / kDwRows);
    const unsigned long long partial_rows = static_cast<unsigned long long>(places) * ((a.segments - 1) * a.R + 1);
    Scratch partial(partial_rows * n.cols * sizeof(float));
    a.partial = partial.as<float>();
    a.err = device_error_word();
    if (paired) launch_ring_nv<false, true, 4>(a, ctas, a.stages * stage);
    else if (skewed) launch_ring<true>(a, groups, ctas, a.stages * stage);
    else launch_ring<false>(a, groups, ctas, a.stages * stage);
    check_launch("norm_bwd_ring");
    launch_dw_finish(a.partial, partial_rows, n.cols, dw);
    return true;
}

void launch_both(const NormBwdArgs& n, float* dw, bool skewed) {
    BothArgs b{};
    b.n = n;
    const unsigned groups = skewed ? (n.cols + 3 + 3) / 4 : n.cols / 4;
    // as many threads a row as there are groups while rows are few, else a
    // quarter; 64 would need a sixteenth named barrier
    const unsigned want = n.rows * groups <= 1024ull * static_cast<unsigned>(sm_count()) ? 1 : 4;
    b.T = 32;
    while (b.T < 1024 && b.T * want < groups) b.T *= b.T == 32 ? 4 : 2;
    const unsigned R = 1024 / b.T, per = (groups + b.T - 1) / b.T;
    const unsigned long long dh_ctas = n.dh ? (n.rows + R - 1) / R : 0;
    const unsigned long long segments = dw ? (n.rows + kDwSpan - 1) / kDwSpan : 0;
    b.column_ctas = (n.cols + 31) / 32;
    const unsigned long long ctas = dh_ctas + segments * b.column_ctas;
    if (ctas > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm_backward: tensor too large");
    b.dh_ctas = static_cast<unsigned>(dh_ctas);
    Scratch partial(segments > 1 ? segments * n.cols * sizeof(float) : 16);
    b.dw = segments > 1 ? partial.as<float>() : dw;
    const auto launch = [&](auto kernel) { kernel<<<static_cast<unsigned>(ctas), 1024, 0, stream()>>>(b); };
    if (skewed && per <= 1) launch(norm_bwd_both<true, 1>);
    else if (skewed) launch(norm_bwd_both<true, 4>);
    else if (per <= 1) launch(norm_bwd_both<false, 1>);
    else launch(norm_bwd_both<false, 4>);
    check_launch("norm_bwd_both");
    if (segments > 1) launch_dw_finish(b.dw, segments, n.cols, dw);
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

// h may be the very tensor it is computed from, where row i of both is the same memory.
void check_in_place(const char* what, const float* h, const float* from, std::size_t stride, std::size_t rows,
                    std::size_t cols) {
    if (h && h == from && stride != cols && rows > 1)
        fail(VC_ERR_INVALID, std::string(what) + ": h can be written over a contiguous tensor only");
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
    check_elements("rms_norm", x, residual, weight, h, y, rstd);
    check_in_place("rms_norm", h, x, x_stride, rows, cols);
    check_in_place("rms_norm", h, residual, residual_stride, rows, cols);
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
    check_elements("rms_norm_q8", x, residual, weight, h, scale);
    check_in_place("rms_norm_q8", h, x, x_stride, rows, cols);
    check_in_place("rms_norm_q8", h, residual, residual_stride, rows, cols);
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
    check_elements("quantize_q8", x, scale);
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
    check_elements("rms_norm_backward", h, weight, rstd, gy, gh, dh, dw);
    if (rows == 0) {  // the sum over no rows
        if (dw) VC_CUDA(cudaMemsetAsync(dw, 0, cols * sizeof(float), stream()));
        return VC_OK;
    }
    if (!h || !weight || !rstd || !gy) fail(VC_ERR_INVALID, "rms_norm_backward: null pointer");
    if (!dh && !dw) return VC_OK;
    if (rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "rms_norm_backward: too many rows");
    NormBwdArgs a{h, weight, rstd, gy, gh, rows, static_cast<unsigned>(cols), dh};
    if (dh && dw && try_bwd_ring(a, dw)) return VC_OK;
    const bool alike = same_skew(h, cols, gy, cols, rows) && same_skew(h, cols, gh, cols, rows) &&
                       same_skew(h, cols, dh, cols, rows);
    const bool skewed = cols % 4 != 0 || !aligned16(h) || !aligned16(weight);
    // dw reads what dh may be written over: then it goes first, in a launch of its own
    const bool over = dh == gy || dh == h, by_itself = dh && (!alike || !fits(a.cols, kNormBwdRegCols, skewed));
    if (dw && dh && (over || by_itself)) {
        a.dh = nullptr;
        launch_both(a, dw, skewed);
        a.dh = dh;
        dw = nullptr;
    }
    if (by_itself) {
        norm_bwd_dh_long<<<static_cast<unsigned>(rows), 1024, 0, stream()>>>(a);
        check_launch("norm_bwd_dh_long");
    } else {
        launch_both(a, dw, skewed);
    }
    VC_API_END
}

}  // extern "C"
