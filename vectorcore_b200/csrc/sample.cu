// sample.cu -- the next token from a row of logits, with temperature, top-k,
// top-p and min-p, from given exponential random numbers.
//
// With m the row's maximum, d = (l - m) / T and w = e^d, the classes are
// ordered by (logit, then lower index). The race is run over the classes that
// every filter leaves:
//   top-k  the first k in order;
//   top-p  those whose predecessors (within the top k) hold less than p of the
//          top k's mass;
//   min-p  w >= min_p (the most likely class has w = 1);
// and the first class in order always stays. The token is the class with the
// largest w / E, E its exponential random number: that draws class i with
// probability w_i / sum of w over the classes left. Its logprob is
// d - log(sum of w over the whole row): the untruncated distribution's.
//
// A class's place in the order is one 64-bit key, (ordered logit bits, ~index),
// unique in the row, so both thresholds are found exactly by descending its
// bits with histograms: of counts for top-k, of masses for top-p. Masses are
// added as integers (w * 2^40), so their sums do not depend on the order in
// which threads add them.
#include "vc_internal.cuh"

#include <cmath>

namespace vc {
namespace {

using u64 = unsigned long long;

constexpr unsigned kSampleThreads = 1024;
constexpr std::size_t kSampleMaxVocab = 1u << 23;  // masses of 2^40 still add up in 64 bits

struct SampleArgs {
    const float* logits;
    u64 ls;  // elements between rows
    const float* noise;
    u64 ns;
    const float* temperature;
    const long long* top_k;
    const float* top_p;
    const float* min_p;
    unsigned vocab;
    long long* token;
    float* logprob;
};

// Floats in order as unsigned integers; -0 counts as +0.
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 key_of(float x, unsigned i) { return static_cast<u64>(ordered(x)) << 32 | ~i; }

__device__ __forceinline__ u64 block_max_u64(u64 v, u64* scratch) {
    for (int m = 16; m > 0; m >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & 31];
    for (int m = 16; m > 0; m >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

struct Weigh {
    float m, t;
    // equal logits weigh 1 (an infinite maximum too)
    __device__ __forceinline__ float distance(float x) const { return x == m ? 0.0f : (x - m) / t; }
    __device__ __forceinline__ float weight(float x) const { return expf(distance(x)); }
    __device__ __forceinline__ u64 mass(float x) const { return static_cast<u64>(weight(x) * 0x1p40f); }
};

__device__ __forceinline__ bool in_play(float x) { return x > -INFINITY; }  // not masked, not NaN

// The key of the class at which the running sum, in order, of 1 (MASS false)
// or of the masses first reaches `target` >= 1; the sum over all classes is at
// least that.
template <bool MASS>
__device__ u64 descend(const float* x, unsigned vocab, const Weigh& wt, u64 target, u64* hist, u64* shared2) {
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        for (unsigned i = threadIdx.x; i < vocab; i += blockDim.x) {
            const float v = x[i];
            if (!in_play(v)) continue;
            const u64 key = key_of(v, i);
            if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
            atomicAdd(&hist[(key >> shift) & 255], MASS ? wt.mass(v) : 1ull);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 left = target;
            int b = 255;
            while (b > 0 && hist[b] < left) left -= hist[b--];
            shared2[0] = prefix | static_cast<u64>(b) << shift;
            shared2[1] = left;
        }
        __syncthreads();
        prefix = shared2[0];
        target = shared2[1];
    }
    return prefix;
}

__global__ void __launch_bounds__(kSampleThreads)
sample_kernel(const SampleArgs a) {
    __shared__ u64 hist[256];
    __shared__ u64 scratch[32];
    __shared__ u64 shared2[2];
    __shared__ double dscratch[32];
    const u64 row = blockIdx.x;
    const float* x = a.logits + row * a.ls;
    const float* noise = a.noise + row * a.ns;
    const unsigned t = threadIdx.x;

    u64 top = 0;
    for (unsigned i = t; i < a.vocab; i += blockDim.x)
        if (in_play(x[i])) top = max(top, key_of(x[i], i));
    top = block_max_u64(top, scratch);
    if (top == 0) {  // nothing in play
        if (t == 0) {
            a.token[row] = -1;
            a.logprob[row] = NAN;
        }
        return;
    }
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    Weigh wt;
    wt.m = from_ordered(static_cast<unsigned>(top >> 32));
    wt.t = greedy ? 1.0f : temp;
    double total = 0.0;
    for (unsigned i = t; i < a.vocab; i += blockDim.x)
        if (in_play(x[i])) total += wt.weight(x[i]);
    total = block_sum(total, dscratch);

    u64 least = 0;  // keys from here on stay
    const long long k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    if (greedy) {
        least = top;
    } else {
        u64 count = 0;
        for (unsigned i = t; i < a.vocab; i += blockDim.x) count += in_play(x[i]);
        count = static_cast<u64>(block_sum(static_cast<double>(count), dscratch));
        if (k > 0 && static_cast<u64>(k) < count)
            least = descend<false>(x, a.vocab, wt, static_cast<u64>(k), hist, shared2);
        if (p < 1.0f) {
            u64 mass = 0;
            for (unsigned i = t; i < a.vocab; i += blockDim.x)
                if (in_play(x[i]) && key_of(x[i], i) >= least) mass += wt.mass(x[i]);
            for (int m = 16; m > 0; m >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, m);
            __syncthreads();
            if ((t & 31) == 0) scratch[t >> 5] = mass;
            __syncthreads();
            mass = scratch[t & 31];
            for (int m = 16; m > 0; m >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, m);
            const double want = ceil(static_cast<double>(p) * static_cast<double>(mass));
            const u64 target = want >= 1.0 ? min(static_cast<u64>(want), mass) : 1;
            least = max(least, descend<true>(x, a.vocab, wt, target, hist, shared2));
        }
    }
    // the race: the largest w / E, the lower index of equal ones
    u64 best = 0;
    for (unsigned i = t; i < a.vocab; i += blockDim.x) {
        if (!in_play(x[i])) continue;
        const u64 key = key_of(x[i], i);
        const float w = wt.weight(x[i]);
        if (key != top && (key < least || w < min_p)) continue;
        const float score = w / noise[i];
        if (score >= 0.0f) best = max(best, static_cast<u64>(__float_as_uint(score)) << 32 | ~i);
    }
    best = block_max_u64(best, scratch);
    if (t == 0) {
        const unsigned token = ~static_cast<unsigned>(greedy || best == 0 ? top : best);
        a.token[row] = token;
        a.logprob[row] = wt.distance(x[token]) - static_cast<float>(log(total));
    }
}

}  // namespace
}  // namespace vc

using namespace vc;

extern "C" {

vc_status vc_cuda_sample(const float* logits, size_t logits_stride, const float* noise, size_t noise_stride,
                         const float* temperature, const int64_t* top_k, const float* top_p, const float* min_p,
                         size_t rows, size_t vocab, int64_t* token, float* logprob) {
    VC_API_BEGIN
    ensure_init();
    if (vocab == 0) fail(VC_ERR_INVALID, "sample: a row needs at least one class");
    if (vocab > kSampleMaxVocab) fail(VC_ERR_OVERFLOW, "sample: more than 2^23 classes");
    if (rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "sample: too many rows");
    if (rows == 0) return VC_OK;
    if (!logits || !noise || !token || !logprob) fail(VC_ERR_INVALID, "sample: null pointer");
    SampleArgs a{};
    a.logits = logits, a.ls = logits_stride, a.noise = noise, a.ns = noise_stride;
    a.temperature = temperature, a.top_k = reinterpret_cast<const long long*>(top_k);
    a.top_p = top_p, a.min_p = min_p, a.vocab = static_cast<unsigned>(vocab);
    a.token = reinterpret_cast<long long*>(token), a.logprob = logprob;
    sample_kernel<<<static_cast<unsigned>(rows), kSampleThreads, 0, stream()>>>(a);
    check_launch("sample_kernel");
    VC_API_END
}

}  // extern "C"
