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
// What is left by each filter is the beginning of the order, so the winner of a
// race over more classes than are left is the answer if it is itself left, and
// if not, what is left lies ahead of it. That spares top-p its threshold: the
// winner among all classes is drawn, the mass ahead of it added up, and with
// probability p that is below p of the whole and the row is done; else the race
// is run again among the classes ahead of it. Sums are added in a fixed order
// (up to eight weights in float, then in double), those over lists in whole
// multiples of 2^-40, so nothing depends on scheduling.
//
// Few classes are left by a small k or by min-p, so these are listed on the way
// and the rest of the work is the list's. None of the top k is below the k-th
// largest of the maxima of some 2k groups of threads: the classes from there on
// go to the row's first CTA, which sorts them. The ones that reach min-p stay with
// their CTA, unless they are too many. A large k, or more equal logits than the
// sorted list holds, has its last class found by up to five histograms of the
// order's key, (ordered logit bits, ~index), 11 bits each, and then a list too.
//
// Without top-k and min-p a row is read once from HBM, the sum and the race
// running against the maximum so far, or one at most 2^8 in weight below it;
// with them, once for its maximum and once, from L1 or L2, for the sum and the
// list.
//
// Weights come in two makes. `weight` is the definition in float: one
// subtraction, one division, expf. `quick` is one product and ex2.approx,
// within 2^-15 of it: it serves the sums, and decides whatever it can decide; a
// race within 2^-14, or a class that near min_p, is decided by `weight`. A warp
// passes over 128 classes at once where none of them is left, or comes near the
// warp's leader.
#include "vc_internal.cuh"

#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

namespace vc {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr unsigned kBins = 2048;       // of a histogram
template <unsigned THREADS>
constexpr unsigned kList = THREADS < 512 ? 2048 : 4096;  // classes a CTA lists
constexpr unsigned kSorted = 512;      // classes that are sorted, of the whole cluster
constexpr unsigned kGroups = 512;      // of threads, over the cluster, whose maxima bound the top k
constexpr unsigned kMaxWarps = 16;
constexpr unsigned kIndexBits = 23;    // a key is 32 ordered logit bits, then these of ~index
constexpr std::size_t kMaxVocab = 1u << kIndexBits;
constexpr unsigned kKeyBits = 32 + kIndexBits;
constexpr unsigned kLevelBits = 11;    // of the key a histogram resolves
constexpr unsigned kMaxCluster = 8;
constexpr float kNear = 0x1p-14f;      // quick results this near to each other are decided exactly
constexpr float kGrown = 8.0f;         // log2 by which the maximum of the one pass grows before weights follow it

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
    unsigned chunk;  // classes a CTA of the row's cluster looks at, a multiple of 4
    long long* token;
    float* logprob;
};

constexpr float kLargest = 3.402823466e38f;
// Floats in order as unsigned integers; -0 counts as +0, +inf as the largest.
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(fminf(x, kLargest) + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
constexpr unsigned kIndexMask = (1u << kIndexBits) - 1;
__device__ __forceinline__ u64 key_of(float x, unsigned i) {
    return static_cast<u64>(ordered(x)) << kIndexBits | (kIndexMask - i);
}
__device__ __forceinline__ float key_logit(u64 key) { return from_ordered(static_cast<unsigned>(key >> kIndexBits)); }
__device__ __forceinline__ unsigned key_index(u64 key) { return kIndexMask - (static_cast<unsigned>(key) & kIndexMask); }

__device__ __forceinline__ bool in_play(float x) { return x > -INFINITY; }  // not masked, not NaN


__device__ __forceinline__ float exp2_quick(float z) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaxf(z, -200.0f)));  // NaN is below -200
    return w;
}
__device__ __forceinline__ float quotient_quick(float a, float b) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
    return a * r;
}

// How a row weighs its classes. +inf counts as the largest float, so that no
// difference of two logits in play is NaN. A temperature below the smallest
// normal float counts as that one: log2(e) / T would be infinite, and 0 (the
// maximum's distance) times it NaN.
constexpr float kColdest = 0x1p-126f;
__device__ __forceinline__ float capped(float x) {  // NaN stays
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(kLargest));
    return y;
}
struct Weigh {
    float m, t;
    float to_log2;  // log2(e) / T
    __device__ __forceinline__ void set(float top, float temperature) {
        m = capped(top);
        t = fminf(fmaxf(temperature, kColdest), kLargest);
        to_log2 = static_cast<float>(1.4426950408889634 / static_cast<double>(t));
    }
    __device__ __forceinline__ float distance(float x) const {
        const float d = capped(x) - m;
        return d == 0.0f ? 0.0f : d / t;
    }
    __device__ __forceinline__ float weight(float x) const { return expf(distance(x)); }
    // three roundings of the argument (2^-16 at the smallest weight) and
    // ex2.approx; 0 for a masked class
    __device__ __forceinline__ float quick(float x) const { return exp2_quick((capped(x) - m) * to_log2); }
    __device__ __forceinline__ float4 quick(const float4& v) const {
        return make_float4(quick(v.x), quick(v.y), quick(v.z), quick(v.w));
    }
    // w >= least, w being the quick weight of x
    __device__ __forceinline__ bool reaches(float least, float w, float x) const {
        if (w >= least * (1.0f + kNear)) return true;
        if (w < least * (1.0f - kNear)) return false;
        return weight(x) >= least;
    }
};

struct Shared {
    unsigned count[kBins];
    u64 pick[kSorted];          // in the first CTA, of the whole cluster
    float4 group[kGroups / 4];  // maxima of groups of threads, over the cluster
    float kth;
    u64 warp64[kMaxWarps];
    double warpd[kMaxWarps];
    unsigned listed, picked;
    unsigned first;  // class that has the row's maximum, of this CTA's (~0: none)
    unsigned found_bin, found_in;  // kBins: none
    u64 found_ahead;
    // written by every CTA of the cluster, by its rank
    u64 top[kMaxCluster], best[2][kMaxCluster];
    double total[kMaxCluster], mass[2][kMaxCluster];
    unsigned firsts[kMaxCluster];
    u64 share[kMaxCluster];
};

__device__ __forceinline__ u64 warp_max64(u64 v) {
    for (int m = 16; m > 0; m >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}
__device__ __forceinline__ u64 block_max64(u64 v, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    v = warp_max64(v);
    __syncthreads();
    if (lane == 0) s.warp64[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max64(lane < warps ? s.warp64[lane] : 0);
}
__device__ __forceinline__ double block_sum_d(double v, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) s.warpd[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < warps ? s.warpd[lane] : 0.0);
}
// The sum of v over the threads before this one, and over all.
struct Scan {
    u64 before, all;
};
__device__ __forceinline__ Scan block_scan(u64 v, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    u64 i = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, i, m);
        if (lane >= m) i += o;
    }
    __syncthreads();
    if (lane == 31) s.warp64[warp] = i;
    __syncthreads();
    u64 w = lane < warps ? s.warp64[lane] : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, w, m);
        if (lane >= m) w += o;
    }
    const u64 ahead = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return Scan{i - v + (warp ? ahead : 0), __shfl_sync(0xffffffffu, w, 31)};
}

__device__ __forceinline__ float block_max_f(float v, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    __syncthreads();
    if (lane == 0) s.warp64[threadIdx.x >> 5] = __float_as_uint(v);
    __syncthreads();
    v = lane < warps ? __uint_as_float(static_cast<unsigned>(s.warp64[lane])) : -INFINITY;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// A barrier of the row's CTAs.
__device__ __forceinline__ void row_sync(const cg::cluster_group& cluster) {
    if (cluster.num_blocks() == 1) __syncthreads();
    else cluster.sync();
}

// f(the shared memory of a CTA) for each of the cluster, by the first threads.
template <typename F>
__device__ __forceinline__ void tell_all(const cg::cluster_group& cluster, Shared& s, F&& f) {
    if (threadIdx.x < cluster.num_blocks()) f(*cluster.map_shared_rank(&s, threadIdx.x));
}

// Classes are passed on by fours: v holds those at i .. i + 3, the ones outside
// the range as masked (-inf), 16 bytes a load where the row allows it. A batch
// is DEPTH quads, THREADS of them apart, loaded together, the last one's missing
// quads masked: f(quads, index of the first quad, loose). Whole warps come along,
// in the order of the classes, but for the ends that are off the 16-byte grid:
// these come last, one in the first place of a batch's first quad and `loose`
// true. One place calls f, which is long: with copies of it for whole batches,
// single quads and ends 16 x 50000 with top-p took 21.7 us, so 20.1.
template <unsigned THREADS, int DEPTH, typename F>
__device__ __forceinline__ void each_batch(const float* __restrict__ x, unsigned begin, unsigned end, F&& f) {
    const unsigned t = threadIdx.x;
    const unsigned skew = static_cast<unsigned>((reinterpret_cast<std::uintptr_t>(x + begin) >> 2) & 3);
    const unsigned head = min(end, begin + ((4 - skew) & 3));
    const unsigned groups = (end - head) >> 2;
    const float4* body = reinterpret_cast<const float4*>(x + head);
    // the ends that are off the 16-byte grid, one class a thread of the first warp
    const unsigned tail = head + 4 * groups, ends = t < 32 ? (head - begin) + (end - tail) : 0;
    bool loose = false;
    for (unsigned g = t; !loose; g += DEPTH * THREADS) {
        float4 v[DEPTH];
        unsigned i = head + 4 * g;
        if ((g | 31u) + (DEPTH - 1) * THREADS < groups) {
#pragma unroll
            for (int j = 0; j < DEPTH; ++j) v[j] = body[g + j * THREADS];
        } else {
#pragma unroll
            for (int j = 0; j < DEPTH; ++j) v[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if ((g & ~31u) < groups) {
#pragma unroll
                for (int j = 0; j < DEPTH; ++j)
                    if (g + j * THREADS < groups) v[j] = body[g + j * THREADS];
            } else {
                if (!ends) break;
                loose = true;
                i = t < head - begin ? begin + t : tail + t - (head - begin);
                if (t < ends) v[0].x = x[i];
            }
        }
        f(v, i, loose);
    }
}

// The first quad on the grid of each thread (masked where there is none), and
// its place.
struct First {
    float4 v;
    unsigned i;
    bool there;
};
__device__ __forceinline__ First first_quad(const float* __restrict__ x, unsigned begin, unsigned end) {
    const unsigned skew = static_cast<unsigned>((reinterpret_cast<std::uintptr_t>(x + begin) >> 2) & 3);
    First f;
    f.i = min(end, begin + ((4 - skew) & 3)) + 4 * threadIdx.x;
    f.there = f.i + 3 < end;
    f.v = f.there ? *reinterpret_cast<const float4*>(x + f.i)
                  : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    return f;
}

template <unsigned THREADS, int DEPTH, typename F>
__device__ __forceinline__ void each_quad(const float* x, unsigned begin, unsigned end, F&& f) {
    each_batch<THREADS, DEPTH>(x, begin, end, [&](const auto& v, unsigned i, bool) {
        constexpr int quads = sizeof(v) / sizeof(float4);
#pragma unroll
        for (int j = 0; j < quads; ++j) f(v[j], i + j * 4 * THREADS);
    });
}

__device__ __forceinline__ float largest(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
template <int N>
__device__ __forceinline__ float largest(const float4 (&v)[N]) {
    float m = largest(v[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, largest(v[j]));
    return m;
}
__device__ __forceinline__ float sum4(const float4& w) { return (w.x + w.y) + (w.z + w.w); }
template <int N>
__device__ __forceinline__ float sum_of(const float4 (&w)[N]) {
    float s = sum4(w[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) s += sum4(w[j]);
    return s;
}

// The largest logit a warp has seen, and the first class that has it. Like
// fmaxf it passes over NaN; +inf counts as the largest float.
struct Peak {
    float high{-INFINITY};
    unsigned at{0xffffffffu};
    // a batch from i on, all lanes of a warp together
    template <unsigned THREADS, int N>
    __device__ __forceinline__ void see(const float4 (&v)[N], unsigned i, bool loose) {
        if (loose) {
            take_loose(v[0], i);
        } else if (grows(largest(v))) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (grows(largest(v[j]))) take(v[j], i + j * 4 * THREADS);
        }
    }
    __device__ __forceinline__ bool grows(float most) const { return __any_sync(0xffffffffu, capped(most) > high); }
    __device__ __forceinline__ void take(const float4& v, unsigned i) {
        float top = capped(largest(v));
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
        const auto is = [&](float u) { return capped(u) == top; };
        const unsigned mine = is(v.x) ? i : is(v.y) ? i + 1 : is(v.z) ? i + 2 : is(v.w) ? i + 3 : 0xffffffffu;
        const unsigned first = __reduce_min_sync(0xffffffffu, mine);
        at = top > high ? first : min(at, first);
        high = top;
    }
    // v at i comes out of order: an equal logit may come before the one known
    __device__ __forceinline__ void take_loose(const float4& v, unsigned i) {
        const float old = high;
        const unsigned before = at;
        if (!__any_sync(0xffffffffu, capped(v.x) >= old && in_play(v.x))) return;
        take(v, i);
        if (high == old) at = min(at, before);
    }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
    __syncthreads();
    for (unsigned b = threadIdx.x; b < kBins; b += blockDim.x) s.count[b] = 0;
    __syncthreads();
}

// The definition's score of a class, as a key: the lower index of equal ones.
__device__ __noinline__ u64 exact_score(float x, float e, unsigned i, float m, float t) {
    Weigh wt;
    wt.m = m, wt.t = t;
    const float score = wt.weight(x) / e;
    return score >= 0.0f ? static_cast<u64>(__float_as_uint(score)) << 32 | ~i : 0;
}

// A thread's race so far: its leader and the leader's quick score, and a bound
// below which no class can win, from the leaders of the whole warp. Scores
// within kNear of each other are compared by the definition. Classes whose
// weight underflows (2^-126) and scores that are not above 0 stay out.
struct Race {
    const float* x;
    const float* noise;
    float lead{0.0f}, bound{0x1p-149f};
    unsigned leader{0xffffffffu};
    __device__ __forceinline__ void restart() { lead = 0.0f, bound = 0x1p-149f, leader = 0xffffffffu; }
    __device__ __forceinline__ u64 exact(const Weigh& wt, unsigned i) const {
        return exact_score(x[i], noise[i], i, wt.m, wt.t);
    }
    __device__ __forceinline__ void one(const Weigh& wt, float score, unsigned i) {
        if (!(score >= bound)) return;
        bool ahead = score > lead;
        if (leader != 0xffffffffu && leader != i && !(fabsf(score - lead) >= lead * kNear))
            ahead = exact(wt, i) > exact(wt, leader);
        if (ahead) lead = score, leader = i;
    }
    // a batch's weights and random numbers, all lanes of a warp together
    template <unsigned THREADS, int N>
    __device__ __forceinline__ void run(const Weigh& wt, const float4 (&w)[N], const float4 (&e)[N], unsigned first) {
        float4 score[N];
#pragma unroll
        for (int j = 0; j < N; ++j) score[j] = scores(w[j], e[j]);
        if (!__any_sync(0xffffffffu, largest(score) >= bound)) return;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float high = largest(score[j]);
            if (!(high >= bound)) continue;
            const unsigned i = first + j * 4 * THREADS;
            const float near = high * (1.0f - kNear);
            const bool x1 = score[j].x >= near, y1 = score[j].y >= near, z1 = score[j].z >= near, w1 = score[j].w >= near;
            one(wt, high, x1 ? i : y1 ? i + 1 : z1 ? i + 2 : i + 3);
            if (x1 + y1 + z1 + w1 > 1) {  // the others that are as good
                if (y1) one(wt, score[j].y, i + 1);
                if (z1) one(wt, score[j].z, i + 2);
                if (w1) one(wt, score[j].w, i + 3);
            }
        }
        float most = lead;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
        bound = fmaxf(most * (1.0f - kNear), bound);
    }
    __device__ __forceinline__ float4 scores(const float4& w, const float4& e) const {
        return make_float4(quotient_quick(w.x, e.x), quotient_quick(w.y, e.y), quotient_quick(w.z, e.z),
                           quotient_quick(w.w, e.w));
    }
    // a score that some class of the race reaches
    __device__ __forceinline__ void start_from(float score) { bound = fmaxf(score * (1.0f - kNear), 0x1p-149f); }
    // the maximum that the weights are relative to grew
    __device__ __forceinline__ void rescale(float less) {
        lead *= less;
        bound = fmaxf(bound * less, 0x1p-149f);
    }
    __device__ __forceinline__ u64 best(const Weigh& wt) const { return leader == 0xffffffffu ? 0 : exact(wt, leader); }

    // The random numbers of the classes from i on, as many as there are before
    // `end`, 16 bytes a load where the row allows it.
    __device__ __forceinline__ float4 numbers(unsigned i, unsigned end, bool loose) const {
        float4 e = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (loose) {
            if (i < end) e.x = noise[i];
        } else if (i + 3 < end) {
            if ((reinterpret_cast<std::uintptr_t>(noise + i) & 15) == 0) return *reinterpret_cast<const float4*>(noise + i);
            e = make_float4(noise[i], noise[i + 1], noise[i + 2], noise[i + 3]);
        }
        return e;
    }
};

// The bin in which the cluster's counts, added from bin 0, first reach `target`
// (kBins if they do not), and the count ahead of it; the same in every CTA.
// Each CTA adds up its share of the bins over the cluster, the shares' sums go
// round, and the CTA whose share holds the target tells the others.
struct Found {
    unsigned bin;
    u64 ahead;
    unsigned in_bin;
};
__device__ __noinline__ Found find_bin(Shared& s, u64 target) {
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const unsigned share = kBins / C, per = share >= blockDim.x ? share / blockDim.x : 1;  // per <= 8
    const unsigned first = rank * share + threadIdx.x * per;
    const bool any = threadIdx.x * per < share;
    __syncthreads();
    if (threadIdx.x == 0) s.found_bin = kBins;
    row_sync(cluster);
    unsigned n[8] = {};
    if (any) {
#pragma unroll
        for (unsigned j = 0; j < 8; ++j) {
            if (j >= per) break;
            unsigned c[kMaxCluster];  // in flight together
#pragma unroll
            for (unsigned r = 0; r < kMaxCluster; ++r)
                c[r] = r < C ? cluster.map_shared_rank(&s, r)->count[first + j] : 0;
#pragma unroll
            for (unsigned r = 0; r < kMaxCluster; ++r) n[j] += c[r];
        }
    }
    u64 mine = 0;
#pragma unroll
    for (unsigned j = 0; j < 8; ++j) mine += n[j];
    const Scan scan = block_scan(mine, s);
    u64 c = scan.before;
    if (C > 1) {
        tell_all(cluster, s, [&](Shared& o) { o.share[rank] = scan.all; });
        cluster.sync();
        for (unsigned r = 0; r < rank; ++r) c += s.share[r];
    }
    if (any && c < target && c + mine >= target) {
        unsigned j = 0, in_bin = n[0];
#pragma unroll
        for (unsigned i = 0; i < 7; ++i)
            if (j == i && c + n[i] < target) c += n[i], in_bin = n[i + 1], ++j;
        for (unsigned r = 0; r < C; ++r) {
            Shared* o = cluster.map_shared_rank(&s, r);
            o->found_bin = first + j;
            o->found_ahead = c;
            o->found_in = in_bin;
        }
    }
    row_sync(cluster);
    return Found{s.found_bin, s.found_ahead, s.found_in};
}

// The k-th largest of n numbers, a power of two from 8 to kGroups: each is told its
// place by the threads that compare it with all, as many threads a number as there are.
template <unsigned THREADS>
__device__ __noinline__ float kth_of(Shared& s, const float4* v, unsigned n, unsigned k) {
    unsigned per = 1;
    while (per < 32 && 2 * per * n <= THREADS && 8 * per <= n) per *= 2;
    const unsigned part = threadIdx.x % per;
    for (unsigned base = 0; base < n; base += THREADS / per) {
        const unsigned g = base + threadIdx.x / per;
        const float mine = reinterpret_cast<const float*>(v)[min(g, n - 1)];
        unsigned place = 0;
#pragma unroll 4
        for (unsigned q = part; q < n / 4; q += per) {
            const float4 o = v[q];
            const unsigned i = 4 * q;
            place += (o.x > mine || (o.x == mine && i < g)) + (o.y > mine || (o.y == mine && i + 1 < g)) +
                     (o.z > mine || (o.z == mine && i + 2 < g)) + (o.w > mine || (o.w == mine && i + 3 < g));
        }
        for (unsigned m = 1; m < per; m <<= 1) place += __shfl_xor_sync(0xffffffffu, place, m);
        if (g < n && place == k - 1) s.kth = mine;
    }
    __syncthreads();
    return s.kth;
}

// Groups a warp, so that there are 2k over all warps if there can be.
__device__ __forceinline__ unsigned groups_a_warp(unsigned warps, u64 k) {
    unsigned per = 1;
    while (per < 32 && 2 * per * warps <= kGroups && per * warps < 2 * k) per *= 2;
    return per;
}
// The maximum of the group of lanes, `per` groups a warp.
__device__ __forceinline__ float group_max(float v, unsigned per) {
    for (unsigned m = 1; m < 32 / per; m <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// The n classes of s.pick in order, largest first, in `sorted`, and their random
// numbers: every class counts the ones before it, shared by as many
// threads as there are -- one barrier, where a sorting network of 256 has 36.
template <unsigned THREADS>
__device__ __noinline__ void sort_picks(const Shared& s, unsigned n, const float* noise, u64* sorted, float* numbers) {
    unsigned per = 1;
    while (per < 32 && 2 * per * n <= THREADS) per *= 2;
    const unsigned part = threadIdx.x % per;
    for (unsigned base = 0; base < n; base += THREADS / per) {
        const unsigned c = base + threadIdx.x / per;
        const u64 mine = s.pick[min(c, n - 1)];
        const float e = part == 0 ? noise[key_index(mine)] : 0.0f;
        unsigned place = 0;
#pragma unroll 4
        for (unsigned i = part; i < n; i += per) place += s.pick[i] > mine;
        for (unsigned m = 1; m < per; m <<= 1) place += __shfl_xor_sync(0xffffffffu, place, m);
        if (c < n && part == 0) sorted[place] = mine, numbers[place] = e;
    }
    __syncthreads();
}

// A key that k classes reach and no more; the lowest if no more than k are in play.
template <unsigned THREADS>
__device__ __noinline__ u64 kth_key(Shared& s, const float* x, unsigned begin, unsigned end, u64 k) {
    u64 prefix = 0;
    for (unsigned shift = kKeyBits; shift > 0;) {
        shift -= kLevelBits;
        clear_bins(s);
        each_quad<THREADS, 1>(x, begin, end, [&](const float4& v, unsigned i) {
            const auto tally = [&](float u, unsigned j) {
                if (!in_play(u)) return;
                const u64 key = key_of(u, j);
                if (shift + kLevelBits < kKeyBits && (key >> (shift + kLevelBits)) != prefix) return;
                atomicAdd(&s.count[kBins - 1 - (static_cast<unsigned>(key >> shift) & (kBins - 1))], 1u);
            };
            tally(v.x, i), tally(v.y, i + 1), tally(v.z, i + 2), tally(v.w, i + 3);
        });
        const Found f = find_bin(s, k);
        if (f.bin == kBins) return key_of(-INFINITY, kIndexMask);  // fewer than k classes: all stay
        k -= f.ahead;
        prefix = prefix << kLevelBits | (kBins - 1 - f.bin);
        if (k == f.in_bin) return prefix << shift;  // the bin's classes are the last of the k
    }
    return prefix;
}

// Which classes are ahead of one in the order.
struct Ahead {
    float x;
    unsigned i;
    float over;  // what is above it is ahead of it: nothing of the largest float, which +inf equals
    __device__ __forceinline__ explicit Ahead(u64 key)
        : x(key_logit(key)), i(key_index(key)), over(x < kLargest ? x : INFINITY) {}
    __device__ __forceinline__ bool of(float u, unsigned j) const { return u > over || (u >= x && j < i); }
    // a quad's weights, 0 for the ones that are not
    __device__ __forceinline__ float4 only(const float4& v, unsigned j, const float4& w) const {
        return make_float4(of(v.x, j) ? w.x : 0.0f, of(v.y, j + 1) ? w.y : 0.0f, of(v.z, j + 2) ? w.z : 0.0f,
                           of(v.w, j + 3) ? w.w : 0.0f);
    }
};

template <unsigned THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
sample_kernel(const SampleArgs a) {
    __shared__ Shared s;
    // (logit, index) of the classes that may be left; later the sorted ones' keys, and their numbers
    __shared__ uint2 list[kList<THREADS>];
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const u64 row = blockIdx.x / C;
    const float* x = a.logits + row * a.ls;
    const unsigned t = threadIdx.x;
    const unsigned begin = min(a.vocab, rank * a.chunk), end = min(a.vocab, begin + a.chunk);
    cg::cluster_group::arrival_token begun = cluster.barrier_arrive();

    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const float min_in = a.min_p ? a.min_p[row] : 0.0f;
    const float p_in = a.top_p ? a.top_p[row] : 1.0f;
    // no other class reaches a min-p above 1, or comes before a mass of nothing
    const bool first_only = greedy || min_in > 1.0f || p_in <= 0.0f;
    const float min_p = min_in > 0.0f && !first_only ? min_in : 0.0f;  // 0: off
    const long long k_in = a.top_k && !first_only ? a.top_k[row] : 0;
    const u64 k = k_in > 0 && k_in < a.vocab ? static_cast<u64>(k_in) : 0;  // 0: off
    const bool by_p = p_in < 1.0f && !first_only;
    const bool at_once = !k && min_p == 0.0f;
    Weigh wt;
    wt.set(0.0f, greedy ? 1.0f : temp);

    Race race{x, a.noise + row * a.ns};
    Peak peak;
    double total = 0.0;
    float own_peak = -INFINITY;  // this thread's
    // Races the classes of the row that `joins(quad, index, weights)` leaves a
    // weight. The best of each thread's first classes is known beforehand, so that
    // few of the rest have to be compared one by one.
    const auto race_those = [&](auto&& joins) {
        {
            const First f = first_quad(x, begin, end);
            const float4 e = race.numbers(f.i, end, false);
            float4 w = wt.quick(f.v);
            joins(f.v, f.i, w);
            race.start_from(fmaxf(block_max_f(largest(race.scores(w, e)), s), 0.0f));
        }
        each_batch<THREADS, 2>(x, begin, end, [&](const auto& v, unsigned first, bool loose) {
            constexpr int quads = sizeof(v) / sizeof(float4);
            float4 w[quads], e[quads];
#pragma unroll
            for (int j = 0; j < quads; ++j) e[j] = race.numbers(first + j * 4 * THREADS, end, loose);
#pragma unroll
            for (int j = 0; j < quads; ++j) {
                w[j] = wt.quick(v[j]);
                joins(v[j], first + j * 4 * THREADS, w[j]);
            }
            if (!__any_sync(0xffffffffu, largest(w) > 0.0f)) return;
            race.template run<THREADS>(wt, w, e, first);
        });
    };

    if (at_once) {
        // one pass: the sum and the race relative to the warp's maximum so far
        const First f = first_quad(x, begin, end);
        const float4 e = first_only ? f.v : race.numbers(f.i, end, false);
        wt.m = fmaxf(capped(block_max_f(largest(f.v), s)), -kLargest);  // no class in play is below that
        if (!first_only) race.start_from(fmaxf(block_max_f(largest(race.scores(wt.quick(f.v), e)), s), 0.0f));
        peak.high = wt.m == 0.0f ? -0x1p-149f : from_ordered(ordered(wt.m) - 1);  // what reaches that maximum is of interest
        each_batch<THREADS, 2>(x, begin, end, [&](const auto& v, unsigned first, bool loose) {
            constexpr int quads = sizeof(v) / sizeof(float4);
            float4 w[quads], e[quads];
            if (!first_only)
#pragma unroll
                for (int j = 0; j < quads; ++j) e[j] = race.numbers(first + j * 4 * THREADS, end, loose);
            peak.template see<THREADS>(v, first, loose);
            // The whole warp; not for every new maximum, since each time rounds the
            // sum and the race once more: what was there at first has left the
            // floats' range (2^-126) after 16 times.
            if ((peak.high - wt.m) * wt.to_log2 > kGrown) {
                const float less = exp2_quick((wt.m - peak.high) * wt.to_log2);
                total *= less;
                race.rescale(less);
                wt.m = peak.high;
            }
#pragma unroll
            for (int j = 0; j < quads; ++j) w[j] = wt.quick(v[j]);
            total += sum_of(w);
            if (!first_only) race.template run<THREADS>(wt, w, e, first);
        });
    } else {
        each_batch<THREADS, 4>(x, begin, end,
                               [&](const auto& v, unsigned, bool) { own_peak = fmaxf(own_peak, largest(v)); });
        own_peak = capped(own_peak);
    }
    u64 top = 0;  // (whose index the next pass finds where there is one)
    if (!at_once && in_play(own_peak)) top = key_of(own_peak, 0);
    if (peak.at != 0xffffffffu) top = key_of(peak.high, peak.at);
    top = block_max64(top, s);
    if (t == 0) s.listed = s.picked = 0, s.first = 0xffffffffu;
    cluster.barrier_wait(std::move(begun));  // every CTA has begun: its shared memory may be written
    // the maxima of groups of neighbouring threads, 2k groups if there are as many
    const bool few = k && k <= kSorted / 2;
    const unsigned warps = C * THREADS / 32;  // of the cluster, at most 128
    const unsigned per_warp = groups_a_warp(warps, k), groups = warps * per_warp;
    if (few) {
        const unsigned lanes = 32 / per_warp;
        const float high = group_max(own_peak, per_warp);
        if (t % lanes == 0)
            for (unsigned r = 0; r < C; ++r)
                reinterpret_cast<float*>(cluster.map_shared_rank(&s, r)->group)[(rank * THREADS + t) / lanes] = high;
    }
    tell_all(cluster, s, [&](Shared& o) { o.top[rank] = top; });
    row_sync(cluster);
    for (unsigned r = 0; r < C; ++r) top = max(top, s.top[r]);
    if (top == 0) {  // nothing in play, in any CTA of the cluster
        if (rank == 0 && t == 0) {
            a.token[row] = -1;
            a.logprob[row] = NAN;
        }
        return;
    }
    const float most = key_logit(top);
    if (at_once) total *= exp2_quick((wt.m - most) * wt.to_log2);
    wt.m = most;

    // The classes that may be left are listed: of a small k, from the k-th largest
    // of the groups' maxima on, and by the first CTA; of min-p, the ones that reach
    // it, each CTA its own.
    float cut = -INFINITY;
    if (few && k <= groups) cut = kth_of<THREADS>(s, s.group, groups, static_cast<unsigned>(k));
    const bool picking = in_play(cut), listing = min_p > 0.0f && !k;
    const auto find_first = [&](const float4& v, unsigned i) {
        const unsigned at = v.x >= most ? i : v.y >= most ? i + 1 : v.z >= most ? i + 2 : v.w >= most ? i + 3 : 0xffffffffu;
        if (at != 0xffffffffu) atomicMin(&s.first, at);
    };
    if (listing) {
        bool full = false;
        const float least = min_p * (1.0f - kNear);  // the rest of the decision is the race's
        each_quad<THREADS, 2>(x, begin, end, [&](const float4& v, unsigned i) {
            const float4 w = wt.quick(v);
            total += sum4(w);
            if (!(largest(w) >= least)) return;
            find_first(v, i);
            const bool x1 = w.x >= least, y1 = w.y >= least, z1 = w.z >= least, w1 = w.w >= least;
            const unsigned n = x1 + y1 + z1 + w1;
            unsigned at = full ? kList<THREADS> : atomicAdd(&s.listed, n);
            full = at + n > kList<THREADS>;
            if (full) return;
            if (x1) list[at++] = make_uint2(__float_as_uint(v.x), i);
            if (y1) list[at++] = make_uint2(__float_as_uint(v.y), i + 1);
            if (z1) list[at++] = make_uint2(__float_as_uint(v.z), i + 2);
            if (w1) list[at] = make_uint2(__float_as_uint(v.w), i + 3);
        });
    } else if (!at_once) {
        Shared* one = cluster.map_shared_rank(&s, 0);
        const float from = picking ? cut : most;
        each_quad<THREADS, 2>(x, begin, end, [&](const float4& v, unsigned i) {
            total += sum4(wt.quick(v));
            if (!(largest(v) >= from)) return;
            find_first(v, i);
            if (!picking) return;
            const auto picks = [&](float u, unsigned j) {
                if (u >= cut && in_play(u)) {
                    const unsigned at = atomicAdd(&one->picked, 1u);
                    if (at < kSorted) one->pick[at] = key_of(u, j);
                }
            };
            picks(v.x, i), picks(v.y, i + 1), picks(v.z, i + 2), picks(v.w, i + 3);
        });
    }
    total = block_sum_d(total, s);
    tell_all(cluster, s, [&](Shared& o) {
        o.total[rank] = total;
        o.firsts[rank] = s.first;
    });
    const auto over_cluster = [&](const double* parts) {
        double all = 0.0;
        for (unsigned r = 0; r < C; ++r) all += parts[r];
        return all;
    };
    // Where a row has a class in play its maximum has been found in a pass: its distance
    // is 0 and its weight 1, which reaches any min-p that is still on.
    const auto first_class = [&] {
        unsigned i = at_once ? key_index(top) : s.firsts[0];
        for (unsigned r = 1; r < C && !at_once; ++r) i = min(i, s.firsts[r]);
        return i;
    };
    const auto answer = [&](u64 won) {
        if (rank != 0 || t != 0) return;
        const unsigned token = won == 0 ? first_class() : ~static_cast<unsigned>(won);
        a.token[row] = token;
        a.logprob[row] = wt.distance(x[token]) - logf(static_cast<float>(over_cluster(s.total)));
    };

    if (picking) {
        row_sync(cluster);
        const unsigned picked = cluster.map_shared_rank(&s, 0)->picked;
        if (picked <= kSorted) {
            if (rank != 0) return;
            // the classes in order, `per` a thread: the filters, then the race of the ones left
            constexpr unsigned per = kSorted > THREADS ? kSorted / THREADS : 1;
            u64* sorted = reinterpret_cast<u64*>(list);
            float* numbers = reinterpret_cast<float*>(list + kSorted);
            sort_picks<THREADS>(s, picked, race.noise, sorted, numbers);
            u64 key[per], mass[per], sum = 0, best = 0;
            float w[per];
#pragma unroll
            for (unsigned j = 0; j < per; ++j) {
                const unsigned at = t * per + j;
                key[j] = at < picked && at < k ? sorted[at] : 0;
                w[j] = key[j] ? wt.quick(key_logit(key[j])) : 0.0f;
                mass[j] = __float2ull_rn(w[j] * 0x1p40f);  // whole numbers: exact sums in any order
                sum += mass[j];
            }
            const Scan scan = block_scan(sum, s);
            u64 before = scan.before;
            const double most = static_cast<double>(p_in) * static_cast<double>(scan.all);
#pragma unroll
            for (unsigned j = 0; j < per; ++j) {
                const float v = key_logit(key[j]);
                if (key[j] && (!by_p || static_cast<double>(before) < most) && wt.reaches(min_p, w[j], v))
                    best = max(best, exact_score(v, numbers[t * per + j], key_index(key[j]), wt.m, wt.t));
                before += mass[j];
            }
            answer(block_max64(best, s));
            if (C > 1) cluster.sync();  // the others have left, or read `picked` first
            return;
        }
    }

    unsigned turn = 0;  // of the slots that go round
    const auto mass_of_all = [&](double mine, unsigned turn) {
        mine = block_sum_d(mine, s);
        tell_all(cluster, s, [&](Shared& o) { o.mass[turn & 1][rank] = mine; });
        row_sync(cluster);
        return over_cluster(s.mass[turn & 1]);
    };
    // Whether this CTA has a list of every class that may be left.
    const bool by_list = k ? k <= kList<THREADS> : listing && s.listed <= kList<THREADS>;
    u64 best = 0;
    const auto race_listed = [&](auto&& joins) {
        constexpr unsigned per = kList<THREADS> / THREADS;
        float e[per];
        best = 0;
#pragma unroll
        for (unsigned j = 0; j < per; ++j)
            if (t + j * THREADS < s.listed) e[j] = race.noise[list[t + j * THREADS].y];
#pragma unroll
        for (unsigned j = 0; j < per; ++j) {
            if (t + j * THREADS >= s.listed) break;
            const uint2 c = list[t + j * THREADS];
            const float u = __uint_as_float(c.x);
            if (joins(u, c.y)) best = max(best, exact_score(u, e[j], c.y, wt.m, wt.t));
        }
    };
    double limit = 0.0;
    if (k) {
        const u64 least = kth_key<THREADS>(s, x, begin, end, k);
        double mass = 0.0;
        each_quad<THREADS, 2>(x, begin, end, [&](const float4& v, unsigned i) {
            if (!(largest(v) >= key_logit(least))) return;
            const auto keep = [&](float u, unsigned j) {
                if (!in_play(u) || key_of(u, j) < least) return 0.0f;
                if (by_list) list[atomicAdd(&s.listed, 1u)] = make_uint2(__float_as_uint(u), j);
                return wt.quick(u);
            };
            mass += sum4(make_float4(keep(v.x, i), keep(v.y, i + 1), keep(v.z, i + 2), keep(v.w, i + 3)));
        });
        limit = static_cast<double>(p_in) * mass_of_all(mass, turn++);
        if (by_list) {
            race_listed([&](float u, unsigned) { return wt.reaches(min_p, wt.quick(u), u); });
        } else {
            race_those([&](const float4& v, unsigned i, float4& w) {
                const auto keep = [&](float u, unsigned j, float& w) {
                    if (!in_play(u) || key_of(u, j) < least || !wt.reaches(min_p, w, u)) w = 0.0f;
                };
                keep(v.x, i, w.x), keep(v.y, i + 1, w.y), keep(v.z, i + 2, w.z), keep(v.w, i + 3, w.w);
            });
        }
    } else if (by_list) {
        race_listed([&](float u, unsigned) { return wt.reaches(min_p, wt.quick(u), u); });
    } else if (!at_once) {
        race_those([&](const float4& v, unsigned, float4& w) {
            if (!wt.reaches(min_p, w.x, v.x)) w.x = 0.0f;
            if (!wt.reaches(min_p, w.y, v.y)) w.y = 0.0f;
            if (!wt.reaches(min_p, w.z, v.z)) w.z = 0.0f;
            if (!wt.reaches(min_p, w.w, v.w)) w.w = 0.0f;
        });
    }

    // The winner over the cluster; with top-p, unless the mass ahead of it is
    // below the limit, the race again among the classes ahead of it.
    u64 won;
    for (bool first_turn = true;; first_turn = false) {
        const u64 mine = block_max64(by_list ? best : race.best(wt), s);
        const unsigned slot = turn++ & 1;
        tell_all(cluster, s, [&](Shared& o) { o.best[slot][rank] = mine; });
        row_sync(cluster);
        won = 0;
        for (unsigned r = 0; r < C; ++r) won = max(won, s.best[slot][r]);
        if (!by_p || won == 0) break;
        if (first_turn && !k) limit = static_cast<double>(p_in) * over_cluster(s.total);
        const unsigned i = ~static_cast<unsigned>(won);
        if (i == first_class()) break;  // nothing is ahead of it
        const Ahead ahead(key_of(x[i], i));
        double mass = 0.0;
        if (by_list) {  // what is ahead of it reaches min-p too
            for (unsigned c = t; c < s.listed; c += THREADS) {
                const float u = __uint_as_float(list[c].x);
                // whole multiples of 2^-40: the same sum in any order
                if (ahead.of(u, list[c].y)) mass += static_cast<double>(__float2ull_rn(wt.quick(u) * 0x1p40f)) * 0x1p-40;
            }
        } else {
            each_quad<THREADS, 4>(x, begin, end, [&](const float4& v, unsigned j) {
                if (__any_sync(0xffffffffu, largest(v) >= ahead.x)) mass += sum4(ahead.only(v, j, wt.quick(v)));
            });
        }
        if (mass_of_all(mass, slot) < limit) break;
        if (by_list) {
            race_listed([&](float u, unsigned j) { return ahead.of(u, j); });
        } else {
            race.restart();
            race_those([&](const float4& v, unsigned j, float4& w) { w = ahead.only(v, j, w); });
        }
    }
    answer(won);
}

template <unsigned THREADS>
void launch_rows(const SampleArgs& a, unsigned rows, unsigned C) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * C);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VC_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<THREADS>, a));
    check_launch("sample_kernel");
}

// Up to here four CTAs of 256 threads an SM are faster than two of 512: a row is
// mostly barriers (512 rows of 4000 classes: 21 us against 26; 256 of 128000,
// the other way, 96 against 88).
constexpr bool vocab_fits_four(unsigned vocab) { return vocab <= 16384; }

// Few rows are bound by the latency of their passes and barriers: as many CTAs a
// row, of 512 threads, as leave each an SM of its own and 1600 classes (16 x 8000:
// 11.9 us, with 3200 classes 12.4), or half an SM and 4800 (64 x 128000: 45 us
// against 67 alone on an SM; 140 x 8000 the other way, 19.5 against 16.9). With more
// rows, two CTAs an SM, so that one's passes run through the other's barriers, and
// as many of them a row (which is read more than once where there are filters) as
// keep the rows that run together within 48 MB: beyond that L2 loses a row between
// its passes (256 x 128000: 88 us, with half as many CTAs a row 99).
void launch_sample(SampleArgs& a, std::size_t rows) {
    const u64 sms = static_cast<unsigned>(sm_count());
    const bool filtered = a.top_k || a.top_p || a.min_p;
    unsigned C = 1;
    while (C < kMaxCluster &&
           ((2 * rows * C <= sms && a.vocab / (2 * C) >= 1600) || (rows * C <= sms && a.vocab / (2 * C) >= 4800) ||
            (filtered && rows * C > sms && 2 * sms / C * a.vocab * sizeof(float) > 48ull << 20)))
        C *= 2;
    a.chunk = ((a.vocab + C - 1) / C + 3) / 4 * 4;
    if (rows * C > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "sample: too many rows");
    const unsigned n = static_cast<unsigned>(rows);
    if (rows * C <= sms || !vocab_fits_four(a.vocab)) launch_rows<512>(a, n, C);
    else launch_rows<256>(a, n, C);
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
    if (vocab > kMaxVocab) fail(VC_ERR_OVERFLOW, "sample: more than 2^23 classes");
    if (rows > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "sample: too many rows");
    if (rows == 0) return VC_OK;
    if (!logits || !noise || !token || !logprob) fail(VC_ERR_INVALID, "sample: null pointer");
    check_elements("sample", logits, noise, temperature, top_k, top_p, min_p, token, logprob);
    SampleArgs a{};
    a.logits = logits, a.ls = logits_stride, a.noise = noise, a.ns = noise_stride;
    a.temperature = temperature, a.top_k = reinterpret_cast<const long long*>(top_k);
    a.top_p = top_p, a.min_p = min_p, a.vocab = static_cast<unsigned>(vocab);
    a.token = reinterpret_cast<long long*>(token), a.logprob = logprob;
    launch_sample(a, rows);
    VC_API_END
}

}  // extern "C"
