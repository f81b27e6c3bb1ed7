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
// Without top-k, top-p and min-p a row is read once: the sum and the race run
// against the maximum so far and are rescaled when it grows. Otherwise it is
// read from HBM for its maximum, and what follows reads it from L1 or L2. A
// class's place in the order is one integer key (ordered logit bits,
// then ~index), unique in the row. No row is sorted: a threshold is found by a
// histogram over 2048 bins of (m - l) / T, 64 a unit, after which the classes
// of the one bin that holds the limit are listed and sorted (a few, in
// practice). Where more classes than the list holds share that bin (equal
// logits, say), the bin is split by the bits of the key until one class is
// left. Two cases need no histogram of the row: a small k, whose classes lie
// in the bins above the k-th largest of the threads' own maxima; and min-p,
// whose classes can be listed directly.
//
// Masses are added as integers (w * 2^32 rounded), so no sum depends on the
// order of the atomics, and the list is sorted, so its order does not matter.
//
// Weights come in two makes. `weight` is the definition in float: one
// subtraction, one division, expf. `quick` is one product and ex2.approx,
// within 2^-15 of it: it serves the row's sum and the masses, and decides
// whatever it can decide; a race within 2^-14, or a class that near min_p, is
// decided by `weight`. A warp looks at scores one by one only where one of its
// classes comes near the warp's leader.
#include "vc_internal.cuh"

#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

namespace vc {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;
using i64 = long long;

constexpr unsigned kBins = 2048;       // of a histogram
constexpr unsigned kCap = 2048;        // classes a CTA lists
constexpr unsigned kSorted = 512;      // classes a sorted list holds, over the cluster
constexpr unsigned kMaxWarps = 32;
constexpr unsigned kIndexBits = 23;    // a key is 32 ordered logit bits, then these of ~index
constexpr std::size_t kMaxVocab = 1u << kIndexBits;
constexpr unsigned kKeyBits = 32 + kIndexBits;
constexpr unsigned kLevelBits = 11;    // of the key a histogram level resolves
constexpr unsigned kMaxCluster = 8;
constexpr float kNear = 0x1p-14f;      // quick results this near to each other are decided exactly
constexpr unsigned kPlainAdds = 32768; // classes whose masses' parts add up in 32 bits

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

// Floats in order as unsigned integers; -0 counts as +0.
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
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

// w * 2^32 rounded to an integer, as high * 2^16 + low with low in +-2^15: the
// integer parts are read off sums with 2^23 and 1.5 * 2^23, which leave no
// room for a fraction.
struct Mass {
    unsigned high;
    int low;
    __device__ __forceinline__ explicit Mass(float w) {
        const float z = w * 65536.0f, a = z + 8388608.0f;
        high = __float_as_uint(a) & 0x7fffffu;
        low = static_cast<int>(__float_as_uint((z - (a - 8388608.0f)) * 65536.0f + 12582912.0f)) - 0x4b400000;
    }
    __device__ __forceinline__ i64 whole() const { return (static_cast<i64>(high) << 16) + low; }
};

// How a row weighs its classes. +inf counts as the largest float, so that no
// difference of two logits in play is NaN.
constexpr float kLargest = 3.402823466e38f;
__device__ __forceinline__ float capped(float x) {  // NaN stays
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(kLargest));
    return y;
}
__device__ __forceinline__ float exp2_quick(float z) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaxf(z, -200.0f)));
    return w;
}
struct Weigh {
    float m, t;
    float to_log2;  // log2(e) / T
    float to_bin;   // 64 / T
    __device__ __forceinline__ void set(float top, float temperature) {
        m = capped(top);
        t = fminf(temperature, kLargest);
        to_log2 = static_cast<float>(1.4426950408889634 / static_cast<double>(t));
        to_bin = fminf(64.0f / t, 1e30f);  // finite: 0 * to_bin is 0
    }
    __device__ __forceinline__ float distance(float x) const {
        const float d = capped(x) - m;
        return d == 0.0f ? 0.0f : d / t;
    }
    __device__ __forceinline__ float weight(float x) const { return expf(distance(x)); }
    // three roundings of the argument (2^-16 at the smallest weight) and
    // ex2.approx; 0 for a masked class (NaN is below -200, like -inf)
    __device__ __forceinline__ float quick(float x) const { return exp2_quick((capped(x) - m) * to_log2); }
    __device__ __forceinline__ float4 quick(const float4& v) const {
        return make_float4(quick(v.x), quick(v.y), quick(v.z), quick(v.w));
    }
    // larger logits never have a larger bin; masked classes have the last
    __device__ __forceinline__ unsigned bin(float x) const {
        const float b = fminf((m - capped(x)) * to_bin, static_cast<float>(kBins - 1)) + 8388608.0f;
        return __float_as_uint(b) & 0x7fffffu;
    }
    // w >= least, w being the quick weight of x
    __device__ __forceinline__ bool reaches(float least, float w, float x) const {
        if (w >= least * (1.0f + kNear)) return true;
        if (w < least * (1.0f - kNear)) return false;
        return weight(x) >= least;
    }
};

struct Found {        // the bin in which a running sum reaches its target
    unsigned bin;     // kBins: it does not
    u64 count;        // of classes, and their mass, in the bins before
    i64 mass;
    u64 in_bin;
};

struct Shared {
    unsigned count[kBins], high[kBins], low[kBins];  // a mass: see bin_mass
    u64 list[kCap];                     // keys
    u64 pick[kSorted], sorted[kSorted];
    u64 warp64[kMaxWarps];
    i64 warp64b[kMaxWarps];
    double warpd[kMaxWarps];
    unsigned listed, picked;
    Found found;
    // written by every CTA of the cluster, by its rank
    u64 top[kMaxCluster], best[kMaxCluster];
    double total[kMaxCluster];
    unsigned in_list[kMaxCluster], in_pick[kMaxCluster];
    u64 slice_count[kMaxCluster];
    i64 slice_mass[kMaxCluster];
    u64 answer[2];
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
// Sums of a and b over the threads before this one, and over all.
struct Scan {
    u64 a, all_a;
    i64 b, all_b;
};
__device__ __forceinline__ Scan block_scan(u64 a, i64 b, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    u64 ia = a;
    i64 ib = b;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const u64 pa = __shfl_up_sync(0xffffffffu, ia, m);
        const i64 pb = __shfl_up_sync(0xffffffffu, ib, m);
        if (lane >= m) ia += pa, ib += pb;
    }
    __syncthreads();
    if (lane == 31) s.warp64[warp] = ia, s.warp64b[warp] = ib;
    __syncthreads();
    u64 wa = lane < warps ? s.warp64[lane] : 0;
    i64 wb = lane < warps ? s.warp64b[lane] : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const u64 pa = __shfl_up_sync(0xffffffffu, wa, m);
        const i64 pb = __shfl_up_sync(0xffffffffu, wb, m);
        if (lane >= m) wa += pa, wb += pb;
    }
    Scan o;
    o.all_a = __shfl_sync(0xffffffffu, wa, 31);
    o.all_b = __shfl_sync(0xffffffffu, wb, 31);
    const u64 pa = __shfl_sync(0xffffffffu, wa, (warp + 31) & 31);
    const i64 pb = __shfl_sync(0xffffffffu, wb, (warp + 31) & 31);
    o.a = ia - a + (warp ? pa : 0);
    o.b = ib - b + (warp ? pb : 0);
    return o;
}

// A barrier of the row's CTAs.
__device__ __forceinline__ void row_sync(const cg::cluster_group& cluster) {
    if (cluster.num_blocks() == 1) __syncthreads();
    else cluster.sync();
}

// f(rank) once for each CTA of the cluster, by the first threads.
template <typename F>
__device__ __forceinline__ void tell_all(const cg::cluster_group& cluster, Shared& s, F&& f) {
    if (threadIdx.x < cluster.num_blocks()) f(*cluster.map_shared_rank(&s, threadIdx.x));
}

// Adding a mass to a bin: its parts by themselves where they cannot overflow
// (`plain`), else the whole with a carry.
__device__ __forceinline__ void add_mass(Shared& s, unsigned bin, float w, bool plain) {
    const Mass q(w);
    if (plain) {
        atomicAdd(&s.high[bin], q.high);
        atomicAdd(&s.low[bin], static_cast<unsigned>(q.low));
    } else {
        const u64 v = static_cast<u64>(q.whole());
        const unsigned low = static_cast<unsigned>(v), old = atomicAdd(&s.low[bin], low);
        const unsigned high = static_cast<unsigned>(v >> 32) + (old + low < old);
        if (high) atomicAdd(&s.high[bin], high);
    }
}
__device__ __forceinline__ i64 bin_mass(unsigned high, unsigned low, bool plain) {
    return plain ? (static_cast<i64>(high) << 16) + static_cast<int>(low)
                 : static_cast<i64>(static_cast<u64>(high) << 32 | low);
}

// Classes are passed on by fours: v holds those at i .. i + 3, the ones outside
// the range as masked (-inf), 16 bytes a load where the row allows it. A batch
// is DEPTH quads, blockDim.x of them apart, loaded together:
// f(quads, index of the first quad, loose). Whole warps come along, in the order
// of the classes, but for the ends that are off the 16-byte grid: these come
// last, one in the first place of a quad and `loose` true.
template <int DEPTH, typename F>
__device__ __forceinline__ void each_batch(const float* __restrict__ x, unsigned begin, unsigned end, F&& f) {
    const unsigned t = threadIdx.x, threads = blockDim.x;
    const unsigned skew = static_cast<unsigned>((reinterpret_cast<std::uintptr_t>(x + begin) >> 2) & 3);
    const unsigned head = min(end, begin + ((4 - skew) & 3));
    const unsigned groups = (end - head) >> 2;
    const float4* body = reinterpret_cast<const float4*>(x + head);
    const float4 masked = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    for (unsigned g = t; (g & ~31u) < groups; g += DEPTH * threads) {
        float4 v[DEPTH];
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) v[j] = g + j * threads < groups ? body[g + j * threads] : masked;
        f(v, head + 4 * g, std::false_type{});
    }
    const unsigned tail = head + 4 * groups, loose = (head - begin) + (end - tail);
    if (t < 32 && loose) {
        const unsigned i = t < head - begin ? begin + t : tail + t - (head - begin);
        float4 v[DEPTH];
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) v[j] = masked;
        if (t < loose) v[0].x = x[i];
        f(v, i, std::true_type{});
    }
}

template <int DEPTH, typename F>
__device__ __forceinline__ void each_quad(const float* x, unsigned begin, unsigned end, F&& f) {
    each_batch<DEPTH>(x, begin, end, [&](const float4 (&v)[DEPTH], unsigned i, auto loose) {
#pragma unroll
        for (int j = 0; j < (decltype(loose)::value ? 1 : DEPTH); ++j) f(v[j], i + j * 4 * blockDim.x, loose);
    });
}

// f(value, index) for each class in play.
template <int DEPTH, typename F>
__device__ __forceinline__ void each_class(const float* x, unsigned begin, unsigned end, F&& f) {
    each_quad<DEPTH>(x, begin, end, [&](const float4& v, unsigned i, auto) {
        if (in_play(v.x)) f(v.x, i);
        if (in_play(v.y)) f(v.y, i + 1);
        if (in_play(v.z)) f(v.z, i + 2);
        if (in_play(v.w)) f(v.w, i + 3);
    });
}

__device__ __forceinline__ float largest(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }

// The largest logit a warp has seen, and the first class that has it. Like
// fmaxf it passes over NaN; +inf counts as the largest float.
struct Peak {
    float high{-INFINITY};
    unsigned at{0xffffffffu};
    // v at i, all lanes of a warp together
    template <typename L>
    __device__ __forceinline__ void see(const float4& v, unsigned i, L) {
        if constexpr (L::value) take_loose(v, i);
        else if (grows(v)) take(v, i);
    }
    __device__ __forceinline__ bool grows(const float4& v) const {
        return __any_sync(0xffffffffu, capped(largest(v)) > high);
    }
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
    __device__ __forceinline__ u64 exact(const Weigh& wt, unsigned i) const {
        return exact_score(x[i], noise[i], i, wt.m, wt.t);
    }
    __device__ __forceinline__ void run(const Weigh& wt, float score, unsigned i) {
        if (!(score >= bound)) return;
        bool ahead = score > lead;
        if (leader != 0xffffffffu && !(fabsf(score - lead) >= lead * kNear)) ahead = exact(wt, i) > exact(wt, leader);
        if (ahead) lead = score, leader = i;
    }
    __device__ __forceinline__ void run(const Weigh& wt, float w, float e, unsigned i) {
        run(wt, __fdividef(w, e), i);
    }
    // all lanes of a warp together
    __device__ __forceinline__ void run(const Weigh& wt, const float4& w, const float4& e, unsigned i) {
        const float4 score =
            make_float4(__fdividef(w.x, e.x), __fdividef(w.y, e.y), __fdividef(w.z, e.z), __fdividef(w.w, e.w));
        if (!__any_sync(0xffffffffu, largest(score) >= bound)) return;
        run(wt, score.x, i), run(wt, score.y, i + 1), run(wt, score.z, i + 2), run(wt, score.w, i + 3);
        float most = lead;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
        bound = fmaxf(most * (1.0f - kNear), 0x1p-149f);
    }
    __device__ __forceinline__ u64 best(const Weigh& wt) const { return leader == 0xffffffffu ? 0 : exact(wt, leader); }

    // The random numbers of a quad's classes with a weight, 16 bytes a load
    // where the row allows it (a loose class has no neighbours).
    __device__ __forceinline__ float4 numbers(const float4& w, unsigned i, bool even) const {
        float4 e = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (even && w.y + w.z + w.w > 0.0f) return *reinterpret_cast<const float4*>(noise + i);
        if (w.x > 0.0f) e.x = noise[i];
        if (w.y > 0.0f) e.y = noise[i + 1];
        if (w.z > 0.0f) e.z = noise[i + 2];
        if (w.w > 0.0f) e.w = noise[i + 3];
        return e;
    }

    // Races the classes of a batch of quads that `joins(quad, index, weights)`
    // leaves a weight: their random numbers are fetched together before any of
    // them is looked at.
    template <int DEPTH, typename J>
    __device__ __forceinline__ void run_batch(const Weigh& wt, const float4 (&v)[DEPTH], unsigned first, J&& joins) {
        float4 w[DEPTH], e[DEPTH];
        const bool even = (reinterpret_cast<std::uintptr_t>(noise + first) & 15) == 0;
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) {
            const unsigned i = first + j * 4 * blockDim.x;
            w[j] = wt.quick(v[j]);
            joins(v[j], i, w[j]);
            e[j] = numbers(w[j], i, even);
        }
#pragma unroll
        for (int j = 0; j < DEPTH; ++j) run(wt, w[j], e[j], first + j * 4 * blockDim.x);
    }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
    __syncthreads();
    for (unsigned b = threadIdx.x; b < kBins; b += blockDim.x) s.count[b] = s.high[b] = s.low[b] = 0;
    __syncthreads();
}

// The least float whose bin is at most b (a warp looks at 32 places at a time):
// comparing with it stands for comparing bins.
__device__ __forceinline__ float bin_end(const Weigh& wt, unsigned b) {
    const unsigned lane = threadIdx.x & 31;
    unsigned low = ordered(-kLargest), high = ordered(wt.m);  // the bin of high is 0
    while (low < high) {
        const unsigned step = (high - low) / 32 + 1;
        const unsigned at = min(low + lane * step, high);
        const unsigned reach = __ballot_sync(0xffffffffu, wt.bin(from_ordered(at)) <= b);
        const unsigned first = reach ? __ffs(reach) - 1 : 32;  // bins fall along the lanes
        if (first == 0) return from_ordered(low);
        high = min(first < 32 ? low + first * step : high, high);
        low = min(low + (first - 1) * step, high) + 1;
    }
    return from_ordered(high);
}

// The bin in which the count (or, by_mass, the mass) of the cluster's
// histograms, added from bin 0, first reaches `target`; the same in every CTA.
// Each CTA adds up its share of the bins over the cluster, the shares' sums go
// round, and the CTA whose share holds the target tells the others. Without
// `masses` the masses are left out.
__device__ __noinline__ Found find_bin(Shared& s, bool by_mass, bool masses, bool plain, u64 target) {
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const unsigned share = kBins / C, per = share >= blockDim.x ? share / blockDim.x : 1;
    const unsigned first = rank * share + threadIdx.x * per;
    const bool any = threadIdx.x * per < share;
    __syncthreads();
    if (threadIdx.x == 0) s.found = Found{kBins, 0, 0, 0};
    row_sync(cluster);
    // every CTA's bins are in flight together: at most 8 of each array a thread
    unsigned n[4] = {};  // per <= 4
    i64 q[4] = {};
    if (any && C == 1) {
#pragma unroll
        for (unsigned j = 0; j < 4; ++j)
            if (j < per) {
                n[j] = s.count[first + j];
                if (masses) q[j] = bin_mass(s.high[first + j], s.low[first + j], plain);
            }
    } else if (any) {
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            if (j >= per) break;
            unsigned c[kMaxCluster], h[kMaxCluster], l[kMaxCluster];
#pragma unroll
            for (unsigned r = 0; r < kMaxCluster; ++r) {
                const Shared* o = cluster.map_shared_rank(&s, r < C ? r : rank);
                c[r] = o->count[first + j];
                h[r] = masses ? o->high[first + j] : 0;
                l[r] = masses ? o->low[first + j] : 0;
            }
#pragma unroll
            for (unsigned r = 0; r < kMaxCluster; ++r)
                if (r < C) n[j] += c[r], q[j] += bin_mass(h[r], l[r], plain);
        }
    }
    const u64 my_n = static_cast<u64>(n[0]) + n[1] + n[2] + n[3];
    const i64 my_q = q[0] + q[1] + q[2] + q[3];
    const Scan in_share = block_scan(my_n, my_q, s);
    u64 c = in_share.a;
    i64 m = in_share.b;
    if (C > 1) {
        tell_all(cluster, s, [&](Shared& o) {
            o.slice_count[rank] = in_share.all_a;
            o.slice_mass[rank] = in_share.all_b;
        });
        cluster.sync();
        for (unsigned r = 0; r < rank; ++r) c += s.slice_count[r], m += s.slice_mass[r];
    }
    const u64 before = by_mass ? static_cast<u64>(m) : c, here = by_mass ? static_cast<u64>(my_q) : my_n;
    if (any && before < target && before + here >= target) {
        unsigned j = 0;
#pragma unroll
        for (unsigned i = 0; i < 3; ++i)
            if (j == i && (by_mass ? static_cast<u64>(m + q[i]) : c + n[i]) < target) c += n[i], m += q[i], ++j;
        const Found f{first + j, c, m, j == 0 ? n[0] : j == 1 ? n[1] : j == 2 ? n[2] : n[3]};
        if (C == 1) s.found = f;
        else
            for (unsigned r = 0; r < C; ++r) cluster.map_shared_rank(&s, r)->found = f;
    }
    row_sync(cluster);
    return s.found;
}

// The classes picked by the CTAs of the cluster (n of them, counts in in_pick),
// in the first CTA's `sorted`, largest first: a warp fetches each CTA's, then
// every class counts the ones before it -- one barrier, where a sorting network
// of 256 has 36.
__device__ __noinline__ void sort_picks(Shared& s, unsigned n) {
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp > 0 && warp < cluster.num_blocks()) {
        unsigned at = 0;
        for (unsigned r = 0; r < warp; ++r) at += s.in_pick[r];
        const Shared* o = cluster.map_shared_rank(&s, warp);
        for (unsigned i = lane; i < s.in_pick[warp]; i += 32) s.pick[at + i] = o->pick[i];
    }
    __syncthreads();
    for (unsigned c = threadIdx.x; c < n; c += blockDim.x) {
        const u64 mine = s.pick[c];
        unsigned place = 0;
#pragma unroll 8
        for (unsigned i = 0; i < n; ++i) place += s.pick[i] > mine;
        s.sorted[place] = mine;
    }
    __syncthreads();
}

template <unsigned THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char shared_bytes[];
    Shared& s = *reinterpret_cast<Shared*>(shared_bytes);
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const u64 row = blockIdx.x / C;
    const float* x = a.logits + row * a.ls;
    const unsigned t = threadIdx.x;
    const unsigned begin = min(a.vocab, rank * a.chunk), end = min(a.vocab, begin + a.chunk);
    const bool plain = a.chunk <= kPlainAdds;
    cg::cluster_group::arrival_token begun = cluster.barrier_arrive();

    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const float min_in = a.min_p && !greedy ? a.min_p[row] : 0.0f;
    const bool first_only = greedy || min_in > 1.0f;  // no other class reaches a min-p above 1
    const float min_p = min_in > 0.0f ? min_in : 0.0f;  // 0: off
    const long long k_in = a.top_k && !first_only ? a.top_k[row] : 0;
    const u64 k = k_in > 0 && k_in < a.vocab ? static_cast<u64>(k_in) : 0;  // 0: off
    const float p_in = a.top_p && !first_only ? a.top_p[row] : 1.0f;
    const bool by_p = p_in < 1.0f;
    const double p = p_in;
    const bool at_once = first_only || (!k && !by_p && min_p == 0.0f);
    Weigh wt;
    wt.set(0.0f, greedy ? 1.0f : temp);

    Race race{x, a.noise + row * a.ns};
    Peak peak;
    double total = 0.0;
    const auto add = [&](const float4& w) { total += (w.x + w.y) + (w.z + w.w); };
    float own_peak = -INFINITY;  // this thread's
    if (at_once) {
        // one pass: the sum and the race relative to the warp's maximum so far
        wt.m = -kLargest;  // no class in play is below it
        each_batch<2>(x, begin, end, [&](const float4 (&v)[2], unsigned first, auto loose) {
            constexpr int quads = decltype(loose)::value ? 1 : 2;
            float4 e[quads];
            const bool even = !decltype(loose)::value && (reinterpret_cast<std::uintptr_t>(race.noise + first) & 15) == 0;
#pragma unroll
            for (int j = 0; j < quads; ++j) {
                const unsigned i = first + j * 4 * THREADS;
                e[j] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                if (first_only) continue;
                if constexpr (decltype(loose)::value) {
                    if (i < end) e[j].x = race.noise[i];
                } else if (i + 3 < end) {  // a quad of the row, not past its last
                    if (even) e[j] = *reinterpret_cast<const float4*>(race.noise + i);
                    else
                        e[j] = make_float4(race.noise[i], race.noise[i + 1], race.noise[i + 2], race.noise[i + 3]);
                }
            }
#pragma unroll
            for (int j = 0; j < quads; ++j) {
                const unsigned i = first + j * 4 * THREADS;
                peak.see(v[j], i, loose);
                if (peak.high > wt.m) {  // the whole warp
                    const float less = exp2_quick((wt.m - peak.high) * wt.to_log2);
                    total *= less;
                    race.lead *= less;
                    race.bound = fmaxf(race.bound * less, 0x1p-149f);
                    wt.m = peak.high;
                }
                const float4 w = wt.quick(v[j]);
                add(w);
                if (!first_only) race.run(wt, w, e[j], i);
            }
        });
    } else {
        each_quad<4>(x, begin, end, [&](const float4& v, unsigned i, auto loose) {
            own_peak = fmaxf(own_peak, largest(v));
            peak.see(v, i, loose);
        });
    }
    const u64 mine = peak.at != 0xffffffffu ? key_of(x[peak.at], peak.at) : 0;
    u64 top = block_max64(mine, s);
    if (t == 0) s.listed = 0;
    cluster.barrier_wait(std::move(begun));  // every CTA has begun: its shared memory may be written
    if (C > 1) {
        tell_all(cluster, s, [&](Shared& o) { o.top[rank] = top; });
        cluster.sync();
        for (unsigned r = 0; r < C; ++r) top = max(top, s.top[r]);
    }
    if (top == 0) {  // nothing in play, in any CTA of the cluster
        if (rank == 0 && t == 0) {
            a.token[row] = -1;
            a.logprob[row] = NAN;
        }
        return;
    }
    if (at_once) {
        const float high = capped(key_logit(top));
        if (peak.at != 0xffffffffu) total *= exp2_quick((wt.m - high) * wt.to_log2);
        else total = 0.0;
    }
    wt.m = capped(key_logit(top));

    u64 least = 0;             // keys from here on are left by the filters before min-p
    bool raced = at_once;      // every class left has been in the race
    unsigned settled = 0;      // classes of the sorted list that are still to be settled (first CTA)
    u64 count_ahead = 0, k_limit = 0;
    i64 mass_ahead = 0;
    double all_mass = 0.0;     // what top-p is a share of; below 0: the sorted classes'

    const auto tally = [&](float v, float w) {
        const unsigned b = wt.bin(v);
        atomicAdd(&s.count[b], 1u);
        if (by_p) add_mass(s, b, w, plain);
    };

    // A small k: the bins of the threads' maxima down to the k-th hold the top k.
    // min-p with top-p: the classes that min-p leaves hold the ones that both do.
    bool listing = false;
    float list_from = -INFINITY;
    if (k && k <= THREADS * C / 4) {
        clear_bins(s);
        if (in_play(own_peak)) atomicAdd(&s.count[wt.bin(own_peak)], 1u);
        const unsigned last_bin = find_bin(s, false, false, plain, k).bin;
        if (last_bin < kBins - 1) {  // the last bin has no lower end
            listing = true;
            list_from = bin_end(wt, last_bin);
        }
    } else {
        listing = !k && by_p && min_p > 0.0f;
    }
    const bool tallying = !raced && !listing && (k || by_p);
    if (tallying) clear_bins(s);

    // The row's sum (four weights in float, then in double), and with it the
    // list, the tally, or the race where nothing but min-p decides who is in it.
    if (listing) {
        const float cut = k ? 0.0f : min_p * (1.0f - kNear);
        each_quad<2>(x, begin, end, [&](const float4& v, unsigned i, auto) {
            const float4 w = wt.quick(v);
            add(w);
            if (!(largest(v) >= list_from) || largest(w) < cut) return;
            const auto lists = [&](float l, float u, unsigned j) {
                if (l >= list_from && u >= cut && in_play(l)) {
                    const unsigned at = atomicAdd(&s.listed, 1u);
                    if (at < kCap) s.list[at] = key_of(l, j);
                }
            };
            lists(v.x, w.x, i), lists(v.y, w.y, i + 1), lists(v.z, w.z, i + 2), lists(v.w, w.w, i + 3);
        });
    } else if (tallying) {
        each_quad<2>(x, begin, end, [&](const float4& v, unsigned, auto) {
            const float4 w = wt.quick(v);
            add(w);
            if (in_play(v.x)) tally(v.x, w.x);
            if (in_play(v.y)) tally(v.y, w.y);
            if (in_play(v.z)) tally(v.z, w.z);
            if (in_play(v.w)) tally(v.w, w.w);
        });
    } else if (!raced) {
        each_batch<2>(x, begin, end, [&](const float4 (&v)[2], unsigned i, auto) {
            race.run_batch(wt, v, i, [&](const float4& l, unsigned, float4& w) {
                add(w);
                if (!wt.reaches(min_p, w.x, l.x)) w.x = 0.0f;
                if (!wt.reaches(min_p, w.y, l.y)) w.y = 0.0f;
                if (!wt.reaches(min_p, w.z, l.z)) w.z = 0.0f;
                if (!wt.reaches(min_p, w.w, l.w)) w.w = 0.0f;
            });
        });
        raced = true;
    }
    total = block_sum_d(total, s);
    tell_all(cluster, s, [&](Shared& o) {
        o.total[rank] = total;
        o.in_list[rank] = s.listed;
    });
    const auto total_of_all = [&] {  // after a barrier of the row's CTAs
        double all = 0.0;
        for (unsigned r = 0; r < C; ++r) all += s.total[r];
        return all;
    };

    if (!raced) {
        row_sync(cluster);
        unsigned n = 0, most = 0;
        if (listing)
            for (unsigned r = 0; r < C; ++r) n += s.in_list[r], most = max(most, s.in_list[r]);
        const bool from_list = listing && most <= kCap;
        double mass_left = total_of_all() * 0x1p32;
        // From here on the classes come from the lists where those are complete,
        // else from the row.
        const auto each_source = [&](auto&& f) {
            if (from_list)
                for (unsigned i = t; i < s.in_list[rank]; i += THREADS) f(key_logit(s.list[i]), key_index(s.list[i]));
            else
                each_class<1>(x, begin, end, f);
        };
        // Collects the picks of all CTAs in order in the first one.
        const auto close_picks = [&](unsigned count) {
            __syncthreads();
            if (C > 1) {
                tell_all(cluster, s, [&](Shared& o) { o.in_pick[rank] = s.picked; });
                cluster.sync();
            }
            if (rank == 0) sort_picks(s, count);
        };
        if (from_list && n <= kSorted) {
            // few enough to be sorted as they are
            if (t < s.in_list[rank]) s.pick[t] = s.list[t];
            if (t == 0) s.picked = s.in_list[rank];
            close_picks(n);
            settled = n;
            k_limit = k;
            all_mass = k ? -1.0 : mass_left;
            raced = true;
        }
        bool counted = tallying;  // the bins hold the source's histogram
        for (int limit = 0; limit < 2 && !raced; ++limit) {
            const bool is_p = limit == 1;
            if (is_p ? !by_p : !k) continue;
            const bool last = is_p || !by_p;
            const double want = ceil(p * mass_left);
            const u64 target = is_p ? (want >= 1.0 ? static_cast<u64>(want) : 1) : k;
            if (!counted) {
                clear_bins(s);
                each_source([&](float v, unsigned) { tally(v, wt.quick(v)); });
                counted = true;
            }
            Found f = find_bin(s, is_p, by_p, plain, target);
            if (f.bin == kBins) continue;  // everything stays
            const unsigned row_bin = f.bin;
            const float bin_from = row_bin < kBins - 1 ? bin_end(wt, row_bin) : -INFINITY;
            const float ahead_from = row_bin > 0 ? bin_end(wt, row_bin - 1) : INFINITY;
            const bool none_ahead = row_bin == 0;
            if (f.in_bin <= kSorted) {
                // sort that bin; in the last search the classes ahead of it race
                if (t == 0) s.picked = 0;
                __syncthreads();
                const bool filtered = least || min_p > 0.0f;
                const auto look = [&](float u, unsigned j, float w) {  // whether it races
                    const bool ahead = !none_ahead && u >= ahead_from;
                    if (!ahead && u >= bin_from && in_play(u)) s.pick[atomicAdd(&s.picked, 1u)] = key_of(u, j);
                    return last && ahead && (!filtered || (key_of(u, j) >= least && wt.reaches(min_p, w, u)));
                };
                if (from_list || !last)
                    each_source([&](float u, unsigned j) {
                        const float w = wt.quick(u);
                        if (look(u, j, w)) race.run(wt, w, race.noise[j], j);
                    });
                else
                    each_batch<2>(x, begin, end, [&](const float4 (&v)[2], unsigned first, auto) {
                        race.run_batch(wt, v, first, [&](const float4& l, unsigned i, float4& w) {
                            if (!look(l.x, i, w.x)) w.x = 0.0f;
                            if (!look(l.y, i + 1, w.y)) w.y = 0.0f;
                            if (!look(l.z, i + 2, w.z)) w.z = 0.0f;
                            if (!look(l.w, i + 3, w.w)) w.w = 0.0f;
                        });
                    });
                close_picks(static_cast<unsigned>(f.in_bin));
                if (last) {
                    // classes that an earlier limit dropped are at the end of the order
                    settled = static_cast<unsigned>(f.in_bin);
                    if (rank == 0)
                        while (settled > 1 && s.sorted[settled - 1] < least) --settled;
                    count_ahead = f.count, mass_ahead = f.mass;
                    k_limit = is_p ? 0 : k;
                    all_mass = mass_left;
                    raced = true;
                } else {
                    if (rank == 0) {
                        const unsigned stay = static_cast<unsigned>(k - f.count);
                        const i64 q = t < stay ? Mass(wt.quick(key_logit(s.sorted[t]))).whole() : 0;
                        const i64 all = block_scan(0, q, s).all_b + f.mass;
                        tell_all(cluster, s, [&](Shared& o) {
                            o.answer[0] = s.sorted[stay - 1];
                            o.answer[1] = static_cast<u64>(all);
                        });
                    }
                    row_sync(cluster);
                    least = s.answer[0];
                    mass_left = static_cast<double>(s.answer[1]);
                }
                continue;
            }
            // too many classes share the bin: split it by the bits of the key
            counted = false;
            u64 prefix = 0, count_before = f.count;
            i64 mass_before = f.mass;
            for (unsigned shift = kKeyBits; shift > 0;) {
                shift -= kLevelBits;
                clear_bins(s);
                each_source([&](float v, unsigned i) {
                    if (wt.bin(v) != row_bin) return;
                    const u64 key = key_of(v, i);
                    if (shift + kLevelBits < kKeyBits && (key >> (shift + kLevelBits)) != prefix) return;
                    const unsigned b = kBins - 1 - (static_cast<unsigned>(key >> shift) & (kBins - 1));
                    atomicAdd(&s.count[b], 1u);
                    if (by_p) add_mass(s, b, wt.quick(v), plain);
                });
                f = find_bin(s, is_p, by_p, plain, target - (is_p ? static_cast<u64>(mass_before) : count_before));
                mass_before += f.mass;
                count_before += f.count;
                prefix = prefix << kLevelBits | (kBins - 1 - f.bin);
            }
            least = max(least, prefix);
            if (!is_p) mass_left = static_cast<double>(mass_before + Mass(wt.quick(key_logit(prefix))).whole());
        }
        if (!raced)
            each_source([&](float v, unsigned i) {
                const float w = wt.quick(v);
                if (key_of(v, i) >= least && wt.reaches(min_p, w, v)) race.run(wt, w, race.noise[i], i);
            });
    }

    if (rank == 0 && settled) {
        // the sorted classes, one a thread: filters, then the race of the ones left
        static_assert(kSorted <= THREADS, "one class a thread");
        const u64 key = t < settled && (!k_limit || count_ahead + t < k_limit) ? s.sorted[t] : 0;
        const float v = key_logit(key), w = key ? wt.quick(v) : 0.0f;
        const float e = key ? race.noise[key_index(key)] : 1.0f;
        const Scan scan = block_scan(0, Mass(w).whole(), s);
        if (all_mass < 0.0) all_mass = static_cast<double>(mass_ahead + scan.all_b);
        const double before = static_cast<double>(mass_ahead + scan.b);
        if (key && (!by_p || before < p * all_mass || key == top) && wt.reaches(min_p, w, v))
            race.run(wt, w, e, key_index(key));
    }
    const u64 best = block_max64(race.best(wt), s);
    if (t == 0) cluster.map_shared_rank(&s, 0)->best[rank] = best;
    row_sync(cluster);
    if (rank == 0 && t == 0) {
        u64 first = 0;
        for (unsigned r = 0; r < C; ++r) first = max(first, s.best[r]);
        const unsigned token = first == 0 ? key_index(top) : ~static_cast<unsigned>(first);
        a.token[row] = token;
        a.logprob[row] = wt.distance(x[token]) - logf(static_cast<float>(total_of_all()));
    }
}

template <unsigned THREADS>
void launch_rows(const SampleArgs& a, unsigned rows, unsigned C) {
    static bool configured = false;
    if (!configured) {
        VC_CUDA(cudaFuncSetAttribute(sample_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     sizeof(Shared)));
        configured = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * C);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(Shared);
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

// Few rows are bound by the latency of their passes: as many CTAs of 1024
// threads a row as leave each an SM of its own and 2048 classes. With more
// rows, two CTAs of 512 threads an SM, so that one's passes run through the
// other's barriers, and as many of them a row as keep the rows that run
// together within 48 MB: beyond that L2 loses a row between its passes.
void launch_sample(SampleArgs& a, std::size_t rows) {
    const u64 sms = static_cast<unsigned>(sm_count());
    unsigned C = 1;
    while (C < kMaxCluster && ((2 * rows * C <= sms && a.vocab / (2 * C) >= 2048) ||
                               (rows > sms && 2 * sms / C * a.vocab * sizeof(float) > 48ull << 20)))
        C *= 2;
    a.chunk = ((a.vocab + C - 1) / C + 3) / 4 * 4;
    if (rows * C > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "sample: too many rows");
    if (rows * C <= sms) launch_rows<1024>(a, static_cast<unsigned>(rows), C);
    else launch_rows<512>(a, static_cast<unsigned>(rows), C);
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
    SampleArgs a{};
    a.logits = logits, a.ls = logits_stride, a.noise = noise, a.ns = noise_stride;
    a.temperature = temperature, a.top_k = reinterpret_cast<const long long*>(top_k);
    a.top_p = top_p, a.min_p = min_p, a.vocab = static_cast<unsigned>(vocab);
    a.token = reinterpret_cast<long long*>(token), a.logprob = logprob;
    launch_sample(a, rows);
    VC_API_END
}

}  // extern "C"
