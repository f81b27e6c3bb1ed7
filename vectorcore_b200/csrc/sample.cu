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
// A row is read from HBM once, for its maximum; what follows reads it from L2.
// A class's place in the order is one integer key (ordered logit bits, then
// ~index), unique in the row. No row is sorted: a threshold is found by a
// histogram over 2048 bins of (m - l) / T, 64 a unit, after which the classes
// of the one bin that holds the limit are listed and sorted (a few, in
// practice). Where more classes than the list holds share that bin (equal
// logits, say), the bin is split by the bits of the key until one class is
// left. Two cases need no histogram of the row: a small k, whose classes lie
// in the bins above the k-th largest of the threads' own maxima; and min-p,
// whose classes can be listed directly.
//
// Masses are added as integers (w * 2^33 rounded), so no sum depends on the
// order of the atomics, and the list is sorted, so its order does not matter.
#include "vc_internal.cuh"

#include <cooperative_groups.h>

#include <cmath>

namespace vc {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr unsigned kThreads = 512;
constexpr unsigned kWarps = kThreads / 32;
constexpr unsigned kBins = 2048;       // of a histogram; kBinsPerThread scan steps a thread
constexpr unsigned kBinsPerThread = kBins / kThreads;
constexpr unsigned kCap = 2048;        // classes a sorted list holds
constexpr unsigned kIndexBits = 23;    // a key is 32 ordered logit bits, then these of ~index
constexpr std::size_t kMaxVocab = 1u << kIndexBits;
constexpr unsigned kKeyBits = 32 + kIndexBits;
constexpr unsigned kLevelBits = 11;    // of the key a histogram level resolves
constexpr unsigned kMaxCluster = 8;

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

// How a row weighs its classes.
struct Weigh {
    float m, t;
    float to_log2;  // log2(e) / T
    float to_bin;   // 64 / T
    __device__ __forceinline__ void set(float top, float temperature) {
        m = top;
        t = fminf(temperature, 3.402823466e38f);
        to_log2 = 1.4426950408889634f / t;
        to_bin = 64.0f / t;
    }
    // equal logits weigh 1 (an infinite maximum too)
    __device__ __forceinline__ float distance(float x) const { return x == m ? 0.0f : (x - m) / t; }
    __device__ __forceinline__ float weight(float x) const { return expf(distance(x)); }
    // for the row's sum and for races not worth running: two more roundings of
    // the argument and ex2.approx (2^-22), 4 operations
    __device__ __forceinline__ float quick(float x) const {
        const float z = (x - m) * to_log2;
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(z));
        return x == m ? 1.0f : w;
    }
    __device__ __forceinline__ u64 mass(float w) const { return __float2ull_rn(w * 0x1p33f); }
    // larger logits never have a larger bin
    __device__ __forceinline__ unsigned bin(float x) const {
        return x == m ? 0u : static_cast<unsigned>(fminf((m - x) * to_bin, static_cast<float>(kBins - 1)));
    }
};

struct Found {        // the bin in which a running sum reaches its target
    unsigned bin;     // kBins: it does not
    u64 count;        // of classes, and their mass, in the bins before
    u64 mass;
    u64 in_bin;
};

struct Shared {
    unsigned count[kBins], lo[kBins], hi[kBins];  // a mass is hi * 2^32 + lo
    u64 list[kCap];
    u64 warp64[kWarps], warp64b[kWarps];
    double warpd[kWarps];
    unsigned listed;
    Found found;
    // this CTA's part, read by the others of the cluster
    u64 top, best;
    double total;
    u64 answer[2];
};

__device__ __forceinline__ u64 warp_max64(u64 v) {
    for (int m = 16; m > 0; m >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}
__device__ __forceinline__ u64 block_max64(u64 v, Shared& s) {
    v = warp_max64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp64[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max64((threadIdx.x & 31) < kWarps ? s.warp64[threadIdx.x & 31] : 0);
}
__device__ __forceinline__ double block_sum_d(double v, Shared& s) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warpd[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum((threadIdx.x & 31) < kWarps ? s.warpd[threadIdx.x & 31] : 0.0);
}
// Sums of a and b over the threads before this one.
__device__ __forceinline__ void block_scan64(u64& a, u64& b, Shared& s) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 ia = a, ib = b;
    for (int m = 1; m < 32; m <<= 1) {
        const u64 pa = __shfl_up_sync(0xffffffffu, ia, m), pb = __shfl_up_sync(0xffffffffu, ib, m);
        if (lane >= m) ia += pa, ib += pb;
    }
    __syncthreads();
    if (lane == 31) s.warp64[warp] = ia, s.warp64b[warp] = ib;
    __syncthreads();
    u64 ba = 0, bb = 0;
    for (unsigned w = 0; w < warp; ++w) ba += s.warp64[w], bb += s.warp64b[w];
    a = ba + ia - a;
    b = bb + ib - b;
}

__device__ __forceinline__ void add_mass(Shared& s, unsigned bin, u64 q) {
    const unsigned low = static_cast<unsigned>(q), old = atomicAdd(&s.lo[bin], low);
    const unsigned high = static_cast<unsigned>(q >> 32) + (old + low < old);
    if (high) atomicAdd(&s.hi[bin], high);
}

// f(value, index) for the classes [begin, end) of a row, 16 bytes a load where
// the row allows it, four loads in flight.
template <typename F>
__device__ __forceinline__ void each_class(const float* __restrict__ x, unsigned begin, unsigned end, F&& f) {
    const unsigned t = threadIdx.x;
    const unsigned skew = static_cast<unsigned>((reinterpret_cast<std::uintptr_t>(x + begin) >> 2) & 3);
    const unsigned head = min(end, begin + ((4 - skew) & 3));
    if (t < head - begin) f(x[begin + t], begin + t);
    const unsigned groups = (end - head) >> 2;
    const float4* body = reinterpret_cast<const float4*>(x + head);
    unsigned g = t;
    for (; g + 3 * kThreads < groups; g += 4 * kThreads) {
        float4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = body[g + j * kThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned i = head + 4 * (g + j * kThreads);
            f(v[j].x, i), f(v[j].y, i + 1), f(v[j].z, i + 2), f(v[j].w, i + 3);
        }
    }
    for (; g < groups; g += kThreads) {
        const float4 v = body[g];
        const unsigned i = head + 4 * g;
        f(v.x, i), f(v.y, i + 1), f(v.z, i + 2), f(v.w, i + 3);
    }
    const unsigned tail = head + 4 * groups;
    if (t < end - tail) f(x[tail + t], tail + t);
}

// A row's race so far: the largest w / E as (score bits, ~index).
struct Race {
    const float* noise;
    u64 best{0};
    __device__ __forceinline__ void run(float w, unsigned i) {
        const float score = w / noise[i];
        if (score >= 0.0f) best = max(best, static_cast<u64>(__float_as_uint(score)) << 32 | ~i);
    }
    // the same, leaving out classes whose quick weight cannot win: it and the
    // quick division are within 2^-18 of the exact ones where w is not tiny,
    // and a tiny one needs no more than to be tried against nothing
    __device__ __forceinline__ void run_quick(const Weigh& wt, float x, unsigned i, float quick, float e) {
        const float about = __fdividef(quick, e);
        const float lead = __uint_as_float(static_cast<unsigned>(best >> 32));
        if (about * 1.00002f >= lead || best == 0) {
            const float score = wt.weight(x) / e;
            if (score >= 0.0f) best = max(best, static_cast<u64>(__float_as_uint(score)) << 32 | ~i);
        }
    }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
    __syncthreads();
    for (unsigned b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
    __syncthreads();
}

// The bin in which the count (or, by_mass, the mass) of the cluster's
// histograms, added from bin 0, first reaches `target`; the same in every CTA.
__device__ Found find_bin(Shared& s, const cg::cluster_group& cluster, bool by_mass, u64 target) {
    cluster.sync();
    if (cluster.block_rank() == 0) {
        const unsigned C = cluster.num_blocks();
        u64 count[kBinsPerThread], mass[kBinsPerThread], all_count = 0, all_mass = 0;
#pragma unroll
        for (unsigned j = 0; j < kBinsPerThread; ++j) {
            const unsigned b = threadIdx.x * kBinsPerThread + j;
            count[j] = mass[j] = 0;
            for (unsigned r = 0; r < C; ++r) {
                const Shared* o = cluster.map_shared_rank(&s, r);
                count[j] += o->count[b];
                mass[j] += static_cast<u64>(o->hi[b]) << 32 | o->lo[b];
            }
            all_count += count[j];
            all_mass += mass[j];
        }
        u64 c = all_count, q = all_mass;
        block_scan64(c, q, s);
        const bool before = by_mass ? q < target : c < target;
        const bool after = by_mass ? q + all_mass >= target : c + all_count >= target;
        if (threadIdx.x == kThreads - 1 && !after)
            for (unsigned r = 0; r < C; ++r) cluster.map_shared_rank(&s, r)->found = Found{kBins, 0, 0, 0};
        if (before && after) {
            unsigned j = 0;
            while ((by_mass ? q + mass[j] : c + count[j]) < target) c += count[j], q += mass[j], ++j;
            const Found f{threadIdx.x * kBinsPerThread + j, c, q, count[j]};
            for (unsigned r = 0; r < C; ++r) cluster.map_shared_rank(&s, r)->found = f;
        }
    }
    cluster.sync();
    return s.found;
}

// How many classes the CTAs of the cluster listed (more than kCap: the lists
// are not complete). Ends with the lists readable by all.
__device__ unsigned listed_in_all(Shared& s, const cg::cluster_group& cluster) {
    cluster.sync();
    unsigned n = 0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) n += cluster.map_shared_rank(&s, r)->listed;
    return n;
}

// The first CTA's list gets the others' classes and is sorted, largest first
// (padded with zeros to a power of two). Returns its n.
__device__ void sort_list(Shared& s, const cg::cluster_group& cluster, unsigned n) {
    unsigned at = s.listed;
    for (unsigned r = 1; r < cluster.num_blocks(); ++r) {
        const Shared* o = cluster.map_shared_rank(&s, r);
        for (unsigned i = threadIdx.x; i < o->listed; i += kThreads) s.list[at + i] = o->list[i];
        at += o->listed;
    }
    unsigned size = 32;
    while (size < n) size <<= 1;
    for (unsigned i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
    for (unsigned k = 2; k <= size; k <<= 1)
        for (unsigned j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (unsigned p = threadIdx.x; p < size / 2; p += kThreads) {
                const unsigned a = 2 * p - (p & (j - 1)), b = a + j;
                const u64 u = s.list[a], v = s.list[b];
                if ((u < v) == ((a & k) == 0)) s.list[a] = v, s.list[b] = u;
            }
        }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const u64 row = blockIdx.x / C;
    const float* x = a.logits + row * a.ls;
    const unsigned t = threadIdx.x;
    const unsigned begin = min(a.vocab, rank * a.chunk), end = min(a.vocab, begin + a.chunk);

    // the maximum, and each thread's own
    u64 mine = 0;
    each_class(x, begin, end, [&](float v, unsigned i) {
        if (in_play(v)) mine = max(mine, key_of(v, i));
    });
    u64 top = block_max64(mine, s);
    if (t == 0) {
        s.top = top;
        s.listed = 0;
    }
    cluster.sync();
    for (unsigned r = 0; r < C; ++r) top = max(top, cluster.map_shared_rank(&s, r)->top);
    if (top == 0) {  // nothing in play, in any CTA of the cluster
        if (rank == 0 && t == 0) {
            a.token[row] = -1;
            a.logprob[row] = NAN;
        }
        cluster.sync();  // the others may still be reading s.top
        return;
    }

    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    Weigh wt;
    wt.set(key_logit(top), greedy ? 1.0f : temp);
    const long long k_in = a.top_k && !greedy ? a.top_k[row] : 0;
    const u64 k = k_in > 0 && k_in < a.vocab ? static_cast<u64>(k_in) : 0;  // 0: off
    const float p_in = a.top_p && !greedy ? a.top_p[row] : 1.0f;
    const bool by_p = p_in < 1.0f;
    const double p = p_in;
    const float min_in = a.min_p && !greedy ? a.min_p[row] : 0.0f;
    const float min_p = min_in > 0.0f ? min_in : 0.0f;  // 0: off

    Race race{a.noise + row * a.ns};
    double total = 0.0;
    u64 least = 0;        // keys from here on are left by the filters before min-p
    bool raced = false;   // every class left has been in the race
    bool summed = false;
    // The row's sum, with what else a pass over the row does with each weight.
    const auto weigh_all = [&](auto&& also) {
        float part = 0.0f;
        unsigned in_part = 0;
        total = 0.0;
        each_class(x, begin, end, [&](float v, unsigned i) {
            const float w = in_play(v) ? wt.quick(v) : 0.0f;
            part += w;
            if (++in_part == 4) {
                total += part;
                part = 0.0f;
                in_part = 0;
            }
            if (in_play(v)) also(v, i, w);
        });
        total += part;
        const double all = block_sum_d(total, s);
        if (t == 0) s.total = all;
        summed = true;
    };
    const auto total_of_all = [&] {  // after a cluster barrier
        double all = 0.0;
        for (unsigned r = 0; r < C; ++r) all += cluster.map_shared_rank(&s, r)->total;
        return all;
    };
    const auto list_class = [&](float v, unsigned i) {
        const unsigned at = atomicAdd(&s.listed, 1u);
        if (at < kCap) s.list[at] = key_of(v, i);
    };
    // Resolves a sorted list (first CTA only) whose classes follow `count`
    // others of mass `mass`: applies the filters, runs the race of those left.
    const auto settle = [&](unsigned n, u64 count, u64 mass, u64 k_limit, bool p_limit, double all_mass) {
        u64 q[kCap / kThreads], sum = 0;
        constexpr unsigned per = kCap / kThreads;
#pragma unroll
        for (unsigned j = 0; j < per; ++j) {
            const unsigned i = t * per + j;
            q[j] = i < n && (!k_limit || count + i < k_limit) ? wt.mass(wt.weight(key_logit(s.list[i]))) : 0;
            sum += q[j];
        }
        u64 before = sum, none = 0;
        block_scan64(before, none, s);
        if (all_mass < 0.0) {  // the top k's own mass
            if (t == kThreads - 1) s.answer[0] = mass + before + sum;
            __syncthreads();
            all_mass = static_cast<double>(s.answer[0]);
        }
        before += mass;
#pragma unroll
        for (unsigned j = 0; j < per; ++j) {
            const unsigned i = t * per + j;
            if (i < n) {
                const u64 key = s.list[i];
                const float w = wt.weight(key_logit(key));
                const bool left = (!k_limit || count + i < k_limit) &&
                                  (!p_limit || static_cast<double>(before) < p * all_mass) && w >= min_p;
                if (left || key == top) race.run(w, key_index(key));
            }
            before += q[j];
        }
    };

    if (greedy) {
        weigh_all([](float, unsigned, float) {});
        raced = true;
    } else if (!k && !by_p) {
        // every class, or the ones above min_p, races
        const float* noise = race.noise;
        weigh_all([&](float v, unsigned i, float w) {
            if (w >= min_p * 0.9999f && (min_p == 0.0f || wt.weight(v) >= min_p || v == wt.m))
                race.run_quick(wt, v, i, w, noise[i]);
        });
        if (min_p > 1.0f && rank == 0 && t == 0) race.run(1.0f, key_index(top));
        raced = true;
    } else {
        // a short cut: list a few classes that hold all that can be left
        bool listing = false;
        unsigned last_bin = kBins;
        float cut = 0.0f;
        if (k && k <= kThreads * C / 4) {
            clear_bins(s);
            if (mine) atomicAdd(&s.count[wt.bin(key_logit(mine))], 1u);
            const Found f = find_bin(s, cluster, false, k);
            listing = f.bin < kBins - 1;  // the last bin has no lower end
            last_bin = f.bin;
        } else if (!k && min_p > 0.0f) {
            listing = true;
            cut = min_p * 0.9999f;
        }
        if (listing) {
            weigh_all([&](float v, unsigned i, float w) {
                if (w >= cut && (last_bin == kBins || wt.bin(v) <= last_bin)) list_class(v, i);
            });
            const unsigned n = listed_in_all(s, cluster);
            if (n <= kCap) {
                if (rank == 0) {
                    sort_list(s, cluster, n);
                    settle(n, 0, 0, k, by_p, k ? -1.0 : total_of_all() * 0x1p33);
                }
                raced = true;
            }
        }
        if (!raced) {
            // the row's histogram, then the limits one after the other
            clear_bins(s);
            const auto tally = [&](float v, unsigned, float) {
                const unsigned b = wt.bin(v);
                atomicAdd(&s.count[b], 1u);
                add_mass(s, b, wt.mass(wt.weight(v)));
            };
            if (!summed)
                weigh_all(tally);
            else
                each_class(x, begin, end, [&](float v, unsigned i) {
                    if (in_play(v)) tally(v, i, 0.0f);
                });
            cluster.sync();
            double mass_left = total_of_all() * 0x1p33;
            bool split = false;  // the bins hold levels of a key
            for (int limit = 0; limit < 2; ++limit) {
                const bool is_p = limit == 1;
                if (is_p ? !by_p : !k) continue;
                const bool last = is_p || !by_p;
                const double want = ceil(p * mass_left);
                u64 target = is_p ? (want >= 1.0 ? static_cast<u64>(want) : 1) : k;
                if (split) {  // tally the row again
                    clear_bins(s);
                    each_class(x, begin, end, [&](float v, unsigned i) {
                        if (in_play(v)) tally(v, i, 0.0f);
                    });
                }
                Found f = find_bin(s, cluster, is_p, target);
                if (f.bin == kBins) continue;  // everything stays
                const unsigned row_bin = f.bin;
                if (f.in_bin <= kCap) {
                    // list that bin; in the last search the classes before it race
                    __syncthreads();
                    if (t == 0) s.listed = 0;
                    __syncthreads();
                    each_class(x, begin, end, [&](float v, unsigned i) {
                        if (!in_play(v)) return;
                        const unsigned b = wt.bin(v);
                        if (b == row_bin) list_class(v, i);
                        else if (last && b < row_bin && key_of(v, i) >= least) {
                            const float w = wt.weight(v);
                            if (w >= min_p || v == wt.m) race.run(w, i);
                        }
                    });
                    const unsigned n = listed_in_all(s, cluster);
                    if (rank == 0) {
                        sort_list(s, cluster, n);
                        if (last) {
                            // classes that an earlier limit dropped are at the end of the order
                            unsigned kept = n;
                            while (kept > 1 && s.list[kept - 1] < least) --kept;
                            settle(kept, f.count, f.mass, is_p ? 0 : k, is_p, mass_left);
                        } else if (t == 0) {
                            const unsigned stay = static_cast<unsigned>(k - f.count);
                            u64 q = f.mass;
                            for (unsigned i = 0; i < stay; ++i) q += wt.mass(wt.weight(key_logit(s.list[i])));
                            for (unsigned r = 0; r < C; ++r) {
                                Shared* o = cluster.map_shared_rank(&s, r);
                                o->answer[0] = s.list[stay - 1];
                                o->answer[1] = q;
                            }
                        }
                    }
                    if (last) {
                        raced = true;
                    } else {
                        cluster.sync();
                        least = s.answer[0];
                        mass_left = static_cast<double>(s.answer[1]);
                    }
                    continue;
                }
                // too many classes share the bin: split it by the bits of the key
                split = true;
                u64 prefix = 0, mass_before = f.mass, count_before = f.count;
                unsigned shift = kKeyBits;
                while (shift > 0) {
                    shift -= kLevelBits;
                    clear_bins(s);
                    each_class(x, begin, end, [&](float v, unsigned i) {
                        if (!in_play(v) || wt.bin(v) != row_bin) return;
                        const u64 key = key_of(v, i);
                        if (shift + kLevelBits < kKeyBits && (key >> (shift + kLevelBits)) != prefix) return;
                        const unsigned b = kBins - 1 - (static_cast<unsigned>(key >> shift) & (kBins - 1));
                        atomicAdd(&s.count[b], 1u);
                        add_mass(s, b, wt.mass(wt.weight(v)));
                    });
                    f = find_bin(s, cluster, is_p, target - (is_p ? mass_before : count_before));
                    mass_before += f.mass;
                    count_before += f.count;
                    prefix = prefix << kLevelBits | (kBins - 1 - f.bin);
                }
                least = max(least, prefix);
                if (!is_p) mass_left = static_cast<double>(mass_before + wt.mass(wt.weight(key_logit(prefix))));
            }
        }
        if (!raced)
            each_class(x, begin, end, [&](float v, unsigned i) {
                if (!in_play(v)) return;
                const u64 key = key_of(v, i);
                const float w = wt.weight(v);
                if (key == top || (key >= least && w >= min_p)) race.run(w, i);
            });
    }

    const u64 best = block_max64(race.best, s);
    if (t == 0) s.best = best;
    cluster.sync();
    if (rank == 0 && t == 0) {
        u64 first = 0;
        for (unsigned r = 0; r < C; ++r) first = max(first, cluster.map_shared_rank(&s, r)->best);
        const unsigned token = greedy || first == 0 ? key_index(top) : ~static_cast<unsigned>(first);
        a.token[row] = token;
        a.logprob[row] = wt.distance(x[token]) - static_cast<float>(log(total_of_all()));
    }
    cluster.sync();  // nobody leaves while its part is read
}

// CTAs a row: enough to fill the GPU when the rows are few (two CTAs an SM, at
// least 2048 classes each), and enough to keep the rows that run together
// within half of L2, since every pass after the first reads them from there.
void launch_sample(SampleArgs& a, std::size_t rows) {
    const u64 slots = 2ull * static_cast<unsigned>(sm_count());
    unsigned C = 1;
    while (C < kMaxCluster && ((rows * C < slots && a.vocab / (2 * C) >= 2048) ||
                               std::min<u64>(rows, slots / C) * a.vocab * sizeof(float) > 64ull << 20))
        C *= 2;
    a.chunk = ((a.vocab + C - 1) / C + 3) / 4 * 4;
    if (rows * C > 0x7fffffffull) fail(VC_ERR_OVERFLOW, "sample: too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * C));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VC_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel, a));
    check_launch("sample_kernel");
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
