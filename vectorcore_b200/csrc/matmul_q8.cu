// matmul_q8.cu -- product of 8-bit rows with a scale for each row of either
// side:
//
//   out[i, j] = (sum over p of a[i, p] * b[j, p]) * (a_scale[i] * b_scale[j]) + bias[j]
//
// The sums are 32-bit integers, so they are exact and do not depend on the
// order of the additions (|a * b| <= 2^14, hence k <= 131071).
//
// A sum is scaled by one float, the product of its two scales. Where that leaves
// the normal floats, though the result need not, the sum and both scales are
// multiplied in double, which holds all of them.
#include "vc_internal.cuh"

namespace vc {
namespace {

constexpr std::size_t kQ8MaxK = 131071;

struct MatmulQ8Args {
    const signed char* a;
    const signed char* b;
    unsigned long long ap, bp;  // bytes between rows
    const float* sa;
    const float* sb;
    const float* bias;  // or null
    float* out;
    unsigned m, n, k;
};

// sum * (sa * sb). The products of a 0 (a row of zeros) are left as they are, those
// of an infinity or a NaN come out the same either way.
__device__ __forceinline__ float scaled(int sum, float sa, float sb) {
    const float s = sa * sb;
    if (!(fabsf(s) >= 0x1p-126f && fabsf(s) < INFINITY) && sa != 0.0f && sb != 0.0f)
        return static_cast<float>(static_cast<double>(sum) * (static_cast<double>(sa) * static_cast<double>(sb)));
    return static_cast<float>(sum) * s;
}
// Any two scales of which this holds have a product that is only rounded.
__device__ __forceinline__ bool is_plain(float s) { return s == 0.0f || (fabsf(s) >= 0x1p-63f && fabsf(s) <= 0x1p63f); }

// ---- few tokens -------------------------------------------------------------------
//
// Up to 8 * NT tokens: the time is the weights' way from HBM, so nothing stands
// between them and the registers. A CTA has 16 weight rows, its eight warps take
// 128-byte pieces of k in turn, 16 bytes a thread and load, and multiply them by
// m16n8k32 products. A product's four groups of k may be any four as long as both
// sides agree, so a thread's 16 consecutive bytes serve as they are; no byte is
// moved between threads. The warps' sums meet in shared memory. 1 x 32000 x 4096
// takes 23 us, 5.7 TB/s (the tensor-core tiles below 30); 1 x 4096 x 4096 5.9.
constexpr unsigned kRowsWarps = 8;
constexpr unsigned kPiece = 128;  // bytes of k a warp takes at a time

__device__ __forceinline__ void mma_s8(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// weights are read once: not kept in L1
__device__ __forceinline__ int4 load_weights(const signed char* p) {
    int4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
// the bytes of a 16-byte group that are below k (`left` of them)
__device__ __forceinline__ int4 keep_bytes(int4 v, int left) {
    const auto word = [&](int w, int at) {
        const int n = left - at;
        return n >= 4 ? w : n <= 0 ? 0 : static_cast<int>(static_cast<unsigned>(w) & ((1u << (8 * n)) - 1));
    };
    return make_int4(word(v.x, 0), word(v.y, 4), word(v.z, 8), word(v.w, 12));
}

template <int NT>
__global__ void __launch_bounds__(kRowsWarps * 32)
matmul_q8_rows(const MatmulQ8Args g) {
    __shared__ int sums[kRowsWarps][16][8 * NT + 1];
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
    const unsigned row0 = blockIdx.x * 16;
    const signed char* w0 = g.b + static_cast<unsigned long long>(min(row0 + r, g.n - 1)) * g.bp + q * 16;
    const signed char* w1 = g.b + static_cast<unsigned long long>(min(row0 + r + 8, g.n - 1)) * g.bp + q * 16;
    const signed char* x[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) x[i] = g.a + static_cast<unsigned long long>(min(r + 8u * i, g.m - 1)) * g.ap + q * 16;
    int acc[NT][4] = {};
    const unsigned whole = g.k / kPiece;
#pragma unroll 2
    for (unsigned piece = warp; piece < whole; piece += kRowsWarps) {
        const unsigned at = piece * kPiece;
        const int4 a0 = load_weights(w0 + at), a1 = load_weights(w1 + at);
        const int4 c0 = load_weights(w0 + at + 64), c1 = load_weights(w1 + at + 64);
        int4 b[NT], d[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            b[i] = __ldg(reinterpret_cast<const int4*>(x[i] + at));
            d[i] = __ldg(reinterpret_cast<const int4*>(x[i] + at + 64));
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            mma_s8(acc[i], a0.x, a1.x, a0.y, a1.y, b[i].x, b[i].y);
            mma_s8(acc[i], a0.z, a1.z, a0.w, a1.w, b[i].z, b[i].w);
            mma_s8(acc[i], c0.x, c1.x, c0.y, c1.y, d[i].x, d[i].y);
            mma_s8(acc[i], c0.z, c1.z, c0.w, c1.w, d[i].z, d[i].w);
        }
    }
    // what is left of k, less than a piece: 64 bytes a warp; a thread's bytes past
    // k are dropped from the tokens, whose products are then zero
    for (unsigned at = whole * kPiece + 64 * warp; at < g.k; at += 64 * kRowsWarps) {
        const int left = static_cast<int>(g.k) - static_cast<int>(at + q * 16);
        const int4 none = make_int4(0, 0, 0, 0);
        const int4 a0 = left > 0 ? load_weights(w0 + at) : none, a1 = left > 0 ? load_weights(w1 + at) : none;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int4 b = left > 0 ? keep_bytes(__ldg(reinterpret_cast<const int4*>(x[i] + at)), left) : none;
            mma_s8(acc[i], a0.x, a1.x, a0.y, a1.y, b.x, b.y);
            mma_s8(acc[i], a0.z, a1.z, a0.w, a1.w, b.z, b.w);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        sums[warp][r][8 * i + 2 * q] = acc[i][0];
        sums[warp][r][8 * i + 2 * q + 1] = acc[i][1];
        sums[warp][r + 8][8 * i + 2 * q] = acc[i][2];
        sums[warp][r + 8][8 * i + 2 * q + 1] = acc[i][3];
    }
    // one output a thread; what scales it is fetched while the sums meet
    static_assert(16 * 8 * NT <= kRowsWarps * 32);
    const unsigned token = threadIdx.x >> 4, row = threadIdx.x & 15;
    const bool mine = token < min(g.m, 8u * NT) && row0 + row < g.n;
    const float sa = mine ? __ldg(g.sa + token) : 0.0f, sb = mine ? __ldg(g.sb + row0 + row) : 0.0f;
    const float bias = mine && g.bias ? __ldg(g.bias + row0 + row) : 0.0f;
    __syncthreads();
    if (!mine) return;
    int sum = 0;
#pragma unroll
    for (unsigned v = 0; v < kRowsWarps; ++v) sum += sums[v][row][token];
    const float p = scaled(sum, sa, sb);
    g.out[static_cast<unsigned long long>(token) * g.n + row0 + row] = g.bias ? p + bias : p;
}

void launch_rows(const MatmulQ8Args& g) {
    const unsigned grid = (g.n + 15) / 16;
    if (g.m <= 8) matmul_q8_rows<1><<<grid, kRowsWarps * 32, 0, stream()>>>(g);
    else matmul_q8_rows<2><<<grid, kRowsWarps * 32, 0, stream()>>>(g);
    check_launch("matmul_q8_rows");
}

// ---- Blackwell tensor cores ------------------------------------------------------
//
// The weights b are the instruction's M side and the tokens a its N side, so a
// tile's accumulators lie in TMEM with one weight row a lane: a warp's store of
// one register is 32 neighbouring outputs of one token, coalesced whatever n's
// alignment, with no trip through shared memory. A warp of a CTA fetches
// 128-byte slices of k of both sides by TMA (128-byte swizzle, zeros past the
// ends, so k, m and n need no alignment), one thread of another issues the
// products (32 bytes of k each), and eight warps scale and store.

constexpr unsigned kTileM = 128;   // weight rows a CTA's tile: TMEM's lanes
constexpr unsigned kSliceK = 128;  // bytes of k a stage: one swizzled row
constexpr unsigned kMmaK = 32;     // bytes of k an instruction
constexpr unsigned kStoreWarps = 8;  // two for each quarter of TMEM's lanes
constexpr unsigned kTcThreads = (kStoreWarps + 2) * 32;

struct TcArgs {
    const float* sa;
    const float* sb;
    const float* bias;
    float* out;
    unsigned m, n;
    unsigned bn;          // tokens a tile, a multiple of 16
    unsigned rows;        // weight rows a CTA's tile, at most kTileM, a multiple of 8
    unsigned steps;       // along k: stages a tile takes
    unsigned tiles_m;     // along the tokens
    unsigned tiles_n;     // along the weights
    unsigned stages;
    unsigned tmem_cols;   // allocated
    unsigned idesc;
    unsigned* err;
};

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_addr(dst)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}

// Shared-memory descriptor of a K-major tile of 128-byte rows in the 128-byte
// swizzle: groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ unsigned long long tile_desc(unsigned addr) {
    return static_cast<unsigned long long>((addr & 0x3ffffu) >> 4) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}

__device__ __forceinline__ void mma_i8(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc,
                                       bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<unsigned>(accumulate))
        : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_load16(unsigned taddr, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ int tmem_load1(unsigned taddr) {
    int v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
                 : "=r"(v)
                 : "r"(taddr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A bounded wait that also ends when another role of the CTA gave up. The
// issuing thread polls without the other kernels' hint to sleep in a poll: waking
// up cost it 3% of the whole product. The others sleep, which leaves the power
// (the limit of a long run) to the products.
constexpr long long kTcPolls = 1ll << 18;  // of up to kWaitHintNs
template <bool SLEEP = true>
__device__ __forceinline__ bool tc_wait(unsigned long long* bar, unsigned parity, volatile unsigned* dead,
                                        unsigned* err) {
    for (long long i = 0; i < (SLEEP ? kTcPolls : kTcPolls << 4); ++i) {
        if constexpr (SLEEP) {
            if (mbar_try_wait(bar, parity)) return true;
        } else {
            unsigned ok;
            asm volatile(
                "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                : "=r"(ok)
                : "r"(smem_addr(bar)), "r"(parity)
                : "memory");
            if (ok) return true;
        }
        if (*dead) return false;
    }
    *dead = 1;
    atomicOr(err, kErrWaitTimeout);
    return false;
}

// A place in the ring of stages, and the parity of its current turn.
struct Place {
    unsigned slot{0}, parity{0};
    __device__ __forceinline__ void next(unsigned stages) {
        if (++slot == stages) slot = 0, parity ^= 1;
    }
};

// The copies still in flight land before their CTA may finish.
__device__ __forceinline__ void drain(unsigned long long* full, unsigned issued, const TcArgs& g) {
    for (unsigned s = issued > g.stages ? issued - g.stages : 0; s < issued; ++s)
        mbar_wait_bounded(full + s % g.stages, (s / g.stages) & 1, g.err, kTcPolls);
}

// Tiles in order: runs of kGroup tiles along the weights for each tile of
// tokens, so the CTAs that run together share both sides in L2.
__device__ __forceinline__ void tile_at(unsigned i, const TcArgs& g, unsigned& tn, unsigned& tm) {
    constexpr unsigned kGroup = 16;
    const unsigned band = i / (kGroup * g.tiles_m), in = i - band * kGroup * g.tiles_m;
    const unsigned width = min(kGroup, g.tiles_n - band * kGroup);
    tm = in / width;
    tn = band * kGroup + in - tm * width;
}

// What a store thread needs beside the sums of its weight row, loaded while the
// sums are on their way: they come from HBM, and fetched after them, with the other
// CTAs' sums one after another, 256 x 4096 x 4096 took 15.8 us, so 13.0. The tokens'
// scales are looked at then too, and read later, from L1.
struct RowScale {
    bool mine;
    float scale, bias;
};
__device__ __forceinline__ RowScale row_scale(const TcArgs& g, unsigned first) {
    const unsigned lane = threadIdx.x & 31, col = first + lane;
    RowScale r{col < g.n && (threadIdx.x >> 5 & 3) * 32 + lane < g.rows, 1.0f, 0.0f};
    if (r.mine) r.scale = __ldg(g.sb + col);
    if (r.mine && g.bias) r.bias = __ldg(g.bias + col);
    return r;
}
// Whether all products of the warp's scales and the tile's tokens' are only rounded:
// of all tokens, alike for both warps of a quarter of the lanes, or of those that the
// warp itself stores (ALL false). (Looked at one by one
// they cost more than the scaling itself: 2048 x 4096 x 1024 25 us, so 17.)
template <bool ALL>
__device__ __forceinline__ bool plain_scales(const TcArgs& g, const RowScale& r, unsigned row0) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool plain = is_plain(r.scale);
#pragma unroll
    for (unsigned q = 0; q < (ALL ? 8 : 4); ++q) {
        const unsigned c = ALL ? lane + 32 * q : (lane & 15) + 16 * (warp >> 2) + 32 * (lane >> 4) + 64 * q;
        if (c < g.bn && row0 + c < g.m) plain &= is_plain(__ldg(g.sa + row0 + c));
    }
    return __all_sync(0xffffffffu, plain);
}

// One output where scales are not plain.
__device__ __forceinline__ void store_far(const TcArgs& g, const RowScale& r, int sum, unsigned row, unsigned col) {
    if (r.mine) {
        const float p = scaled(sum, __ldg(g.sa + row), r.scale);
        g.out[static_cast<unsigned long long>(row) * g.n + col] = g.bias ? p + r.bias : p;
    }
    __syncwarp();
}

// A warp's share of a finished tile: 32 weight rows (TMEM lanes, `first` the
// lowest) and every other 16 tokens, scaled and stored, 128 bytes of one token at
// a time. The next 16 leave TMEM while the present ones are stored.
__device__ __forceinline__ void store_tile(const TcArgs& g, const RowScale& r, bool plain, unsigned tmem,
                                           unsigned first, unsigned row0) {
    const unsigned warp = threadIdx.x >> 5, col = first + (threadIdx.x & 31);
    const unsigned rows = min(g.bn, g.m - row0), step = 16 * (kStoreWarps / 4);
    const unsigned taddr = tmem + ((warp & 3) * 32 << 16);
    const float* sa = g.sa + row0;
    const bool wide = (reinterpret_cast<std::uintptr_t>(sa) & 15) == 0;
    unsigned c = 16 * (warp >> 2);
    int v[16];
    __syncwarp();
    if (!plain) {
        // one token at a time: unrolled beside the rest, this kept every tile waiting for instructions
#pragma unroll 1
        for (; c < rows; c += c % 16 == 15 ? step - 15 : 1) store_far(g, r, tmem_load1(taddr + c), row0 + c, col);
        return;
    }
    if (c < rows) tmem_load16(taddr + c, v);
    for (; c < rows; c += step) {
        float s[16];
        if (wide && c + 16 <= rows) {
#pragma unroll
            for (unsigned j = 0; j < 4; ++j) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(sa + c) + j);
                s[4 * j] = f.x, s[4 * j + 1] = f.y, s[4 * j + 2] = f.z, s[4 * j + 3] = f.w;
            }
        } else {
#pragma unroll
            for (unsigned j = 0; j < 16; ++j) s[j] = c + j < rows ? __ldg(sa + c + j) : 1.0f;
        }
        __syncwarp();
        tmem_load_wait();
#pragma unroll
        for (unsigned j = 0; j < 16; ++j) s[j] = static_cast<float>(v[j]) * (s[j] * r.scale);
        if (g.bias) {
#pragma unroll
            for (unsigned j = 0; j < 16; ++j) s[j] += r.bias;
        }
        if (c + step < rows) tmem_load16(taddr + c + step, v);
        float* out = g.out + static_cast<unsigned long long>(row0 + c) * g.n + col;
        if (r.mine && c + 16 <= rows) {
#pragma unroll
            for (unsigned j = 0; j < 16; ++j) out[static_cast<unsigned long long>(j) * g.n] = s[j];
        } else if (r.mine) {
#pragma unroll
            for (unsigned j = 0; j < 16; ++j)
                if (c + j < rows) out[static_cast<unsigned long long>(j) * g.n] = s[j];
        }
    }
}

// Too few tiles for the SMs: a cluster of S CTAs shares a tile, each taking its
// part of k. A CTA hands every other one the sums of a share of the tokens and
// adds up its own share, which it scales and stores. The sums meet in scratch
// memory, which stays in L2: the cluster's shared memory takes some 15 bytes a
// clock from its neighbours, L2 four times that (256 x 4096 x 4096 spent 12 of 21
// us on the exchange by way of shared memory, 16 in all without it). Clusters of
// eight found fewer places on the GPU: 64 x 2048 x 4096 took 18 us with them, 10
// with four. One tile a CTA, no double buffer.
constexpr unsigned kMostSplit = 4;
struct SplitArgs {
    TcArgs g;
    unsigned split;       // CTAs a tile, 1, 2 or 4
    unsigned part;        // steps along k a CTA
    int* sums;            // scratch: [tile][CTA of the cluster][token][weight row]
};

__device__ __forceinline__ unsigned in_cta(const void* p, unsigned rank) {
    unsigned a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(kTcThreads, 1)
matmul_q8_split(const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap amap, const SplitArgs a) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ unsigned long long full[8], empty[8], acc_full[1];
    __shared__ unsigned tmem_base, dead_flag;
    volatile unsigned* dead = &dead_flag;
    const TcArgs& g = a.g;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned tile = blockIdx.x / a.split, rank = blockIdx.x - tile * a.split;
    const unsigned tm = tile / g.tiles_n, tn = tile - tm * g.tiles_n;
    const unsigned first = rank * a.part, last = min(g.steps, first + a.part);
    constexpr unsigned a_at = kTileM * kSliceK;
    const unsigned stage_bytes = a_at + g.bn * kSliceK;
    const auto fetch = [&](unsigned step, unsigned slot) {
        unsigned char* dst = tiles + slot * stage_bytes;
        mbar_expect_tx(full + slot, stage_bytes);
        const int x = static_cast<int>(step * kSliceK);
        tma_load_2d(dst, &bmap, full + slot, x, static_cast<int>(tn * kTileM));
        tma_load_2d(dst + a_at, &amap, full + slot, x, static_cast<int>(tm * g.bn));
    };
    const unsigned ahead = min(g.stages, last - first);
    if (warp == kStoreWarps && lane == 0) {
        dead_flag = 0;
        for (unsigned s = 0; s < g.stages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        mbar_init(acc_full, 1);
        mbar_fence_init();
        // the first stages are on their way while the others set up
        for (unsigned s = 0; s < ahead; ++s) fetch(first + s, s);
    }
    if (warp == kStoreWarps + 1)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(g.tmem_cols)
                     : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_base;
    RowScale r{};
    bool plain = true;

    if (warp == kStoreWarps) {  // fetch
        if (lane == 0) {
            unsigned issued = ahead;
            Place at;
            for (unsigned s = first + ahead; s < last; ++s, ++issued, at.next(g.stages)) {
                if (!tc_wait<false>(empty + at.slot, at.parity, dead, g.err)) break;
                fetch(s, at.slot);
            }
            drain(full, issued, g);
        }
    } else if (warp == kStoreWarps + 1) {  // products
        if (lane == 0) {
            Place at;
            bool ok = true;
            const unsigned long long da0 = tile_desc(smem_addr(tiles)), db0 = da0 + (a_at >> 4);
            for (unsigned s = first; s < last; ++s, at.next(g.stages)) {
                if (!(ok = tc_wait<false>(full + at.slot, at.parity, dead, g.err))) break;
                const unsigned long long skip = at.slot * (stage_bytes >> 4);
#pragma unroll
                for (unsigned j = 0; j < kSliceK / kMmaK; ++j)
                    mma_i8(tmem, da0 + skip + j * (kMmaK >> 4), db0 + skip + j * (kMmaK >> 4), g.idesc, s - first + j != 0);
                mma_commit(empty + at.slot);
            }
            if (ok) mma_commit(acc_full);
        }
    } else {
        r = row_scale(g, tn * kTileM + (warp & 3) * 32);
        plain = plain_scales<true>(g, r, tm * g.bn);
        const bool ok = tc_wait<false>(acc_full, 0, dead, g.err);
        tc_fence_after();
        if (ok && a.split == 1) store_tile(g, r, plain, tmem, tn * kTileM + (warp & 3) * 32, tm * g.bn);
    }
    if (a.split > 1) {
        const unsigned share = g.bn / a.split, mine0 = rank * share;
        int* sums = a.sums + static_cast<unsigned long long>(tile) * a.split * g.bn * kTileM;  // the tile's
        const unsigned l = (warp & 3) * 32 + lane, taddr = tmem + ((warp & 3) * 32 << 16);
        constexpr unsigned stride = 16 * (kStoreWarps / 4);
        if (warp < kStoreWarps) {
            // tokens 16 at a time, a lane the sums of one weight row; its own share stays
            int* own = sums + static_cast<unsigned long long>(rank) * g.bn * kTileM + l;
            for (unsigned c = 16 * (warp >> 2); c < g.bn; c += stride) {
                int v[16];
                tmem_load16(taddr + c, v);
                tmem_load_wait();
#pragma unroll
                for (unsigned j = 0; j < 16; ++j)
                    if (c + j - mine0 >= share) __stcg(own + (c + j) * kTileM, v[j]);
            }
            __threadfence();
        }
        __syncwarp();
        cluster_barrier();
        if (warp < kStoreWarps) {
            const unsigned col = tn * kTileM + l;
            if (!plain) {
#pragma unroll 1
                for (unsigned t = mine0 + (warp >> 2); t < min(mine0 + share, g.m - tm * g.bn); t += kStoreWarps / 4) {
                    int sum = tmem_load1(taddr + t);
                    for (unsigned q = 1; q < a.split; ++q) {
                        const unsigned from = (rank + q) % a.split;
                        sum += __ldcg(sums + (static_cast<unsigned long long>(from) * g.bn + t) * kTileM + l);
                    }
                    store_far(g, r, sum, tm * g.bn + t, col);
                }
            }
            for (unsigned c = mine0 / 16 * 16 + 16 * (warp >> 2); plain && c < mine0 + share; c += stride) {
                int v[16];
                tmem_load16(taddr + c, v);
                int o[kMostSplit - 1][16];  // the others', in flight together
#pragma unroll
                for (unsigned q = 0; q < kMostSplit - 1; ++q) {
                    const unsigned from = (rank + 1 + q) % a.split;
                    const int* other = sums + static_cast<unsigned long long>(from) * g.bn * kTileM + l;
#pragma unroll
                    for (unsigned j = 0; j < 16; ++j)
                        o[q][j] = q + 1 < a.split && c + j - mine0 < share ? __ldcg(other + (c + j) * kTileM) : 0;
                }
                __syncwarp();
                tmem_load_wait();
#pragma unroll
                for (unsigned q = 0; q < kMostSplit - 1; ++q)
#pragma unroll
                    for (unsigned j = 0; j < 16; ++j) v[j] += o[q][j];
                const unsigned row0 = tm * g.bn + c;
#pragma unroll
                for (unsigned j = 0; j < 16; ++j)
                    if (c + j - mine0 < share && r.mine && row0 + j < g.m) {
                        const float p = static_cast<float>(v[j]) * (__ldg(g.sa + row0 + j) * r.scale);
                        g.out[static_cast<unsigned long long>(row0 + j) * g.n + col] = g.bias ? p + r.bias : p;
                    }
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kStoreWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols));
    }
}

// Tiles enough for all SMs: pairs of CTAs walk tiles of 256 weight rows by up to
// 256 tokens. Each CTA fetches its own 128 weight rows and half of the tokens, and
// the instruction, issued by the first CTA of the pair, reads both CTAs' shared
// memory: a third less to fetch and to hold for a stage than one CTA's 128 x 256
// tile. The previous tile leaves the other half of TMEM meanwhile. A stage holds
// 256 bytes of k, eight products: with 128 the one thread's wait, issue and commit
// took longer than the four products they bring (8192^3: 385 us with one CTA a
// tile and 128 bytes, 313 this way on the same card; 345 alone on another, 3.2 Pop/s,
// and 2.6 in a long run under the 1000 W limit).
constexpr unsigned kPairSlices = 2;

__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, unsigned bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc,
                                            bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<unsigned>(accumulate))
        : "memory");
}
// arrives at the barrier of this place in both CTAs
__device__ __forceinline__ void mma_commit_pair(unsigned long long* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"(static_cast<unsigned short>(3))
        : "memory");
}
__device__ __forceinline__ void arrive_at(unsigned bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__global__ void __launch_bounds__(kTcThreads, 1)
matmul_q8_pair(const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap amap, const TcArgs g) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ unsigned long long full[8], empty[8], acc_full[2], acc_empty[2];
    __shared__ unsigned tmem_base, dead_flag;
    volatile unsigned* dead = &dead_flag;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = blockIdx.x & 1, pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
    const unsigned half_bn = g.bn / 2;
    constexpr unsigned a_at = kPairSlices * kTileM * kSliceK;
    const unsigned stage_bytes = a_at + kPairSlices * half_bn * kSliceK;
    const unsigned copied = kPairSlices * (g.rows + half_bn) * kSliceK;  // of a stage
    const unsigned ntiles = g.tiles_m * g.tiles_n;
    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (unsigned s = 0; s < g.stages; ++s) {
            mbar_init(full + s, 1);   // the first CTA's are used
            mbar_init(empty + s, 1);
        }
        for (unsigned s = 0; s < 2; ++s) {
            mbar_init(acc_full + s, 1);
            mbar_init(acc_empty + s, 2 * kStoreWarps);  // the first CTA's: the warps of both
        }
        mbar_fence_init();
    }
    if (warp == kStoreWarps + 1)
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(g.tmem_cols)
                     : "memory");
    tc_fence_before();
    __syncthreads();
    cluster_barrier();
    tc_fence_after();
    const unsigned tmem = tmem_base;

    if (warp == kStoreWarps) {  // fetch
        if (lane == 0) {
            Place at;
            unsigned issued = 0;
            bool ok = true;
            const unsigned bars = in_cta(full, 0);
            for (unsigned i = first; ok && i < ntiles; i += pairs) {
                unsigned tn, tm;
                tile_at(i, g, tn, tm);
                const int row_b = static_cast<int>((2 * tn + rank) * g.rows), row_a = static_cast<int>(tm * g.bn + rank * half_bn);
                for (unsigned s = 0; s < g.steps; ++s, ++issued, at.next(g.stages)) {
                    if (issued >= g.stages && !(ok = tc_wait<false>(empty + at.slot, at.parity ^ 1, dead, g.err))) break;
                    unsigned char* dst = tiles + at.slot * stage_bytes;
                    const unsigned bar = bars + at.slot * 8;
                    if (rank == 0) mbar_expect_tx(full + at.slot, 2 * copied);
                    for (unsigned j = 0; j < kPairSlices; ++j) {
                        const int x = static_cast<int>((s * kPairSlices + j) * kSliceK);
                        tma_load_2d_pair(dst + j * kTileM * kSliceK, &bmap, bar, x, row_b);
                        tma_load_2d_pair(dst + a_at + j * half_bn * kSliceK, &amap, bar, x, row_a);
                    }
                }
            }
            // the second CTA's copies are waited for by the first (cluster barrier below)
            if (rank == 0) drain(full, issued, g);
        }
    } else if (warp == kStoreWarps + 1) {  // products, issued by the first CTA
        if (lane == 0 && rank == 0) {
            Place at;
            unsigned turn = 0;
            bool ok = true;
            const unsigned long long da0 = tile_desc(smem_addr(tiles)), db0 = da0 + (a_at >> 4);
            for (unsigned i = first; ok && i < ntiles; i += pairs, ++turn) {
                const unsigned half = turn & 1, d = tmem + half * g.bn;
                if (turn > 1 && !(ok = tc_wait<false>(acc_empty + half, ((turn >> 1) - 1) & 1, dead, g.err))) break;
                tc_fence_after();
                for (unsigned s = 0; s < g.steps; ++s, at.next(g.stages)) {
                    if (!(ok = tc_wait<false>(full + at.slot, at.parity, dead, g.err))) break;
                    const unsigned long long skip = at.slot * (stage_bytes >> 4);
#pragma unroll
                    for (unsigned p = 0; p < kPairSlices; ++p) {
                        const unsigned long long da = da0 + skip + p * (kTileM * kSliceK >> 4);
                        const unsigned long long db = db0 + skip + p * (half_bn * kSliceK >> 4);
#pragma unroll
                        for (unsigned j = 0; j < kSliceK / kMmaK; ++j)
                            mma_i8_pair(d, da + j * (kMmaK >> 4), db + j * (kMmaK >> 4), g.idesc, s + p + j != 0);
                    }
                    mma_commit_pair(empty + at.slot);
                }
                if (ok) mma_commit_pair(acc_full + half);
            }
        }
    } else {  // scale and store
        unsigned turn = 0;
        for (unsigned i = first; i < ntiles; i += pairs, ++turn) {
            const unsigned half = turn & 1;
            unsigned tn, tm;
            tile_at(i, g, tn, tm);
            const RowScale r = row_scale(g, (2 * tn + rank) * g.rows + (warp & 3) * 32);
            const bool plain = plain_scales<false>(g, r, tm * g.bn);
            if (!tc_wait(acc_full + half, (turn >> 1) & 1, dead, g.err)) break;
            tc_fence_after();
            store_tile(g, r, plain, tmem + half * g.bn, (2 * tn + rank) * g.rows + (warp & 3) * 32, tm * g.bn);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(in_cta(acc_empty + half, 0));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // neither CTA's shared memory is read or arrived at any more
    if (warp == kStoreWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols));
    }
}

// k = 0: the sums are zero.
__global__ void __launch_bounds__(256)
matmul_q8_empty(const float* sa, const float* sb, const float* bias, unsigned m, unsigned n, float* out) {
    const unsigned long long count = static_cast<unsigned long long>(m) * n;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < count; i += gridDim.x * 256ull) {
        const unsigned r = static_cast<unsigned>(i / n), c = static_cast<unsigned>(i - static_cast<unsigned long long>(r) * n);
        const float v = scaled(0, sa[r], sb[c]);
        out[i] = bias ? v + bias[c] : v;
    }
}

// Rows of 128-byte slices, `box` of them a copy; zeros past k and past the rows.
CUtensorMap slice_map(const signed char* p, unsigned rows, unsigned k, unsigned long long pitch, unsigned box) {
    const cuuint64_t dims[2] = {k, rows};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t boxes[2] = {kSliceK, box};
    const cuuint32_t steps[2] = {1, 1};
    CUtensorMap map;
    const auto encode = encode_tiled();
    if (!encode) fail(VC_ERR_RUNTIME, "matmul_q8: cuTensorMapEncodeTiled is not available");
    const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<signed char*>(p), dims, strides, boxes,
                              steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(VC_ERR_RUNTIME, "matmul_q8: the tensor map was refused (" + std::to_string(r) + ")");
    return map;
}

// Stages take up to 220 KB; 1 KB more aligns them.
constexpr int kTcSmem = 222 * 1024;

void launch_pair(const MatmulQ8Args& a) {
    TcArgs g{};
    g.sa = a.sa, g.sb = a.sb, g.bias = a.bias, g.out = a.out, g.m = a.m, g.n = a.n;
    g.err = device_error_word();
    g.bn = std::min(256u, (a.m + 31) / 32 * 32);
    g.steps = (a.k + kPairSlices * kSliceK - 1) / (kPairSlices * kSliceK);
    g.tiles_m = (a.m + g.bn - 1) / g.bn;
    // With one tile of tokens the weights' way from HBM counts: as many tiles as the
    // turns that full ones take have room for, of fewer rows (100 x 20000 x 4096:
    // 24.9 us, with full ones in the same two turns 27.9). A single turn has no
    // more to gain, and products bound by the tensor cores lose (1000 x 14336 x
    // 4096: 56 against 54).
    const unsigned pairs = static_cast<unsigned>(sm_count()) / 2, full = (a.n + 2 * kTileM - 1) / (2 * kTileM);
    const unsigned long long turns = (static_cast<unsigned long long>(full) * g.tiles_m + pairs - 1) / pairs;
    const unsigned room = static_cast<unsigned>(turns * pairs / g.tiles_m);  // tiles along the weights
    g.rows = g.tiles_m == 1 && turns > 1 ? (a.n + 16 * room - 1) / (16 * room) * 8 : kTileM;
    g.tiles_n = (a.n + 2 * g.rows - 1) / (2 * g.rows);
    const unsigned stage = kPairSlices * (kTileM + g.bn / 2) * kSliceK;  // in each CTA
    g.stages = std::min(8u, 220u * 1024 / stage);
    g.tmem_cols = 32;
    while (g.tmem_cols < 2 * g.bn) g.tmem_cols *= 2;
    // 32-bit integer accumulators, signed 8-bit sides, both K-major
    g.idesc = 2u << 4 | 1u << 7 | 1u << 10 | (g.bn >> 3) << 17 | (2 * kTileM >> 4) << 24;
    if (static_cast<unsigned long long>(g.tiles_m) * g.tiles_n > 0x7fffffffull)
        fail(VC_ERR_OVERFLOW, "matmul_q8: too many tiles");
    const CUtensorMap bmap = slice_map(a.b, a.n, a.k, a.bp, g.rows), amap = slice_map(a.a, a.m, a.k, a.ap, g.bn / 2);
    allow_smem<matmul_q8_pair, kTcSmem>();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * std::min(g.tiles_m * g.tiles_n, pairs));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = g.stages * stage + 1024;
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VC_CUDA(cudaLaunchKernelEx(&cfg, matmul_q8_pair, bmap, amap, g));
    check_launch("matmul_q8_pair");
}

// The least steps along k that are worth a CTA of their own (with 2 or 8 the
// sizes above run the same within 1%).
constexpr unsigned kSplitSteps = 4;

void launch_split(const MatmulQ8Args& a) {
    SplitArgs p{};
    TcArgs& g = p.g;
    g.sa = a.sa, g.sb = a.sb, g.bias = a.bias, g.out = a.out, g.m = a.m, g.n = a.n;
    g.err = device_error_word();
    const unsigned token_tiles = (a.m + 255) / 256;
    g.bn = ((a.m + token_tiles - 1) / token_tiles + 15) / 16 * 16;
    g.rows = kTileM;
    g.steps = (a.k + kSliceK - 1) / kSliceK;
    g.tiles_m = (a.m + g.bn - 1) / g.bn;
    g.tiles_n = (a.n + kTileM - 1) / kTileM;
    const unsigned stage = (kTileM + g.bn) * kSliceK;
    const unsigned ntiles = g.tiles_m * g.tiles_n, sms = static_cast<unsigned>(sm_count());
    g.stages = std::min(8u, 220u * 1024 / stage);
    p.split = 1;
    while (p.split < kMostSplit && 2 * p.split * ntiles <= sms && g.steps >= 2 * p.split * kSplitSteps) p.split *= 2;
    p.part = (g.steps + p.split - 1) / p.split;
    while (p.split > 1 && (p.split - 1) * p.part >= g.steps) p.split /= 2, p.part = (g.steps + p.split - 1) / p.split;
    g.tmem_cols = 32;
    while (g.tmem_cols < g.bn) g.tmem_cols *= 2;
    Scratch sums(p.split > 1 ? static_cast<std::size_t>(ntiles) * p.split * g.bn * kTileM * sizeof(int) : 16);
    p.sums = sums.as<int>();
    g.idesc = 2u << 4 | 1u << 7 | 1u << 10 | (g.bn >> 3) << 17 | (kTileM >> 4) << 24;
    const CUtensorMap bmap = slice_map(a.b, a.n, a.k, a.bp, kTileM), amap = slice_map(a.a, a.m, a.k, a.ap, g.bn);
    allow_smem<matmul_q8_split, kTcSmem>();
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ntiles * p.split);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = g.stages * stage + 1024;
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VC_CUDA(cudaLaunchKernelEx(&cfg, matmul_q8_split, bmap, amap, p));
    check_launch("matmul_q8_split");
}

void check_q8_in(const char* name, const void* p, std::size_t pitch, std::size_t k) {
    if (pitch < k || pitch % 16 != 0 || !aligned16(p))
        fail(VC_ERR_INVALID, std::string("matmul_q8: the rows of ") + name +
                                 " need a pitch of at least k, and a multiple of 16 bytes, on a 16-byte aligned base");
}

}  // namespace
}  // namespace vc

using namespace vc;

extern "C" {

vc_status vc_cuda_matmul_q8(const int8_t* a, size_t a_pitch, const float* a_scale, const int8_t* b, size_t b_pitch,
                            const float* b_scale, const float* bias, size_t m, size_t n, size_t k, float* out) {
    VC_API_BEGIN
    ensure_init();
    if (k > kQ8MaxK) fail(VC_ERR_OVERFLOW, "matmul_q8: k is limited to 131071 (32-bit sums)");
    if (m > 0x3fffffffu || n > 0x3fffffffu || (m && n > (1ull << 60) / m))
        fail(VC_ERR_OVERFLOW, "matmul_q8: matrix too large");
    if (m == 0 || n == 0) return VC_OK;
    if (!a_scale || !b_scale || !out || (k && (!a || !b))) fail(VC_ERR_INVALID, "matmul_q8: null pointer");
    check_elements("matmul_q8", a_scale, b_scale, bias, out);
    check_q8_in("a", a, a_pitch, k);
    check_q8_in("b", b, b_pitch, k);
    MatmulQ8Args g{};
    g.a = reinterpret_cast<const signed char*>(a), g.b = reinterpret_cast<const signed char*>(b);
    g.ap = a_pitch, g.bp = b_pitch, g.sa = a_scale, g.sb = b_scale, g.bias = bias, g.out = out;
    g.m = static_cast<unsigned>(m), g.n = static_cast<unsigned>(n), g.k = static_cast<unsigned>(k);
    if (k == 0) {
        matmul_q8_empty<<<grid_for(m * n, 256), 256, 0, stream()>>>(a_scale, b_scale, bias, g.m, g.n, out);
        check_launch("matmul_q8_empty");
    } else {
        // Tiles of 128 weight rows and up to 256 tokens, against the SMs (all in
        // us, k = 4096): below half of them a tile is shared (64 x 4096: 9.5, in
        // pairs 13.3; 200 x 8192, at half: 17.0 and 17.9), else pairs walk the
        // tiles (64 x 11008: 15.2, one CTA a tile 16.2; 4096 x 4096: 54 and 79).
        // Up to 8 tokens the weights go straight to registers (8 x 32000: 26, in
        // pairs 30), up to 16 while the tiles are few (16 x 4096: 6.8, shared
        // 9.1; 16 x 8192 the other way, 13.1 and 12.2).
        const size_t sms = static_cast<size_t>(sm_count());
        const size_t tiles = ((n + kTileM - 1) / kTileM) * ((m + 255) / 256);
        if (m <= 8 || (m <= 16 && 4 * tiles <= sms)) launch_rows(g);
        else if (2 * tiles <= sms) launch_split(g);
        else launch_pair(g);
    }
    VC_API_END
}

}  // extern "C"
