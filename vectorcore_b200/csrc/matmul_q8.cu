// matmul_q8.cu -- product of 8-bit rows with a scale for each row of either
// side:
//
//   out[i, j] = (sum over p of a[i, p] * b[j, p]) * (a_scale[i] * b_scale[j]) + bias[j]
//
// The sums are 32-bit integers, so they are exact and do not depend on the
// order of the additions (|a * b| <= 2^14, hence k <= 131071).
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

// ---- Blackwell tensor cores ------------------------------------------------------
//
// The weights b are the instruction's M side and the tokens a its N side, so a
// tile's accumulators lie in TMEM with one weight row a lane: a warp's store of
// one register is 32 neighbouring outputs of one token, coalesced whatever n's
// alignment, with no trip through shared memory.
//
// One CTA an SM walks the tiles: a warp fetches 128-byte slices of k of both
// sides by TMA (128-byte swizzle, zeros past the ends, so k, m and n need no
// alignment), one thread of another issues the products (32 bytes of k each),
// and four warps scale and store the previous tile out of the other half of
// TMEM meanwhile.

constexpr unsigned kTileM = 128;   // weight rows a tile: TMEM's lanes
constexpr unsigned kSliceK = 128;  // bytes of k a stage: one swizzled row
constexpr unsigned kMmaK = 32;     // bytes of k an instruction
constexpr unsigned kTcThreads = 192;
constexpr long long kTcPolls = 1ll << 18;  // a wait gives up after about half a second

struct TcArgs {
    const float* sa;
    const float* sb;
    const float* bias;
    float* out;
    unsigned m, n;
    unsigned bn;          // tokens a tile, a multiple of 16
    unsigned slices;      // of k
    unsigned tiles_m;     // along the tokens
    unsigned tiles_n;     // along the weights
    unsigned stages;
    unsigned tmem_cols;   // allocated: both halves
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
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A bounded wait that also ends when another role of the CTA gave up.
__device__ __forceinline__ bool tc_wait(unsigned long long* bar, unsigned parity, volatile unsigned* dead,
                                        unsigned* err) {
    for (long long i = 0; i < kTcPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*dead) return false;
    }
    *dead = 1;
    atomicOr(err, kErrWaitTimeout);
    return false;
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

__global__ void __launch_bounds__(kTcThreads, 1)
matmul_q8_tc(const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap amap, const TcArgs g) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ unsigned long long full[8], empty[8], acc_full[2], acc_empty[2];
    __shared__ unsigned tmem_base, dead_flag;
    volatile unsigned* dead = &dead_flag;
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned stage_bytes = (kTileM + g.bn) * kSliceK;
    const unsigned ntiles = g.tiles_m * g.tiles_n;
    if (threadIdx.x == 0) {
        dead_flag = 0;
        for (unsigned s = 0; s < g.stages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (unsigned s = 0; s < 2; ++s) {
            mbar_init(acc_full + s, 1);
            mbar_init(acc_empty + s, 4);
        }
        mbar_fence_init();
    }
    if (warp == 5)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(g.tmem_cols)
                     : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_base;

    if (warp == 4) {  // fetch
        if (lane == 0) {
            unsigned issued = 0;
            bool ok = true;
            for (unsigned i = blockIdx.x; ok && i < ntiles; i += gridDim.x) {
                unsigned tn, tm;
                tile_at(i, g, tn, tm);
                for (unsigned s = 0; s < g.slices; ++s, ++issued) {
                    const unsigned slot = issued % g.stages, turn = issued / g.stages;
                    if (turn && !(ok = tc_wait(empty + slot, (turn - 1) & 1, dead, g.err))) break;
                    unsigned char* at = tiles + slot * stage_bytes;
                    mbar_expect_tx(full + slot, stage_bytes);
                    tma_load_2d(at, &bmap, full + slot, static_cast<int>(s * kSliceK), static_cast<int>(tn * kTileM));
                    tma_load_2d(at + kTileM * kSliceK, &amap, full + slot, static_cast<int>(s * kSliceK),
                                static_cast<int>(tm * g.bn));
                }
            }
            // the copies still in flight land before the CTA may finish
            for (unsigned s = issued > g.stages ? issued - g.stages : 0; s < issued; ++s)
                mbar_wait_bounded(full + s % g.stages, (s / g.stages) & 1, g.err, kTcPolls);
        }
    } else if (warp == 5) {  // products
        if (lane == 0) {
            unsigned used = 0, turn = 0;
            bool ok = true;
            for (unsigned i = blockIdx.x; ok && i < ntiles; i += gridDim.x, ++turn) {
                const unsigned half = turn & 1;
                if (turn > 1 && !(ok = tc_wait(acc_empty + half, ((turn >> 1) - 1) & 1, dead, g.err))) break;
                tc_fence_after();
                for (unsigned s = 0; s < g.slices; ++s, ++used) {
                    const unsigned slot = used % g.stages;
                    if (!(ok = tc_wait(full + slot, (used / g.stages) & 1, dead, g.err))) break;
                    tc_fence_after();
                    const unsigned at = smem_addr(tiles + slot * stage_bytes);
                    const unsigned long long da = tile_desc(at), db = tile_desc(at + kTileM * kSliceK);
#pragma unroll
                    for (unsigned j = 0; j < kSliceK / kMmaK; ++j)
                        mma_i8(tmem + half * g.bn, da + j * (kMmaK >> 4), db + j * (kMmaK >> 4), g.idesc, s + j != 0);
                    mma_commit(empty + slot);
                }
                if (ok) mma_commit(acc_full + half);
            }
        }
    } else {  // scale and store
        unsigned turn = 0;
        for (unsigned i = blockIdx.x; i < ntiles; i += gridDim.x, ++turn) {
            const unsigned half = turn & 1;
            if (!tc_wait(acc_full + half, (turn >> 1) & 1, dead, g.err)) break;
            tc_fence_after();
            unsigned tn, tm;
            tile_at(i, g, tn, tm);
            const unsigned col = tn * kTileM + warp * 32 + lane;
            const bool mine = col < g.n;
            const float sb = mine ? g.sb[col] : 0.0f, bias = mine && g.bias ? g.bias[col] : 0.0f;
            const unsigned row0 = tm * g.bn, rows = min(g.bn, g.m - row0);
            float* out = g.out + static_cast<unsigned long long>(row0) * g.n + col;
            const unsigned taddr = tmem + (warp * 32 << 16) + half * g.bn;
            for (unsigned c = 0; c < rows; c += 16) {
                int v[16];
                __syncwarp();
                tmem_load16(taddr + c, v);
                tmem_load_wait();
                if (mine) {
#pragma unroll
                    for (unsigned j = 0; j < 16; ++j)
                        if (c + j < rows) {
                            const float p = static_cast<float>(v[j]) * (__ldg(g.sa + row0 + c + j) * sb);
                            out[static_cast<unsigned long long>(c + j) * g.n] = g.bias ? p + bias : p;
                        }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + half);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols));
    }
}

// k = 0: the sums are zero.
__global__ void __launch_bounds__(256)
matmul_q8_empty(const float* sa, const float* sb, const float* bias, unsigned m, unsigned n, float* out) {
    const unsigned long long count = static_cast<unsigned long long>(m) * n;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < count; i += gridDim.x * 256ull) {
        const unsigned r = static_cast<unsigned>(i / n), c = static_cast<unsigned>(i - static_cast<unsigned long long>(r) * n);
        const float v = 0.0f * (sa[r] * sb[c]);
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

void launch_tc(const MatmulQ8Args& a) {
    TcArgs g{};
    g.sa = a.sa, g.sb = a.sb, g.bias = a.bias, g.out = a.out, g.m = a.m, g.n = a.n;
    g.err = device_error_word();
    g.bn = std::min(256u, (a.m + 15) / 16 * 16);
    g.slices = (a.k + kSliceK - 1) / kSliceK;
    g.tiles_m = (a.m + g.bn - 1) / g.bn;
    g.tiles_n = (a.n + kTileM - 1) / kTileM;
    const unsigned stage = (kTileM + g.bn) * kSliceK;
    g.stages = std::min(8u, 220u * 1024 / stage);
    g.tmem_cols = 32;
    while (g.tmem_cols < 2 * g.bn) g.tmem_cols *= 2;
    // 32-bit integer accumulators, signed 8-bit sides, both K-major
    g.idesc = 2u << 4 | 1u << 7 | 1u << 10 | (g.bn >> 3) << 17 | (kTileM >> 4) << 24;
    if (static_cast<unsigned long long>(g.tiles_m) * g.tiles_n > 0x7fffffffull)
        fail(VC_ERR_OVERFLOW, "matmul_q8: too many tiles");
    const CUtensorMap bmap = slice_map(a.b, a.n, a.k, a.bp, kTileM), amap = slice_map(a.a, a.m, a.k, a.ap, g.bn);
    constexpr unsigned kMaxSmem = 222 * 1024;
    static bool configured = false;
    if (!configured) {
        VC_CUDA(cudaFuncSetAttribute(matmul_q8_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
        configured = true;
    }
    const unsigned grid = std::min(g.tiles_m * g.tiles_n, static_cast<unsigned>(sm_count()));
    matmul_q8_tc<<<grid, kTcThreads, g.stages * stage + 1024, stream()>>>(bmap, amap, g);
    check_launch("matmul_q8_tc");
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
        launch_tc(g);
    }
    VC_API_END
}

}  // extern "C"
