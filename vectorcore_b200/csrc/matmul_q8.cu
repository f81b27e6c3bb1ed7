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

// 64 x 64 outputs a CTA, 4 x 4 a thread, k in steps of 32 bytes through shared
// memory, four products an instruction (dp4a).
__global__ void __launch_bounds__(256)
matmul_q8_dp4a(const MatmulQ8Args g) {
    __shared__ int as[64][9];
    __shared__ int bs[64][9];
    const unsigned row0 = blockIdx.y * 64, col0 = blockIdx.x * 64;
    const unsigned tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (unsigned k0 = 0; k0 < g.k; k0 += 32) {
        for (unsigned i = threadIdx.x; i < 512; i += 256) {
            const unsigned r = i >> 3, c = i & 7, at = k0 + 4 * c;
            unsigned va = 0, vb = 0;
            if (at < g.k) {
                // bytes past k are dropped from a alone: their products are zero
                const unsigned mask = g.k - at >= 4 ? 0xffffffffu : (1u << (8 * (g.k - at))) - 1;
                if (row0 + r < g.m) va = *reinterpret_cast<const unsigned*>(g.a + (row0 + r) * g.ap + at) & mask;
                if (col0 + r < g.n) vb = *reinterpret_cast<const unsigned*>(g.b + (col0 + r) * g.bp + at);
            }
            as[r][c] = static_cast<int>(va);
            bs[r][c] = static_cast<int>(vb);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(as[ty * 4 + i][c], bs[tx * 4 + j][c], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const unsigned r = row0 + ty * 4 + i, c = col0 + tx * 4 + j;
            if (r >= g.m || c >= g.n) continue;
            const float v = static_cast<float>(acc[i][j]) * (g.sa[r] * g.sb[c]);
            g.out[static_cast<unsigned long long>(r) * g.n + c] = g.bias ? v + g.bias[c] : v;
        }
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
    const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>((m + 63) / 64));
    if (grid.y > 65535) fail(VC_ERR_OVERFLOW, "matmul_q8: too many rows");
    matmul_q8_dp4a<<<grid, 256, 0, stream()>>>(g);
    check_launch("matmul_q8_dp4a");
    VC_API_END
}

}  // extern "C"
