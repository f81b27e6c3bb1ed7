// The C++ forms of the language-model operators for ctypes: host arrays in and
// out, and calls that have to be refused.
#include "cuda_backend.hpp"

#include "vc_cuda.h"

#include <functional>
#include <stdexcept>
#include <vector>

using namespace vectorcore;

namespace {

using Ptr = std::shared_ptr<Storage>;

std::shared_ptr<CudaStorage> room(std::size_t elements, std::size_t bytes = sizeof(float)) {
    return std::make_shared<CudaStorage>(elements, Device::cuda(), bytes);
}
template <typename T>
std::shared_ptr<CudaStorage> up(const T* data, std::size_t elements) {
    auto s = room(elements, sizeof(T));
    if (vc_cuda_upload(s->raw(), data, elements * sizeof(T)) != VC_OK) throw std::runtime_error(vc_cuda_last_error());
    return s;
}
template <typename T>
void down(const Ptr& s, T* data, std::size_t elements) {
    const auto& c = dynamic_cast<const CudaStorage&>(*s);
    if (vc_cuda_download(data, c.raw(), elements * sizeof(T)) != VC_OK) throw std::runtime_error(vc_cuda_last_error());
}

// What f throws, as the C ABI's status; 0 if nothing.
int status_of(const std::function<void()>& f) {
    try {
        f();
    } catch (const std::invalid_argument&) {
        return VC_ERR_INVALID;
    } catch (const std::out_of_range&) {
        return VC_ERR_OUT_OF_RANGE;
    } catch (const std::overflow_error&) {
        return VC_ERR_OVERFLOW;
    } catch (const std::exception&) {
        return VC_ERR_RUNTIME;
    }
    return VC_OK;
}

}  // namespace

extern "C" {

int form_rms_norm(const float* x, const float* r, const float* w, std::size_t rows, std::size_t cols, float eps,
                  const float* gy, const float* gh, float* y, float* h, float* rstd, float* dh, float* dw) {
    return status_of([&] {
        auto& be = CudaBackend::instance();
        const std::size_t n = rows * cols;
        const auto dx = up(x, n), dwt = up(w, cols), dgy = up(gy, n);
        const auto dr = r ? up(r, n) : nullptr, dgh = gh ? up(gh, n) : nullptr;
        const auto f = be.rms_norm(*dx, dr.get(), *dwt, rows, cols, eps);
        if (!r != !f.h) throw std::logic_error("h comes with a residual");
        const Storage& hs = f.h ? *f.h : *dx;
        const auto b = be.rms_norm_backward(hs, *dwt, *f.rstd, *dgy, dgh.get(), rows, cols);
        down(f.y, y, n), down(f.rstd, rstd, rows), down(b.dh, dh, n), down(b.dw, dw, cols);
        if (f.h) down(f.h, h, n);
    });
}

// rows through the norm (or as they are, w null) in 8 bits, times the 8-bit rows of b
int form_q8(const float* x, const float* r, const float* w, std::size_t rows, std::size_t cols, const float* b,
            std::size_t n, const float* bias, signed char* q, float* scale, float* h, float* out) {
    return status_of([&] {
        auto& be = CudaBackend::instance();
        const auto dx = up(x, rows * cols), db = up(b, n * cols);
        const auto dr = r ? up(r, rows * cols) : nullptr, dw = w ? up(w, cols) : nullptr, dbias = bias ? up(bias, n) : nullptr;
        CudaBackend::Q8Matrix a;
        if (w) {
            auto f = be.rms_norm_q8(*dx, dr.get(), *dw, rows, cols, 1e-6f);
            if (!r != !f.h) throw std::logic_error("h comes with a residual");
            if (f.h) down(f.h, h, rows * cols);
            a = f.q;
        } else {
            a = be.quantize_q8(*dx, rows, cols);
        }
        down(be.matmul_q8(a, be.quantize_q8(*db, n, cols), dbias.get()), out, rows * n);
        down(a.values, q, rows * a.pitch), down(a.scale, scale, rows);
    });
}

int form_sample(const float* x, const float* noise, std::size_t rows, std::size_t vocab, const float* temperature,
                const std::int64_t* top_k, const float* top_p, const float* min_p, std::int64_t* token,
                float* logprob) {
    return status_of([&] {
        const auto dx = up(x, rows * vocab), dn = up(noise, rows * vocab);
        const auto t = temperature ? up(temperature, rows) : nullptr, k = top_k ? up(top_k, rows) : nullptr,
                   p = top_p ? up(top_p, rows) : nullptr, m = min_p ? up(min_p, rows) : nullptr;
        const auto s = CudaBackend::instance().sample(*dx, *dn, {t.get(), k.get(), p.get(), m.get()}, rows, vocab);
        down(s.token, token, rows), down(s.logprob, logprob, rows);
    });
}

// Calls with one storage too short or of another type, of 6 rows of 10; the
// status each is refused with, in order, as many as there are.
int form_refusals(int* status, int most) {
    auto& be = CudaBackend::instance();
    const std::size_t R = 6, C = 10, N = 60;
    const auto ok = room(N), w = room(C), rs = room(R), shorter = room(N - 1), w9 = room(C - 1), r5 = room(R - 1);
    const auto wide = room(N, 8), k64 = room(R, 8), k5 = room(R - 1, 8), q = room(R * 16, 1), q_short = room(5 * 16 + 9, 1);
    using Settings = CudaBackend::SampleSettings;
    using Q8 = CudaBackend::Q8Matrix;
    const Q8 a{q, rs, R, C, 16};
    const std::vector<std::function<void()>> calls = {
        [&] { (void)be.rms_norm(*shorter, nullptr, *w, R, C, 1e-6f); },
        [&] { (void)be.rms_norm(*ok, shorter.get(), *w, R, C, 1e-6f); },
        [&] { (void)be.rms_norm(*ok, nullptr, *w9, R, C, 1e-6f); },
        [&] { (void)be.rms_norm_backward(*shorter, *w, *rs, *ok, nullptr, R, C); },
        [&] { (void)be.rms_norm_backward(*ok, *w9, *rs, *ok, nullptr, R, C); },
        [&] { (void)be.rms_norm_backward(*ok, *w, *r5, *ok, nullptr, R, C); },
        [&] { (void)be.rms_norm_backward(*ok, *w, *rs, *shorter, nullptr, R, C); },
        [&] { (void)be.rms_norm_backward(*ok, *w, *rs, *ok, shorter.get(), R, C); },
        [&] { (void)be.rms_norm_q8(*shorter, nullptr, *w, R, C, 1e-6f); },
        [&] { (void)be.rms_norm_q8(*ok, shorter.get(), *w, R, C, 1e-6f); },
        [&] { (void)be.rms_norm_q8(*ok, nullptr, *w9, R, C, 1e-6f); },
        [&] { (void)be.quantize_q8(*shorter, R, C); },
        [&] { (void)be.matmul_q8(Q8{q_short, rs, R, C, 16}, a, nullptr); },
        [&] { (void)be.matmul_q8(a, Q8{q_short, rs, R, C, 16}, nullptr); },
        [&] { (void)be.matmul_q8(Q8{q, r5, R, C, 16}, a, nullptr); },
        [&] { (void)be.matmul_q8(a, Q8{q, r5, R, C, 16}, nullptr); },
        [&] { (void)be.matmul_q8(a, a, r5.get()); },
        [&] { (void)be.sample(*shorter, *ok, {}, R, C); },
        [&] { (void)be.sample(*ok, *shorter, {}, R, C); },
        [&] { (void)be.sample(*ok, *ok, Settings{r5.get(), nullptr, nullptr, nullptr}, R, C); },
        [&] { (void)be.sample(*ok, *ok, Settings{nullptr, k5.get(), nullptr, nullptr}, R, C); },
        [&] { (void)be.sample(*ok, *ok, Settings{nullptr, nullptr, r5.get(), nullptr}, R, C); },
        [&] { (void)be.sample(*ok, *ok, Settings{nullptr, nullptr, nullptr, r5.get()}, R, C); },
        // products that wrap round to what the storages hold
        [&] { (void)be.rms_norm(*ok, nullptr, *w, (std::size_t{1} << 63) + 6, 2, 1e-6f); },
        [&] { (void)be.sample(*ok, *ok, {}, (std::size_t{1} << 62) + 1, 4); },
        // other types
        [&] { (void)be.rms_norm(*wide, nullptr, *w, R, C, 1e-6f); },
        [&] { (void)be.quantize_q8(*q, R, C); },
        [&] { (void)be.matmul_q8(Q8{ok, rs, R, C, 16}, a, nullptr); },
        [&] { (void)be.matmul_q8(a, Q8{q, q, R, C, 16}, nullptr); },
        [&] { (void)be.matmul_q8(a, Q8{nullptr, rs, R, C, 16}, nullptr); },
        [&] { (void)be.matmul_q8(a, Q8{q, nullptr, R, C, 16}, nullptr); },
        [&] { (void)be.sample(*ok, *ok, Settings{nullptr, rs.get(), nullptr, nullptr}, R, C); },
        [&] { (void)be.sample(*ok, *ok, Settings{k64.get(), nullptr, nullptr, nullptr}, R, C); },
    };
    const int n = static_cast<int>(calls.size());
    for (int i = 0; i < n && i < most; ++i) status[i] = status_of(calls[i]);
    return n;
}

}  // extern "C"
