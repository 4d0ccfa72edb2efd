// Root-mean-square norm of a residual stream, with the addition before it, and its gradient.
//
//   s = residual + m x / (1 - p),   r = (mean s^2 + eps)^(-1/2),   n = s r,   y = n w
//   c = max |y| / (largest 8-bit value), q = y / c rounded (the 8-bit form)
//   g = dy w,   ds += r (g - n mean(g n)),   dx = m ds / (1 - p),   dw = sum over rows of dy n
//
// Bound by HBM.  A row stays in the registers of the lanes that own it, so everything is read
// once and written once: a wave owns a row of up to 2048 elements (no wait for other waves), a
// workgroup a longer one, and the next row is on its way while one is worked on.  8192 rows of
// 4096, bf16, with a residual: forward 51 us (5.3 TB/s), backward 46 (5.9) and the join of dw 4;
// 16384 rows of 2048 into 8 bits 54 us (4.3); a copy of 2 GiB moves 4.9.  Fewer rows do not fill
// the chip: 1531 of 1001 halves take 9 + 12 + 4.5 us, where 24 MB would take 5.
// The squares are summed in float64, where no 16-bit or float32 value over- or underflows.
// The backward pass reads s as it was rounded for its caller: dw of 16 bits is off by 2.5e-3 (bfloat16)
// where its own rounding is 1.7e-3.  s in float32, or x and the residual in its place, would be a
// tensor more to keep from the forward pass and to read, a quarter of the backward pass's bytes.
// dw: a workgroup takes rows in strides of the grid and sums its columns in registers, the
// workgroups' sums are added in a second launch, always in the same order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_internal.h"
#include "common.h"
#include "philox.h"
#include "rows8.h"

namespace gefen {
namespace {

constexpr int kForwardBlocks = 2048;  // workgroups of a launch
constexpr int kBackwardBlocks = 512;  // and of one that leaves partial sums of dw

struct Params {
    const void *x, *residual, *weight, *grad_y, *grad_sum;
    void *sum, *y, *grad_x, *grad_residual, *grad_weight;
    float *scales, *rstd, *partial;
    int64_t rows, width, x_stride, residual_stride, grad_y_stride, grad_sum_stride;
    double eps;
    Dropout drop;
    int32_t out8;  // GEFEN_RMS_*
};

// LANES threads own a row (64: a wave, and a workgroup of four takes four rows), CHUNKS times
// eight elements each.
template <int LANES_, int CHUNKS_>
struct Shape {
    static constexpr int LANES = LANES_, CHUNKS = CHUNKS_;
    static constexpr int THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    static constexpr int WIDTH = LANES * CHUNKS * 8;
    // 16 waves on a CU leave 128 registers a lane: no row is loaded ahead and the weight is read again
    static constexpr bool LEAN = LANES == 1024;
};

// The sum over the lanes of a row.  slot: LDS for a value of each wave.
template <int LANES, typename V>
__device__ __forceinline__ V row_sum(V v, V* slot) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; ++w) v += slot[w];
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ float row_max(float v, float* slot) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = nanmax(v, __shfl_xor(v, off, 64));
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; ++w) v = nanmax(v, slot[w]);
    }
    return v;
}

// Eight values over scale as 8-bit floating point, the largest ones clamped.  What is rounded is
// the float32 quotient: a product with inv = 1 / scale crosses a middle between two values of the
// format now and then.  NEAR (scale is finite, and not so small that what follows underflows): that
// product, and what it is off by, exact or nearly so in one fused operation, times inv once more;
// it differs from the quotient where that lies within 2^-22 steps of float32 of a middle between
// two of those.  16384 rows of 2048: 53 to 54 us, 57 with a division, 51 with the product alone.
template <bool NEAR>
__device__ __forceinline__ uint64_t eight_bits(const float* v, float scale, float inv, bool e5m2) {
    const float most = e5m2 ? 57344.0f : 448.0f;
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = v[4 * h + i];
            if constexpr (NEAR) {
                const float q = a * inv;
                a = __builtin_fmaf(-__builtin_fmaf(q, scale, -a), inv, q);  // this way round -0 stays
            } else {
                a /= scale;
            }
            t[i] = a != a ? a : fminf(fmaxf(a, -most), most);
        }
        int w = 0;
        if (e5m2) {
            w = __builtin_amdgcn_cvt_pk_bf8_f32(t[0], t[1], w, false);
            w = __builtin_amdgcn_cvt_pk_bf8_f32(t[2], t[3], w, true);
        } else {
            w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], w, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
        }
        out[h] = (uint32_t)w;
    }
    return (uint64_t)out[1] << 32 | out[0];
}

template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS) k_rms_forward(Params a) {
    __shared__ double slots[S::THREADS / 64];
    __shared__ float slots_max[S::THREADS / 64];
    const int lane = threadIdx.x % S::LANES;
    const int width = (int)a.width;
    const uint64_t seed = a.drop.cut ? dropout_seed(a.drop) : 0;
    Eight<T> w[S::CHUNKS];
    auto load_weight = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8;
            if (at < width) w[c].load(static_cast<const T*>(a.weight) + at, width - at);
        }
    };
    if (!S::LEAN) load_weight();
    const int64_t step = (int64_t)gridDim.x * S::ROWS;
    int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / S::LANES;
    Eight<T> x[S::CHUNKS], r[S::CHUNKS];  // of the next row, on its way while this one is worked on
    auto load = [&](int64_t at_row) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0 || at_row >= a.rows) continue;
            x[c].load(static_cast<const T*>(a.x) + at_row * a.x_stride + at, have);
            if (a.residual) r[c].load(static_cast<const T*>(a.residual) + at_row * a.residual_stride + at, have);
        }
    };
    if (!S::LEAN) load(row);
    for (; row < a.rows; row += step) {
        if (S::LEAN) load(row);
        float s[S::CHUNKS][8];
        double sq = 0.0;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0) continue;
            const uint32_t keep = a.drop.cut ? dropout_keep(a.drop, seed, row * a.width + at) : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = x[c][i];
                if (a.drop.cut) v = dropped(v, keep, i, a.drop.scale);
                if (a.residual) v += r[c][i];
                s[c][i] = v;
                sq = __builtin_fma((double)v, (double)v, sq);
                x[c].set(i, v);
            }
            if (a.sum) x[c].store(static_cast<T*>(a.sum) + row * a.width + at, have);
        }
        if (S::LEAN) load_weight();
        else load(row + step);
        sq = row_sum<S::LANES>(sq, slots);
        const float rstd = (float)(1.0 / sqrt(sq / (double)width + a.eps));
        if (a.rstd && lane == 0) a.rstd[row] = rstd;
        float most = 0.0f;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0) continue;
            Eight<T> y;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[c][i] = s[c][i] * rstd * w[c][i];
                if (i < have) most = nanmax(most, fabsf(s[c][i]));
                y.set(i, s[c][i]);
            }
            if (!a.out8) y.store(static_cast<T*>(a.y) + row * a.width + at, have);
        }
        if (!a.out8) continue;
        most = row_max<S::LANES>(most, slots_max);
        const bool e5m2 = a.out8 == GEFEN_RMS_E5M2;
        // a scale below float32's normal range would have few bits
        float scale = most / (e5m2 ? 57344.0f : 448.0f);
        if (most > 0.0f) scale = fmaxf(scale, 1.17549435e-38f);
        if (lane == 0) a.scales[row] = scale;
        const float by = most == 0.0f ? 1.0f : scale, inv = 1.0f / by;
        const bool near = by >= 0x1p-100f && by < INFINITY;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0) continue;
            const uint64_t q = near ? eight_bits<true>(s[c], by, inv, e5m2) : eight_bits<false>(s[c], by, inv, e5m2);
            uint8_t* out = static_cast<uint8_t*>(a.y) + row * a.width + at;
            if (have >= 8) {
                typedef uint64_t __attribute__((aligned(1))) any_t;
                *reinterpret_cast<any_t*>(out) = q;
            } else {
                for (int i = 0; i < have; ++i) out[i] = (uint8_t)(q >> (8 * i));
            }
        }
    }
}

template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS) k_rms_backward(Params a) {
    __shared__ float slots[S::THREADS / 64];
    __shared__ float columns[S::ROWS > 1 ? (S::ROWS - 1) * S::WIDTH : 1];
    const int lane = threadIdx.x % S::LANES;
    const int width = (int)a.width;
    const uint64_t seed = a.drop.cut ? dropout_seed(a.drop) : 0;
    const float over = 1.0f / (float)width;
    Eight<T> w[S::CHUNKS];
    float dw[S::CHUNKS][8];
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c) {
        const int at = (c * S::LANES + lane) * 8;
        if (at < width) w[c].load(static_cast<const T*>(a.weight) + at, width - at);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[c][i] = 0.0f;
    }
    const int64_t step = (int64_t)gridDim.x * S::ROWS;
    int64_t row = (int64_t)blockIdx.x * S::ROWS + threadIdx.x / S::LANES;
    struct Row {
        Eight<T> s[S::CHUNKS], dy[S::CHUNKS], more[S::CHUNKS];
        float rstd;
    };
    auto load = [&](Row& x, int64_t at_row) __attribute__((always_inline)) {
        if (at_row >= a.rows) return;
        x.rstd = a.rstd[at_row];
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0) continue;
            x.s[c].load(static_cast<const T*>(a.x) + at_row * a.x_stride + at, have);
            x.dy[c].load(static_cast<const T*>(a.grad_y) + at_row * a.grad_y_stride + at, have);
            if (a.grad_sum) x.more[c].load(static_cast<const T*>(a.grad_sum) + at_row * a.grad_sum_stride + at, have);
        }
    };
    Row x, next;
    if (!S::LEAN) load(next, row);
    for (; row < a.rows; row += step) {
        if constexpr (S::LEAN) {
            load(x, row);
        } else {
            x = next;
            load(next, row + step);  // on its way while this one is worked on
        }
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int have = width - (c * S::LANES + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= have) continue;
                const float n = x.s[c][i] * x.rstd, t = x.dy[c][i] * n;
                dot = __builtin_fmaf(t, w[c][i], dot);
                dw[c][i] += t;
            }
        }
        if (!a.grad_x && !a.grad_residual) continue;
        const float mean = row_sum<S::LANES>(dot, slots) * over;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c) {
            const int at = (c * S::LANES + lane) * 8, have = width - at;
            if (have <= 0) continue;
            Eight<T> dx;
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = x.rstd * (x.dy[c][i] * w[c][i] - x.s[c][i] * x.rstd * mean);
                if (a.grad_sum) d[i] += x.more[c][i];
                dx.set(i, d[i]);
            }
            if (a.grad_residual) dx.store(static_cast<T*>(a.grad_residual) + row * a.width + at, have);
            if (a.grad_x) {
                if (a.drop.cut) {
                    const uint32_t keep = dropout_keep(a.drop, seed, row * a.width + at);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dx.set(i, dropped(d[i], keep, i, a.drop.scale));
                }
                dx.store(static_cast<T*>(a.grad_x) + row * a.width + at, have);
            }
        }
    }
    if (!a.partial) return;
    if constexpr (S::ROWS > 1) {
        const int wave = threadIdx.x / S::LANES;
        if (wave > 0) {
#pragma unroll
            for (int c = 0; c < S::CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) columns[(wave - 1) * S::WIDTH + (c * S::LANES + lane) * 8 + i] = dw[c][i];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int c = 0; c < S::CHUNKS; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                for (int k = 0; k < S::ROWS - 1; ++k) dw[c][i] += columns[k * S::WIDTH + (c * S::LANES + lane) * 8 + i];
    }
#pragma unroll
    for (int c = 0; c < S::CHUNKS; ++c) {
        const int at = (c * S::LANES + lane) * 8, have = width - at;
        if (have <= 0) continue;
        Eight<float> out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out.v[i] = dw[c][i];
        out.store(a.partial + blockIdx.x * a.width + at, have);
    }
}

// dw from the workgroups' sums: 32 columns a workgroup, the rows in kSlices of its threads.
constexpr int kSlices = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kSlices) k_rms_join(const float* partial, int blocks, int width, T* out) {
    __shared__ float part[kSlices][33];
    const int lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, slice = threadIdx.x >> 5;
    float sum = 0.0f;
    if (col < width) {
#pragma unroll 4
        for (int b = slice; b < blocks; b += kSlices) sum += partial[(int64_t)b * width + col];
    }
    part[slice][lane] = sum;
    for (int half = kSlices / 2; half > 0; half /= 2) {
        __syncthreads();
        if (slice < half) part[slice][lane] += part[slice + half][lane];
    }
    if (slice == 0 && col < width) out[col] = from_f32<T>(part[0][lane]);
}

// Calls f with the shape that rows of `width` take: a wave a row as long as its elements fit
// the lanes' registers (16384 rows of 2048: 63 us by a workgroup each and not ahead, 51 so), then
// as few lanes as do.
constexpr int kWaveWidth = 2048;
template <typename T, typename F>
int with_shape(int64_t width, F f) {
    if (width <= 512) return f(Shape<64, 1>{});
    if (width <= 1024) return f(Shape<64, 2>{});
    if (width <= kWaveWidth) return f(Shape<64, 4>{});
    if (width <= 4096) return f(Shape<256, 2>{});
    if constexpr (sizeof(T) == 4) {
        if (width <= 8192) return f(Shape<512, 2>{});
        if (width <= 16384) return f(Shape<1024, 2>{});
    } else {
        if (width <= 8192) return f(Shape<256, 4>{});
        if (width <= 16384) return f(Shape<512, 4>{});
    }
    return f(Shape<1024, 4>{});
}
template <typename F>
int with_type(int dtype, F f) {
    if (dtype == GEFEN_F32) return f(float{});
    if (dtype == GEFEN_F16) return f(f16_t{});
    return f(bf16_t{});
}
int blocks_of(int64_t rows, int64_t width, int most) {
    const int64_t each = width <= kWaveWidth ? 4 : 1, want = (rows + each - 1) / each;
    return (int)(want < most ? want : most);
}

int check_task(const gefen_rms_norm_task* t) {
    if (!t) return fail_inval("rms_norm: no task");
    if (!valid_dtype(t->dtype)) return fail_inval("rms_norm: unknown dtype %d", t->dtype);
    if (t->rows < 0 || t->rows >= (int64_t)1 << 40) return fail_inval("rms_norm: rows out of range");
    if (t->width < 1 || t->width > GEFEN_RMS_MAX_WIDTH)
        return fail_inval("rms_norm: width must be 1 to %d, got %lld", GEFEN_RMS_MAX_WIDTH, (long long)t->width);
    if (!(t->eps >= 0.0) || !isfinite(t->eps)) return fail_inval("rms_norm: eps must be finite and not negative");
    if (!(t->dropout >= 0.0 && t->dropout <= 1.0)) return fail_inval("rms_norm: dropout must be in [0, 1]");
    if (!aligned(t->seed_at, 8)) return fail_inval("rms_norm: the seed must be aligned");
    return GEFEN_OK;
}
int check_tensor(const gefen_rms_norm_task& t, const void* p, bool needed, const char* name) {
    if (needed && t.rows && !p) return fail_inval("rms_norm: %s is missing", name);
    if (!aligned(p, dtype_size(t.dtype))) return fail_inval("rms_norm: %s must be aligned to its elements", name);
    return GEFEN_OK;
}
Params params_of(const gefen_rms_norm_task& t) {
    Params a{};
    a.x = t.x;
    a.residual = t.residual;
    a.weight = t.weight;
    a.grad_y = t.grad_y;
    a.grad_sum = t.grad_sum;
    a.sum = t.sum;
    a.y = t.y;
    a.grad_x = t.grad_x;
    a.grad_residual = t.grad_residual;
    a.grad_weight = t.grad_weight;
    a.scales = t.scales;
    a.rstd = t.rstd;
    a.rows = t.rows;
    a.width = t.width;
    a.x_stride = t.x_row_stride;
    a.residual_stride = t.residual_row_stride;
    a.grad_y_stride = t.grad_y_row_stride;
    a.grad_sum_stride = t.grad_sum_row_stride;
    a.eps = t.eps;
    a.out8 = t.out;
    dropout_of(t.dropout, t.seed_at, t.seed, t.offset, &a.drop);
    return a;
}

}  // namespace
}  // namespace gefen

using namespace gefen;

extern "C" size_t gefen_rms_norm_backward_workspace_size(const gefen_rms_norm_task* task) {
    if (check_task(task) != GEFEN_OK) return 0;
    return (size_t)blocks_of(task->rows, task->width, kBackwardBlocks) * task->width * 4 + 16;
}

extern "C" int gefen_rms_norm_forward(const gefen_rms_norm_task* task, gefen_stream_t stream) {
    if (int rc = check_task(task)) return rc;
    const gefen_rms_norm_task& t = *task;
    if (t.out < GEFEN_RMS_SAME || t.out > GEFEN_RMS_E5M2) return fail_inval("rms_norm: unknown output %d", t.out);
    if (int rc = check_tensor(t, t.x, true, "x")) return rc;
    if (int rc = check_tensor(t, t.residual, false, "residual")) return rc;
    if (int rc = check_tensor(t, t.weight, true, "weight")) return rc;
    if (int rc = check_tensor(t, t.sum, false, "sum")) return rc;
    if (t.rows && !t.y) return fail_inval("rms_norm: y is missing");
    if (t.out == GEFEN_RMS_SAME && !aligned(t.y, dtype_size(t.dtype)))
        return fail_inval("rms_norm: y must be aligned to its elements");
    if (t.rows && t.out != GEFEN_RMS_SAME && !t.scales) return fail_inval("rms_norm: scales are missing");
    if (!aligned(t.scales, 4) || !aligned(t.rstd, 4)) return fail_inval("rms_norm: scales and rstd must be aligned");
    if (t.rows == 0) return GEFEN_OK;
    const Params a = params_of(t);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return with_type(t.dtype, [&](auto v) {
        using T = decltype(v);
        return with_shape<T>(t.width, [&](auto s) {
            using S = decltype(s);
            k_rms_forward<T, S><<<blocks_of(t.rows, t.width, kForwardBlocks), S::THREADS, 0, st>>>(a);
            return launch_status("rms_norm");
        });
    });
}

extern "C" int gefen_rms_norm_backward(const gefen_rms_norm_task* task, void* workspace, size_t workspace_bytes,
                                       gefen_stream_t stream) {
    if (int rc = check_task(task)) return rc;
    const gefen_rms_norm_task& t = *task;
    if (int rc = check_tensor(t, t.x, true, "x")) return rc;
    if (int rc = check_tensor(t, t.weight, true, "weight")) return rc;
    if (int rc = check_tensor(t, t.grad_y, true, "grad_y")) return rc;
    if (int rc = check_tensor(t, t.grad_sum, false, "grad_sum")) return rc;
    if (int rc = check_tensor(t, t.grad_x, false, "grad_x")) return rc;
    if (int rc = check_tensor(t, t.grad_residual, false, "grad_residual")) return rc;
    if (int rc = check_tensor(t, t.grad_weight, false, "grad_weight")) return rc;
    if ((t.rows && !t.rstd) || !aligned(t.rstd, 4)) return fail_inval("rms_norm: rstd must be aligned float32 memory");
    if (t.grad_weight && (!workspace || !aligned(workspace, 16) ||
                          workspace_bytes < gefen_rms_norm_backward_workspace_size(task)))
        return fail_inval("rms_norm: workspace too small, missing or not aligned to 16 bytes");
    Params a = params_of(t);
    a.partial = t.grad_weight ? static_cast<float*>(workspace) : nullptr;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return with_type(t.dtype, [&](auto v) {
        using T = decltype(v);
        const int blocks = blocks_of(t.rows, t.width, kBackwardBlocks);
        if (t.rows && (a.grad_x || a.grad_residual || a.partial)) {
            const int rc = with_shape<T>(t.width, [&](auto s) {
                using S = decltype(s);
                k_rms_backward<T, S><<<blocks, S::THREADS, 0, st>>>(a);
                return launch_status("rms_norm");
            });
            if (rc) return rc;
        }
        if (a.partial) {
            k_rms_join<T><<<(uint32_t)((t.width + 31) / 32), 32 * kSlices, 0, st>>>(a.partial, blocks, (int)t.width,
                                                                           static_cast<T*>(a.grad_weight));
            return launch_status("rms_norm");
        }
        return (int)GEFEN_OK;
    });
}
