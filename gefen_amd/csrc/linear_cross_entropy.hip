// Softmax cross entropy of an output matrix, with its gradients, without the logits.
//
//   l[n, v] = h_n . W_v,  lse_n = log sum_v exp l[n, v]
//   loss_n  = lse_n - (1 - e) l[n, y_n] - (e / V) sum_v l[n, v]
//   G[n, v] = exp(l[n, v] - lse_n) - (1 - e) [v = y_n] - e / V
//   dh = c G W,   dW = c G^T h        (c: the loss's gradient, over the count for a mean)
//
// Three MFMA products (lce_gemm.h) with float32 accumulation, 6 N V D operations:
// the kernels are bound by the matrix cores once N is in the hundreds, and by reading
// W for a few rows.
//
// * Positions whose target is ignore_index take no part: the rows that count are
//   gathered first (k_rows, k_pack), so a masked prompt costs nothing and whatever it
//   holds (NaN included) reaches nothing.
// * The logits' product keeps, for every row and slot of 64 columns, the slot's
//   maximum m and sum of exp(l - m), both float32, and when gradients are wanted
//   exp(l - m) itself in 16 bits: an unsigned format of its own with three significant
//   bits more than bf16 (two more than half), so that G is in effect rounded once.
// * One pass over those values turns them into G (k_gradient_rows): a row's lse comes
//   from its slots, and exp(m - lse) scales each slot.  The target's entry is formed in
//   float32 from its own logit, so that p - 1 of a confident row does not cancel in
//   16 bits.  Rounding G to the operands' type is the one rounding below float32 on the
//   way to the gradients: its errors are independent between the many terms of each sum
//   and stay below that of the gradients' own rounding.
// * For few rows one term can be most of a sum, and the products wait for W or dW
//   anyway: G is then two planes, twice the type's bits (kTwoPlaneRows).
// * Rows are taken in pieces whose G fits a bounded workspace; the logits of a piece
//   exist only as these 16-bit values, and never all of them at once when the
//   positions do not fit.  dW is summed over the pieces in float32.
//
// A half-precision G is scaled by 2^15 (and its products by 2^-15), which keeps
// probabilities down to 1e-9 out of half's subnormals.  float32 runs as two half planes
// per operand and three products, each matrix scaled by the power of two that brings its
// largest finite element to 2^14: elements keep 22 bits down to 2^-29 of the largest
// one, at five times the rate of the float32 matrix instructions.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_internal.h"
#include "common.h"
#include "lce_gemm.h"

namespace gefen {
namespace lce {

constexpr float kHalfScale = 32768.0f;  // of a half-precision G
constexpr int kSlot = 64;               // columns that share a maximum
constexpr int kRowAlign = 256;          // rows of a piece, columns of G
constexpr int kMaxVocab = 4 << 20;      // 256 rows of G within 2^31 bytes
constexpr int kMaxWidth = 1 << 20;

// Device scalars of a call.
struct Meta {
    int32_t count;    // rows that take part
    float grad_max;   // largest |gradient| of a row (per-row gradients)
    uint32_t top[2];  // float32: largest finite magnitude of hidden and weight, as bits
};

__device__ __forceinline__ int piece_rows(const Meta* m, int from, int most) {
    return max(0, min(m->count - from, most));
}

__device__ __forceinline__ int64_t target_at(const void* t, int is32, int64_t n) {
    return is32 ? (int64_t) static_cast<const int32_t*>(t)[n] : static_cast<const int64_t*>(t)[n];
}

// map = the rows that take part, in order, then the ignored ones; targets in that
// order (-1: not a column, whose loss is NaN).  One workgroup.
constexpr int kRowsThreads = 1024;
__global__ __launch_bounds__(kRowsThreads) void k_rows(const void* __restrict__ targets, int is32, int n, int v,
                                                       int64_t ignore, const float* __restrict__ row_grad,
                                                       int32_t* __restrict__ map, int32_t* __restrict__ tgt,
                                                       Meta* __restrict__ meta) {
    __shared__ int wave_sum[kRowsThreads / 64];
    __shared__ float wave_max[kRowsThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;  // rows that take part before this stretch
    float gmax = 0.0f;
    for (int at = 0; at < n; at += kRowsThreads) {
        const int i = at + (int)threadIdx.x;
        const int64_t y = i < n ? target_at(targets, is32, i) : ignore;
        const bool live = i < n && y != ignore;
        const uint64_t ball = __ballot(live);
        const int before = __popcll(ball & ((1ull << lane) - 1ull));
        if (lane == 0) wave_sum[wave] = __popcll(ball);
        __syncthreads();
        int off = 0, all = 0;
        for (int w = 0; w < kRowsThreads / 64; ++w) {
            if (w < wave) off += wave_sum[w];
            all += wave_sum[w];
        }
        if (live) {
            map[base + off + before] = i;
            tgt[base + off + before] = (y >= 0 && y < v) ? (int)y : -1;
            if (row_grad) gmax = nanmax(gmax, fabsf(row_grad[i]));
        } else if (i < n) {
            map[n - 1 - (i - base - off - before)] = i;
        }
        base += all;
        __syncthreads();
    }
    for (int off = 32; off > 0; off >>= 1) gmax = nanmax(gmax, __shfl_xor(gmax, off, 64));
    if (lane == 0) wave_max[wave] = gmax;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowsThreads / 64; ++w) gmax = nanmax(gmax, wave_max[w]);
        meta->count = base;
        meta->grad_max = gmax;
        meta->top[0] = meta->top[1] = 0;
    }
}

// x (scaled into half's range) as a half and what it leaves times kLowScale.
__device__ __forceinline__ void split_half(float x, uint16_t* hi, uint16_t* lo) {
    const f16_t h = from_f32<f16_t>(x);
    *hi = h.bits;
    // what is not finite has no remainder worth adding: inf - inf is NaN
    *lo = (h.bits & 0x7c00) == 0x7c00 ? 0 : from_f32<f16_t>((x - to_f32(h)) * kLowScale).bits;
}
__device__ __forceinline__ void split_bf16(float x, uint16_t* hi, uint16_t* lo) {
    const bf16_t h = from_f32<bf16_t>(x);
    *hi = h.bits;
    *lo = (h.bits & 0x7f80) == 0x7f80 ? 0 : from_f32<bf16_t>(x - to_f32(h)).bits;
}

// exp(l - m) in [0, 1] as 16 unsigned bits on its way to G: 4 exponent and 12 mantissa
// bits for a half G, 6 and 10 for a bf16 one, with subnormals.  The float's own exponent
// is brought down by a product with a power of two (subnormal results are rounded by the
// hardware), and the mantissa is rounded to nearest.  Relative error 2^-13 down to 2^-14
// (bf16: 2^-11 down to 2^-62), 2^-27 absolute below.
template <bool F16>
__device__ __forceinline__ uint16_t pack_exp(float e) {
    constexpr int drop = F16 ? 11 : 13;
    const uint32_t u = __float_as_uint(e * (F16 ? 0x1p-112f : 0x1p-64f));
    return (uint16_t)((u + ((1u << (drop - 1)) - 1) + ((u >> drop) & 1u)) >> drop);
}
template <bool F16>
__device__ __forceinline__ float unpack_exp(uint16_t x) {
    return __uint_as_float((uint32_t)x << (F16 ? 11 : 13)) * (F16 ? 0x1p112f : 0x1p64f);
}

// Exponent that brings a matrix's largest finite magnitude (its bits in `top`) to 2^14.
__device__ __forceinline__ int half_exponent(uint32_t top) {
    return top == 0 ? 0 : 14 - max((int)(top >> 23) - 127, -112);
}

// meta->top[which] = the largest finite magnitude of a float32 matrix, as its bits; with
// a map, of the rows that take part.  Maxima of integers: any order gives the same.
struct Top {
    const float* src;
    int64_t row_stride, col_stride;
    int32_t n, d;
    const int32_t* map;
    Meta* meta;
    int32_t which;
};
__global__ __launch_bounds__(256) void k_top(const Top t) {
    const int rows = t.map ? t.meta->count : t.n;
    uint32_t top = 0;
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* s = t.src + (int64_t)(t.map ? t.map[r] : r) * t.row_stride;
        for (int c = threadIdx.x; c < t.d; c += 256) {
            const uint32_t u = abs_key(s[(int64_t)c * t.col_stride]);
            top = u < 0x7f800000u && u > top ? u : top;
        }
    }
    top = wave_group_max_u32(top, 64);
    if ((threadIdx.x & 63) == 0) atomicMax(&t.meta->top[t.which], top);
}

// Rows of a matrix of any strides as the products read them: dp = D rounded up to 64
// columns, zero-padded, one plane or those of a float32 operand, scaled.  With a map: row r is src row map[r]
// for r < meta->count and zero up to the next multiple of kRowAlign, and the rows that
// take no part get a zero gradient and a zero loss.
constexpr int kPackPlanes = 3;  // of a float32 operand: high, low, high where finite
struct Pack {
    const void* src;
    int64_t row_stride, col_stride;
    int32_t n, d, dp;
    int32_t f32;
    uint16_t* dst;
    int64_t plane;
    const int32_t* map;
    const Meta* meta;
    int32_t which;      // float32: whose largest magnitude in meta->top
    void* zero_rows;    // [n, d] gradient, rows of d elements of `size` bytes (may be null)
    float* zero_losses;  // [n] (may be null)
};
__global__ __launch_bounds__(256) void k_pack(const Pack p) {
    const int r = blockIdx.x;
    int64_t row = r;
    bool live = r < p.n;
    if (p.map) {
        const int count = p.meta->count;
        live = r < count;
        if (r < p.n) row = p.map[r];
        if (!live && r < p.n) {
            if (p.zero_losses && threadIdx.x == 0 && blockIdx.y == 0) p.zero_losses[row] = 0.0f;
            if (p.zero_rows) {
                const int col = (int)(blockIdx.y * 256 + threadIdx.x) * 8;
                for (int e = col; e < min(col + 8, p.d); ++e) {
                    if (p.f32) static_cast<float*>(p.zero_rows)[row * p.d + e] = 0.0f;
                    else static_cast<uint16_t*>(p.zero_rows)[row * p.d + e] = 0;
                }
            }
        }
        if (r >= (count + kRowAlign - 1) / kRowAlign * kRowAlign) return;
    }
    const int c0 = (int)(blockIdx.y * 256 + threadIdx.x) * 8;
    if (c0 >= p.dp) return;
    uint16_t out[kPackPlanes][8] = {};
    if (live) {
        if (p.f32) {
            const int ex = half_exponent(p.meta->top[p.which]);
            const float* s = static_cast<const float*>(p.src) + row * p.row_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e < p.d) {
                    split_half(ldexpf(s[(int64_t)(c0 + e) * p.col_stride], ex), &out[0][e], &out[1][e]);
                    out[2][e] = (out[0][e] & 0x7c00) == 0x7c00 ? 0 : out[0][e];
                }
        } else {
            const uint16_t* s = static_cast<const uint16_t*>(p.src) + row * p.row_stride;
            if (p.col_stride == 1 && c0 + 8 <= p.d) {
                const AnyVec<uint16_t, 8> x = *reinterpret_cast<const AnyVec<uint16_t, 8>*>(s + c0);
#pragma unroll
                for (int e = 0; e < 8; ++e) out[0][e] = x.v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c0 + e < p.d) out[0][e] = s[(int64_t)(c0 + e) * p.col_stride];
            }
        }
    }
    const int planes = p.f32 ? kPackPlanes : 1;
    for (int k = 0; k < planes; ++k) {
        Vec<uint16_t, 8> x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] = out[k][e];
        vstore(p.dst + k * p.plane, (int64_t)r * p.dp + c0, x);
    }
}

// The logits' product of a piece of rows and what is kept of it.
struct Logits {
    Operand w, x;       // w: [V, dp] K-major, x: the piece's rows [.., dp] K-major
    int32_t v, steps, segs, tiles_m, from, most;  // steps of BK; the piece is rows [from, from + most)
    int32_t slots;      // per row
    float2* stats;      // [row][slot]: maximum, sum of exp(l - maximum)
    float* sums;        // [row][slot]: sum of l (null without label smoothing)
    float* target_logit;  // [row], over all pieces
    const int32_t* tgt;
    const Meta* meta;
    uint16_t* g;        // [row][ldg] exp(l - slot maximum), packed or in two planes (null: loss only)
    int64_t ldg, g_plane;
    int32_t planes, f32;
};

template <typename C>
__global__ __launch_bounds__(C::TT, C::EU) void k_logits(const Logits a) {
    constexpr int WI = C::WI, WJ = C::WJ;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[C::NST * C::STAGE];
    const int rows = piece_rows(a.meta, a.from, a.most);
    const int tiles_n = (rows + C::TN - 1) / C::TN;
    const int live = tiles_n * a.tiles_m;
    if ((int)blockIdx.x >= live) return;
    int ti, tj;
    tile_of<C::GROUP_M>(logical_block(blockIdx.x, live), a.tiles_m, tiles_n, &ti, &tj);
    const int m0 = ti * C::TM, n0 = tj * C::TN;
    f32x4 acc[WI][WJ];
    product_tile<C>(a.w, a.x, m0, n0, 0, a.steps, a.segs, smem, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = m0 + (wave / C::WAVES_N) * C::WM, wn = n0 + (wave % C::WAVES_N) * C::WN;
    const int hi = 4 * (lane >> 4);
    const int slot = wm / kSlot;
    static_assert(C::WM == kSlot, "a wave's columns are a slot");
    if (wm >= a.v && !a.g) return;
    const int ex = a.f32 ? -half_exponent(a.meta->top[0]) - half_exponent(a.meta->top[1]) : 0;
    const bool part = wm + C::WM > a.v;  // the last columns end inside this wave's
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        const int n = wn + j * 16 + (lane & 15);
        float m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (a.f32) acc[i][j][r] = ldexpf(acc[i][j][r], ex);
                if (part && wm + i * 16 + hi + r >= a.v) acc[i][j][r] = -INFINITY;
                m = fmaxf(m, acc[i][j][r]);  // skips NaN, which the sum of exp keeps
            }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (a.sums) {
#pragma unroll
            for (int i = 0; i < WI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += !part || wm + i * 16 + hi + r < a.v ? acc[i][j][r] : 0.0f;
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
        }
        const int y = n < rows ? a.tgt[a.from + n] - wm : -1;
        if (y >= 0 && y < C::WM && (y & 12) == hi) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < WI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (i * 16 + hi + r == y) t = acc[i][j][r];
            a.target_logit[a.from + n] = t;
        }
        // a slot of no finite value: exp(-inf - 0) = 0
        const float ref = m == -INFINITY ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = acc[i][j][r] - ref;
                acc[i][j][r] = a.f32 ? expf(x) : __expf(x);
                s += acc[i][j][r];
            }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (n < rows && lane < 16 && wm < a.v) {
            const int64_t at = (int64_t)n * a.slots + slot;
            a.stats[at] = make_float2(m, s);
            if (a.sums) a.sums[at] = sum;
        }
        if (!a.g) continue;
        // rows past the piece's end stay inside the workspace (it holds whole tiles)
        uint16_t* row = a.g + (int64_t)n * a.ldg + wm + hi;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            uint16_t o[2][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = acc[i][j][r];
                if (a.planes == 1) o[0][r] = pack_exp<C::F16>(e);
                else if constexpr (C::F16) split_half(e * kHalfScale, &o[0][r], &o[1][r]);
                else split_bf16(e, &o[0][r], &o[1][r]);
            }
            for (int k = 0; k < a.planes; ++k)
                *reinterpret_cast<uint2*>(row + i * 16 + k * a.g_plane) =
                    make_uint2((uint32_t)o[k][0] | ((uint32_t)o[k][1] << 16),
                               (uint32_t)o[k][2] | ((uint32_t)o[k][3] << 16));
        }
    }
}

// Loss of each row from its slots, and (g) the row's values turned into G.
struct Rows {
    const float2* stats;
    const float* sums;
    const float* target_logit;
    const int32_t* tgt;
    const int32_t* map;
    const Meta* meta;
    const float* row_grad;  // gradient of each row's loss (null: one for all)
    float* losses;          // [n], original order
    uint16_t* g;
    int64_t ldg, g_plane;
    int32_t v, slots, from, most, planes;
    float smoothing;
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
    const float m = nanmax(a.x, b.x);
    const float ref = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * expf(a.x - ref) + b.y * expf(b.x - ref));
}

constexpr int kGradThreads = 256;
template <bool F16>
__global__ __launch_bounds__(kGradThreads) void k_gradient_rows(const Rows a) {
    __shared__ float2 part[kGradThreads / 64];
    __shared__ float part_sum[kGradThreads / 64];
    const int r = blockIdx.x;
    const int rows = piece_rows(a.meta, a.from, a.most);
    const int chunks = (int)(a.ldg / 8);
    if (r >= rows) {  // zero rows up to the end of the last K step of dW
        if (!a.g || r >= (rows + 63) / 64 * 64) return;
        Vec<uint16_t, 8> z = {};
        for (int k = 0; k < a.planes; ++k)
            for (int c = blockIdx.y * kGradThreads + threadIdx.x; c < chunks; c += gridDim.y * kGradThreads)
                vstore(a.g + k * a.g_plane, (int64_t)r * a.ldg + c * 8, z);
        return;
    }
    float2 st = make_float2(-INFINITY, 0.0f);
    float sum = 0.0f;
    const float2* stats = a.stats + (int64_t)r * a.slots;
    for (int s = threadIdx.x; s < a.slots; s += kGradThreads) {
        st = join_stats(st, stats[s]);
        if (a.sums) sum += a.sums[(int64_t)r * a.slots + s];
    }
    for (int off = 32; off > 0; off >>= 1) {
        st = join_stats(st, make_float2(__shfl_xor(st.x, off, 64), __shfl_xor(st.y, off, 64)));
        sum += __shfl_xor(sum, off, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = st;
        part_sum[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    st = part[0];
    sum = part_sum[0];
    for (int w = 1; w < kGradThreads / 64; ++w) {
        st = join_stats(st, part[w]);
        sum += part_sum[w];
    }
    const float lse = st.x + logf(st.y);
    const int y = a.tgt[a.from + r];
    const float tl = y >= 0 ? a.target_logit[a.from + r] : NAN;
    const float e = a.smoothing;
    const int64_t n = a.map[a.from + r];
    if (a.losses && blockIdx.y == 0 && threadIdx.x == 0) {
        // (1 - e) (lse - l_y) + e (lse - mean l): the first difference is exact to a rounding
        float loss = (1.0f - e) * (lse - tl);
        if (e > 0.0f) loss += e * (lse - sum / (float)a.v);
        a.losses[n] = loss;
    }
    if (!a.g) return;
    float w = F16 ? kHalfScale : 1.0f;
    if (a.row_grad) {
        const float g = a.row_grad[n], top = a.meta->grad_max;
        w *= top == 0.0f ? 0.0f : g / top;
    }
    const float unit = e > 0.0f ? e / (float)a.v : 0.0f;
    if (y < 0) w = NAN;
    // the target's entry from its own logit: p - 1 without cancellation in 16 bits
    const float at_target = expm1f(tl - lse) + e - unit;
    const float back = F16 && a.planes == 2 ? 1.0f / kHalfScale : 1.0f;
    for (int c = blockIdx.y * kGradThreads + threadIdx.x; c < chunks; c += gridDim.y * kGradThreads) {
        const int v0 = c * 8;
        uint16_t* p = a.g + (int64_t)r * a.ldg + v0;
        Vec<uint16_t, 8> x[2];
        if (v0 >= a.v) {
            x[0] = x[1] = Vec<uint16_t, 8>{};
        } else {
            const float f = expf(stats[v0 / kSlot].x - lse) * back;
            for (int k = 0; k < a.planes; ++k) x[k] = vload<uint16_t, 8>(p + k * a.g_plane, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float q;
                if (a.planes == 1) q = F16 ? unpack_exp<true>(x[0].v[i]) : unpack_exp<false>(x[0].v[i]);
                else if (F16) q = to_f32(f16_t{x[0].v[i]}) + to_f32(f16_t{x[1].v[i]}) * (1.0f / kLowScale);
                else q = to_f32(bf16_t{x[0].v[i]}) + to_f32(bf16_t{x[1].v[i]});
                q = q * f - unit;
                if (v0 + i == y) q = at_target;
                q = v0 + i < a.v ? q * w : 0.0f;
                if (a.planes == 1) x[0].v[i] = F16 ? from_f32<f16_t>(q).bits : from_f32<bf16_t>(q).bits;
                else if (F16) split_half(q, &x[0].v[i], &x[1].v[i]);
                else split_bf16(q, &x[0].v[i], &x[1].v[i]);
            }
        }
        for (int k = 0; k < a.planes; ++k) vstore(p + k * a.g_plane, 0, x[k]);
    }
}

// The sum of the rows' losses in float64, over the count for a mean (0 / 0 = NaN
// where no row takes part, as the mean of nothing is).
__global__ __launch_bounds__(1024) void k_loss(const float* __restrict__ losses, int n, const Meta* __restrict__ meta,
                                               int mean, float* __restrict__ out) {
    __shared__ double part[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += (double)losses[i];
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += part[w];
        *out = (float)(mean ? s / (double)meta->count : s);
    }
}

// A gradient's product: out[n, m] = factor * (prev[n, m] + sum_k A[m, k] B[n, k]) for
// m < D, rows n of the piece (dh, through the map) or of the vocabulary (dW).
struct Grad {
    Operand a, b;
    int32_t d, tiles_m, steps, segs, splits;
    int32_t n;              // rows of the result (dW: V); dh: the piece's, from meta
    int32_t dh;             // dh: rows through the map, all of K; dW: K = the piece's rows
    int32_t from, most;
    const int32_t* map;
    const Meta* meta;
    const float* grad;      // gradient of the loss (null: 1)
    int32_t mean, by_row;   // by_row: G is scaled by 1 / meta->grad_max
    float* parts;           // [splits][n][d] float32 (splits > 1), to be joined by k_join
    float* sum;             // running float32 sum over the pieces (null: one piece)
    int32_t first, last;    // piece of the sum
    void* out;
    int32_t dtype;
};

__device__ __forceinline__ float grad_factor(const Grad& g) {
    float f = g.dtype == GEFEN_BF16 ? 1.0f : 1.0f / kHalfScale;
    if (g.dtype == GEFEN_F32) f = ldexpf(f, -half_exponent(g.meta->top[g.dh ? 1 : 0]));
    if (g.by_row) return f * g.meta->grad_max;
    if (g.grad) f *= *g.grad;
    if (g.mean) f = g.meta->count ? f / (float)g.meta->count : 0.0f;
    return f;
}
// four results of row n from column m: cnt of them are inside
__device__ __forceinline__ void finish(const Grad& g, int64_t row, int64_t n, int m, float v[4], float factor) {
    const int cnt = min(4, g.d - m);
    if (g.sum) {
        float* s = g.sum + n * g.d + m;
        for (int e = 0; e < cnt; ++e) {
            if (!g.first) v[e] += s[e];
            if (!g.last) s[e] = v[e];
        }
        if (!g.last) return;
    }
    const int64_t at = row * g.d + m;
    if (g.dtype == GEFEN_F32) {
        float* o = static_cast<float*>(g.out) + at;
        if (cnt == 4) *reinterpret_cast<AnyVec<float, 4>*>(o) = AnyVec<float, 4>{{v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor}};
        else for (int e = 0; e < cnt; ++e) o[e] = v[e] * factor;
    } else {
        AnyVec<uint16_t, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x.v[e] = g.dtype == GEFEN_F16 ? from_f32<f16_t>(v[e] * factor).bits : from_f32<bf16_t>(v[e] * factor).bits;
        uint16_t* o = static_cast<uint16_t*>(g.out) + at;
        if (cnt == 4) *reinterpret_cast<AnyVec<uint16_t, 4>*>(o) = x;
        else for (int e = 0; e < cnt; ++e) o[e] = x.v[e];
    }
}

template <typename C>
__global__ __launch_bounds__(C::TT, C::EU) void k_grad(const Grad g) {
    constexpr int WI = C::WI, WJ = C::WJ;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[C::NST * C::STAGE];
    const int rows = piece_rows(g.meta, g.from, g.most);
    const int n_all = g.dh ? rows : g.n;
    const int tiles_n = (n_all + C::TN - 1) / C::TN;
    const int live = tiles_n * g.tiles_m * g.splits;
    if ((int)blockIdx.x >= live) return;
    const int lb = logical_block(blockIdx.x, live);
    const int split = lb / (tiles_n * g.tiles_m);
    int ti, tj;
    tile_of<C::GROUP_M>(lb - split * tiles_n * g.tiles_m, g.tiles_m, tiles_n, &ti, &tj);
    const int m0 = ti * C::TM, n0 = tj * C::TN;
    const int steps = g.dh ? g.steps : (rows + C::BK - 1) / C::BK;
    const int k0 = (int)((int64_t)steps * split / g.splits), k1 = (int)((int64_t)steps * (split + 1) / g.splits);
    f32x4 acc[WI][WJ];
    product_tile<C>(g.a, g.b, m0, n0, k0, k1, g.segs, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = m0 + (wave / C::WAVES_N) * C::WM, wn = n0 + (wave % C::WAVES_N) * C::WN;
    const float factor = grad_factor(g);
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        const int n = wn + j * 16 + (lane & 15);
        if (n >= n_all) continue;
        const int64_t row = g.dh ? g.map[g.from + n] : n;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int m = wm + i * 16 + 4 * (lane >> 4);
            if (m >= g.d) continue;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r];
            if (g.parts) {
                float* p = g.parts + ((int64_t)split * n_all + n) * g.d + m;
                for (int e = 0; e < min(4, g.d - m); ++e) p[e] = v[e];
            } else {
                finish(g, row, n, m, v, factor);
            }
        }
    }
}

// The splits of a product added up in order.
__global__ __launch_bounds__(256) void k_join(const Grad g) {
    const int n_all = g.dh ? piece_rows(g.meta, g.from, g.most) : g.n;
    const int per = (g.d + 3) / 4;
    const float factor = grad_factor(g);
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < (int64_t)n_all * per; q += (int64_t)gridDim.x * 256) {
        const int64_t n = q / per;
        const int m = (int)(q - n * per) * 4;
        const int cnt = min(4, g.d - m);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < g.splits; ++s) {
            const float* p = g.parts + ((int64_t)s * n_all + n) * g.d + m;
            for (int e = 0; e < cnt; ++e) v[e] += p[e];
        }
        finish(g, g.dh ? g.map[g.from + n] : n, n, m, v, factor);
    }
}

// ------------------------------------------------------------------ host side
namespace {

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

template <bool F16> using LogitsBig = Cfg<F16, 256, 256, 64, 128, 64, 2, false, false, 4>;
template <bool F16> using LogitsSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, false, false, 4>;
template <bool F16> using LogitsRow = Cfg<F16, 256, 32, 64, 32, 64, 4, false, false, 4>;
template <bool F16> using HiddenBig = Cfg<F16, 256, 256, 64, 128, 64, 2, true, false, 8>;
template <bool F16> using HiddenSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, true, false, 8>;
template <bool F16> using WeightBig = Cfg<F16, 256, 256, 128, 64, 64, 2, true, true, 4>;
template <bool F16> using WeightSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, true, true, 4>;

// Rows up to which G has two planes.  The gradients' products of so few rows take the
// time of reading W and writing dW (4 V D bytes at 5 TB/s) rather than of their
// 8 n V D operations (at 1.2 PFLOP/s: n = 120).
constexpr int kTwoPlaneRows = 64;

enum LogitsTile { kRowTile, kSmallTile, kBigTile };

// How a call runs: fixed by its sizes, types, alignment and workspace.
struct Plan {
    int n, v, d, dtype;
    bool train, dh, dw, pack_w, smooth;
    int planes;         // of G
    bool halves;        // products of half-precision operands
    int64_t dp, ldg;
    int rows, pieces;   // rows of a piece
    LogitsTile tile;
    int slots;
    bool dh_big, dw_big;
    int dh_splits, dw_splits;
    // byte offsets into the workspace
    size_t o_meta, o_map, o_tgt, o_tlogit, o_losses, o_x, o_w, o_stats, o_sums, o_g, o_wsum, o_parts, bytes;
};

// Workgroups that fill the chip: one big tile or two small ones per CU.
constexpr int kCus = 256;

void split_rule(int64_t m, int64_t n, int64_t steps, bool* big, int* splits) {
    const int64_t tb = up(m, 256) / 256 * (up(n, 256) / 256), ts = up(m, 128) / 128 * (up(n, 128) / 128);
    *big = tb >= kCus / 2 || (m >= 256 && n >= 256 && tb * steps >= kCus * 8);
    const int64_t tiles = *big ? tb : ts, room = *big ? kCus : 2 * kCus;
    int64_t s = room / tiles;
    if (s > steps / 4) s = steps / 4;  // at least four K steps of work per part
    *splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

int make_plan(const gefen_linear_cross_entropy_task& t, Plan* p, const char* what) {
    if (t.n < 0 || t.n > (1 << 30)) return fail_inval("%s: %lld rows", what, (long long)t.n);
    if (t.v < 1 || t.v > kMaxVocab) return fail_inval("%s: %lld columns (1 to %d)", what, (long long)t.v, kMaxVocab);
    if (t.d < 1 || t.d > kMaxWidth) return fail_inval("%s: width %lld (1 to %d)", what, (long long)t.d, kMaxWidth);
    if (!valid_dtype(t.dtype)) return fail_inval("%s: unknown dtype %d", what, t.dtype);
    if (!(t.label_smoothing >= 0.0 && t.label_smoothing <= 1.0))
        return fail_inval("%s: label_smoothing must lie in [0, 1], got %g", what, t.label_smoothing);
    if (t.reduction < GEFEN_REDUCE_NONE || t.reduction > GEFEN_REDUCE_SUM)
        return fail_inval("%s: unknown reduction %d", what, t.reduction);
    p->n = (int)t.n;
    p->v = (int)t.v;
    p->d = (int)t.d;
    p->dtype = t.dtype;
    p->dh = t.grad_hidden != nullptr;
    p->dw = t.grad_weight != nullptr;
    p->train = p->dh || p->dw;
    p->smooth = t.label_smoothing > 0.0;
    p->planes = t.dtype == GEFEN_F32 || t.n <= kTwoPlaneRows ? 2 : 1;
    p->halves = t.dtype != GEFEN_BF16;
    p->dp = up(t.d, 64);
    p->ldg = up(t.v, kRowAlign);
    p->pack_w = t.dtype == GEFEN_F32 || t.d % 64 != 0 || t.weight_col_stride != 1 || t.weight_row_stride % 8 != 0 ||
                t.weight_row_stride > kMaxWidth || t.weight_row_stride < t.d || !aligned(t.weight, 16);
    // pieces of rows whose G and slots stay within the limit, of about the same size
    const int64_t limit = t.workspace_limit > 0 ? t.workspace_limit : GEFEN_LCE_DEFAULT_LIMIT;
    const int64_t row_bytes = (p->train ? p->ldg * 2 * p->planes : 0) + up(t.v, kSlot) / kSlot * 12;
    const int64_t all = up(t.n > 0 ? t.n : 1, kRowAlign);
    const int64_t most = limit / row_bytes / kRowAlign * kRowAlign;
    const int64_t fit = most < kRowAlign ? kRowAlign : most;
    const int64_t want = (all + fit - 1) / fit;
    const int64_t rows = up((all + want - 1) / want, kRowAlign);
    p->pieces = (int)((all + rows - 1) / rows);
    p->rows = (int)rows;
    const int64_t n = t.n < rows ? (t.n > 0 ? t.n : 1) : rows;
    const int64_t tiles = up(t.v, 256) / 256 * (up(n, 256) / 256);
    p->tile = n <= 32 ? kRowTile : tiles >= kCus / 2 ? kBigTile : kSmallTile;
    p->slots = (int)(up(t.v, kSlot) / kSlot);
    split_rule(t.d, n, up(t.v, 64) / 64, &p->dh_big, &p->dh_splits);
    split_rule(t.d, t.v, up(n, 64) / 64, &p->dw_big, &p->dw_splits);

    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 1023) / 1024 * 1024;
        return o;
    };
    const size_t n_up = (size_t)up(t.n > 0 ? t.n : 1, kRowAlign) + (size_t)p->rows;
    const int in_planes = t.dtype == GEFEN_F32 ? kPackPlanes : 1;
    p->o_meta = take(sizeof(Meta));
    p->o_map = take(n_up * 4);
    p->o_tgt = take(n_up * 4);
    p->o_tlogit = take(n_up * 4);
    p->o_losses = take(n_up * 4);
    p->o_x = take((size_t)in_planes * p->rows * p->pieces * p->dp * 2);
    p->o_w = p->pack_w ? take((size_t)in_planes * p->v * p->dp * 2) : at;
    p->o_stats = take((size_t)p->rows * p->slots * sizeof(float2));
    p->o_sums = p->smooth ? take((size_t)p->rows * p->slots * 4) : at;
    p->o_g = p->train ? take((size_t)p->planes * p->rows * p->ldg * 2) : at;
    p->o_wsum = p->dw && p->pieces > 1 ? take((size_t)p->v * p->d * 4) : at;
    size_t parts = 0;
    if (p->dh && p->dh_splits > 1) parts = (size_t)p->dh_splits * (size_t)n * p->d * 4;
    if (p->dw && p->dw_splits > 1) {
        const size_t b = (size_t)p->dw_splits * p->v * p->d * 4;
        parts = b > parts ? b : parts;
    }
    p->o_parts = take(parts);
    p->bytes = at;
    return GEFEN_OK;
}

template <typename C>
void launch_logits(Logits a, int most, hipStream_t st) {
    a.tiles_m = (a.v + C::TM - 1) / C::TM;
    const int grid = a.tiles_m * ((most + C::TN - 1) / C::TN);
    hipLaunchKernelGGL(k_logits<C>, dim3(grid), dim3(C::TT), 0, st, a);
}
template <typename C>
void launch_grad(Grad g, int n, hipStream_t st) {
    g.tiles_m = (g.d + C::TM - 1) / C::TM;
    const int grid = g.tiles_m * ((n + C::TN - 1) / C::TN) * g.splits;
    hipLaunchKernelGGL(k_grad<C>, dim3(grid), dim3(C::TT), 0, st, g);
    if (g.splits > 1) {
        const int64_t work = ((int64_t)n * ((g.d + 3) / 4) + 255) / 256;
        hipLaunchKernelGGL(k_join, dim3((unsigned)(work < 8192 ? work : 8192)), dim3(256), 0, st, g);
    }
}

template <bool F16>
void launch_products(const Plan& p, int which, const Logits& l, const Grad& g, int n, hipStream_t st) {
    if (which == 0) {
        if (p.tile == kBigTile) launch_logits<LogitsBig<F16>>(l, n, st);
        else if (p.tile == kSmallTile) launch_logits<LogitsSmall<F16>>(l, n, st);
        else launch_logits<LogitsRow<F16>>(l, n, st);
    } else if (which == 1) {
        if (p.dh_big) launch_grad<HiddenBig<F16>>(g, n, st);
        else launch_grad<HiddenSmall<F16>>(g, n, st);
    } else {
        if (p.dw_big) launch_grad<WeightBig<F16>>(g, n, st);
        else launch_grad<WeightSmall<F16>>(g, n, st);
    }
}

}  // namespace
}  // namespace lce
}  // namespace gefen

using namespace gefen;
using namespace gefen::lce;

extern "C" size_t gefen_linear_cross_entropy_workspace_size(const gefen_linear_cross_entropy_task* task) {
    Plan p;
    if (!task || make_plan(*task, &p, "gefen_linear_cross_entropy_workspace_size")) return 0;
    return p.bytes;
}

extern "C" int gefen_linear_cross_entropy(const gefen_linear_cross_entropy_task* task, void* workspace,
                                          size_t workspace_bytes, gefen_stream_t stream) {
    const char* what = "gefen_linear_cross_entropy";
    if (!task) return fail_inval("%s: no task", what);
    const gefen_linear_cross_entropy_task& t = *task;
    Plan p;
    const int bad = make_plan(t, &p, what);
    if (bad) return bad;
    if (!t.weight || (t.n && (!t.hidden || !t.targets))) return fail_inval("%s: null input", what);
    const int size = dtype_size(t.dtype);
    if (!aligned(t.hidden, size) || !aligned(t.weight, size) || !aligned(t.grad_hidden, size) ||
        !aligned(t.grad_weight, size) || !aligned(t.targets, t.targets_int32 ? 4 : 8))
        return fail_inval("%s: an operand is not aligned to its elements", what);
    if (t.n && !t.losses && !t.loss && !p.train) return fail_inval("%s: nothing to compute", what);
    if (t.loss && t.reduction == GEFEN_REDUCE_NONE) return fail_inval("%s: no reduction for a loss", what);
    if (t.reduction == GEFEN_REDUCE_NONE && p.train && t.n && !t.grad)
        return fail_inval("%s: gradients without a reduction need one gradient per row", what);
    if (!workspace || workspace_bytes < p.bytes)
        return fail_inval("%s: workspace of %zu bytes, needs %zu", what, workspace_bytes, p.bytes);
    if (!aligned(workspace, 16)) return fail_inval("%s: the workspace must be 16-byte aligned", what);

    hipStream_t st = stream;
    char* ws = static_cast<char*>(workspace);
    Meta* meta = reinterpret_cast<Meta*>(ws + p.o_meta);
    int32_t* map = reinterpret_cast<int32_t*>(ws + p.o_map);
    int32_t* tgt = reinterpret_cast<int32_t*>(ws + p.o_tgt);
    float* losses = t.losses ? t.losses : reinterpret_cast<float*>(ws + p.o_losses);
    uint16_t* x = reinterpret_cast<uint16_t*>(ws + p.o_x);
    uint16_t* wp = reinterpret_cast<uint16_t*>(ws + p.o_w);
    uint16_t* gbuf = reinterpret_cast<uint16_t*>(ws + p.o_g);
    const bool by_row = p.train && t.reduction == GEFEN_REDUCE_NONE;

    hipLaunchKernelGGL(k_rows, dim3(1), dim3(kRowsThreads), 0, st, t.targets, t.targets_int32, p.n, p.v, t.ignore_index,
                       by_row ? t.grad : nullptr, map, tgt, meta);
    const int x_rows = p.rows * p.pieces;
    Pack pk{};
    pk.src = t.hidden;
    pk.row_stride = t.hidden_row_stride;
    pk.col_stride = t.hidden_col_stride;
    pk.n = p.n;
    pk.d = p.d;
    pk.dp = (int)p.dp;
    pk.f32 = t.dtype == GEFEN_F32;
    pk.dst = x;
    pk.plane = (int64_t)x_rows * p.dp;
    pk.map = map;
    pk.meta = meta;
    pk.which = 0;
    pk.zero_rows = t.grad_hidden;
    pk.zero_losses = losses;
    if (pk.f32) {
        Top tx{static_cast<const float*>(t.hidden), t.hidden_row_stride, t.hidden_col_stride, p.n, p.d, map, meta, 0};
        hipLaunchKernelGGL(k_top, dim3(p.n < 2048 ? (p.n ? p.n : 1) : 2048), dim3(256), 0, st, tx);
        Top tw{static_cast<const float*>(t.weight), t.weight_row_stride, t.weight_col_stride, p.v, p.d, nullptr, meta, 1};
        hipLaunchKernelGGL(k_top, dim3(p.v < 2048 ? p.v : 2048), dim3(256), 0, st, tw);
    }
    const unsigned pack_y = (unsigned)((p.dp + 2047) / 2048);
    hipLaunchKernelGGL(k_pack, dim3((unsigned)x_rows, pack_y), dim3(256), 0, st, pk);
    if (p.pack_w) {
        Pack pw{};
        pw.src = t.weight;
        pw.row_stride = t.weight_row_stride;
        pw.col_stride = t.weight_col_stride;
        pw.n = p.v;
        pw.d = p.d;
        pw.dp = (int)p.dp;
        pw.f32 = pk.f32;
        pw.dst = wp;
        pw.plane = (int64_t)p.v * p.dp;
        pw.meta = meta;
        pw.which = 1;
        hipLaunchKernelGGL(k_pack, dim3((unsigned)p.v, pack_y), dim3(256), 0, st, pw);
    }
    Operand w{};
    w.p = p.pack_w ? wp : static_cast<const uint16_t*>(t.weight);
    w.ld = p.pack_w ? p.dp : t.weight_row_stride;
    w.plane = (int64_t)p.v * p.dp;
    // segments of the logits' product: low x high, high x low, high x high
    w.planes = pk.f32 ? 1 | 2 << 2 | 0 << 4 : 0;
    w.rows = p.v;
    w.cols = (int)p.dp;

    for (int piece = 0; piece < p.pieces; ++piece) {
        const int from = piece * p.rows;
        const int most = p.n - from < p.rows ? (p.n - from > 0 ? p.n - from : 0) : p.rows;
        Operand xo{};
        xo.p = x + (int64_t)from * p.dp;
        xo.ld = p.dp;
        xo.plane = pk.plane;
        xo.planes = pk.f32 ? 2 | 1 << 2 | 0 << 4 : 0;
        xo.rows = p.rows;
        xo.cols = (int)p.dp;
        Logits l{};
        l.w = w;
        l.x = xo;
        l.v = p.v;
        l.steps = (int)(p.dp / 64);
        l.segs = pk.f32 ? 3 : 1;
        l.f32 = pk.f32;
        l.from = from;
        l.most = most;
        l.slots = p.slots;
        l.stats = reinterpret_cast<float2*>(ws + p.o_stats);
        l.sums = p.smooth ? reinterpret_cast<float*>(ws + p.o_sums) : nullptr;
        l.target_logit = reinterpret_cast<float*>(ws + p.o_tlogit);
        l.tgt = tgt;
        l.meta = meta;
        l.g = p.train ? gbuf : nullptr;
        l.ldg = p.ldg;
        l.g_plane = (int64_t)p.rows * p.ldg;
        l.planes = p.planes;
        Grad g{};
        const bool f16 = p.halves;
        if (most > 0) {
            if (f16) launch_products<true>(p, 0, l, g, most, st);
            else launch_products<false>(p, 0, l, g, most, st);
            Rows r{};
            r.stats = l.stats;
            r.sums = l.sums;
            r.target_logit = l.target_logit;
            r.tgt = tgt;
            r.map = map;
            r.meta = meta;
            r.row_grad = by_row ? t.grad : nullptr;
            r.losses = losses;
            r.g = l.g;
            r.ldg = p.ldg;
            r.g_plane = l.g_plane;
            r.v = p.v;
            r.slots = p.slots;
            r.from = from;
            r.most = most;
            r.planes = p.planes;
            r.smoothing = (float)t.label_smoothing;
            // a row per workgroup, or parts of it where the rows do not fill the chip
            const int64_t rows_up = p.train ? up(most, 64) : most;
            int64_t parts = p.train ? 2048 / rows_up : 1;
            const int64_t chunks = p.ldg / 8 / kGradThreads;
            if (parts > chunks) parts = chunks;
            if (parts < 1) parts = 1;
            const dim3 grid((unsigned)rows_up, (unsigned)parts);
            if (f16) hipLaunchKernelGGL(k_gradient_rows<true>, grid, dim3(kGradThreads), 0, st, r);
            else hipLaunchKernelGGL(k_gradient_rows<false>, grid, dim3(kGradThreads), 0, st, r);
        }
        if (!p.train) continue;
        Operand go{};
        go.p = gbuf;
        go.ld = p.ldg;
        go.plane = l.g_plane;
        // with W or hidden of one plane: low, high; float32: as hidden in the logits' product
        go.planes = pk.f32 ? 0 | 1 << 2 | 0 << 4 : p.planes == 2 ? 1 | 0 << 2 : 0;
        go.rows = p.rows;
        go.cols = (int)p.ldg;
        g.d = p.d;
        g.segs = pk.f32 ? 3 : p.planes;
        g.from = from;
        g.most = most;
        g.map = map;
        g.meta = meta;
        g.grad = by_row ? nullptr : t.grad;
        g.mean = t.reduction == GEFEN_REDUCE_MEAN;
        g.by_row = by_row;
        g.dtype = t.dtype;
        float* parts = reinterpret_cast<float*>(ws + p.o_parts);
        if (p.dh && most > 0) {
            g.a = w;
            g.b = go;
            g.dh = 1;
            g.n = most;
            g.steps = (p.v + 63) / 64;
            g.splits = p.dh_splits;
            g.parts = g.splits > 1 ? parts : nullptr;
            g.sum = nullptr;
            g.out = t.grad_hidden;
            if (f16) launch_products<true>(p, 1, l, g, most, st);
            else launch_products<false>(p, 1, l, g, most, st);
        }
        if (p.dw) {
            g.a = xo;
            g.a.planes = w.planes;
            g.b = go;
            g.dh = 0;
            g.n = p.v;
            g.splits = p.dw_splits;
            g.parts = g.splits > 1 ? parts : nullptr;
            g.sum = p.pieces > 1 ? reinterpret_cast<float*>(ws + p.o_wsum) : nullptr;
            g.first = piece == 0;
            g.last = piece == p.pieces - 1;
            g.out = t.grad_weight;
            if (f16) launch_products<true>(p, 2, l, g, p.v, st);
            else launch_products<false>(p, 2, l, g, p.v, st);
        }
    }
    if (t.loss)
        hipLaunchKernelGGL(k_loss, dim3(1), dim3(1024), 0, st, losses, p.n, meta, t.reduction == GEFEN_REDUCE_MEAN,
                           t.loss);
    return launch_status(what);
}
