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
//   bits more than bf16 (one more than half; pack_exp2).
// * One pass over those values turns them into G (k_gradient_rows): a row's lse comes
//   from its slots, and exp(m - lse) scales each slot.  The target's entry is formed in
//   float32 from its own logit, so that p - 1 of a confident row does not cancel in
//   16 bits.  G is then rounded to the operands' type: with the kept values' smaller one,
//   the rounding below float32 on the way to the gradients.  Element by element it is up to
//   half an ulp of each term, so where one term dominates (the row of dW of a token that
//   occurs once, dh of a row far from its target) it scales the whole row and is as large as
//   the output's own rounding; over many terms the errors are independent (1.9e-3 of a bf16
//   gradient in all where the output's rounding alone is 1.7e-3; half 2.6e-4 and 2.1e-4).
// * 16-bit outputs are rounded once, after the loss's own gradient (factor).
// * For few rows one term can be most of a sum, and the products wait for W or dW
//   anyway: G is then two planes, twice the type's bits (kTwoPlaneRows).
// * Rows are taken in pieces whose G fits a bounded workspace; the logits of a piece
//   exist only as these 16-bit values, and never all of them at once when the
//   positions do not fit.  dW is summed over the pieces in float32.
//
// A half-precision G is scaled by 2^15 (and its products by 2^-15), which keeps
// probabilities down to 1e-9 out of half's subnormals.  float32 runs as two half planes
// per operand and three products, weight scaled by the power of two that brings its
// largest finite element to 2^14 and each row of hidden by its own: elements keep 22 bits
// down to 2^-28 of the largest one, and what they keep ends at 2^-49 of it (2^-50 for G,
// whose largest is 1), at five times the rate of the float32 matrix instructions.  dW sums
// rows, and takes all of hidden at one scale.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <utility>

#include "capi_internal.h"
#include "common.h"
#include "lce_gemm.h"

namespace gefen {
namespace lce {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kHalfScale = 32768.0f;  // of a half-precision G
constexpr int kSlot = 64;               // columns that share a maximum
constexpr int kRowAlign = 256;          // rows of a piece, columns of G
constexpr int kMaxVocab = 4 << 20;      // 256 rows of G within 2^31 bytes
constexpr int kMaxWidth = 1 << 20;

// Device scalars of a call.
struct Meta {
    int32_t count;    // rows that take part
    float grad_max;   // largest finite |gradient| of a row (per-row gradients)
    uint32_t top[2];  // largest finite magnitude of hidden and weight, as bits, where they are scaled
    float factor[2];  // what the sums of dW and dh are multiplied by
};

__device__ __forceinline__ int piece_rows(const Meta* m, int from, int most) {
    return max(0, min(m->count - from, most));
}

__device__ __forceinline__ int64_t target_at(const void* t, int is32, int64_t n) {
    return is32 ? (int64_t) static_cast<const int32_t*>(t)[n] : static_cast<const int64_t*>(t)[n];
}

// Which rows take part.
struct Select {
    const void* targets;
    int32_t targets_int32, n, v;
    int64_t ignore;
    const float* row_grad;  // gradient of each row's loss (null: one for all)
    int32_t* map;
    int32_t* tgt;
    Meta* meta;
    int32_t again;  // all but grad_max is there from a forward call
};
// map = the rows that take part, in order, then the ignored ones; tgt = their targets in
// that order (-1: not a column, whose loss is NaN; may be null).  One workgroup.
template <int THREADS>
__device__ __forceinline__ Meta select_rows(const Select& s, int32_t* map, int32_t* tgt) {
    __shared__ int wave_sum[THREADS / 64];
    __shared__ float wave_max[THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Meta m = {0, 0.0f, {0, 0}, {0.0f, 0.0f}};
    // a wave takes 64 kEach consecutive rows of each stretch, so that one barrier serves
    // kEach loads in flight
    constexpr int kEach = 4;
    for (int at = 0; at < s.n; at += THREADS * kEach) {
        const int first = at + wave * 64 * kEach + lane;
        int64_t y[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            y[k] = first + 64 * k < s.n ? target_at(s.targets, s.targets_int32, first + 64 * k) : s.ignore;
        uint64_t ball[kEach];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            ball[k] = __ballot(y[k] != s.ignore);
            mine += __popcll(ball[k]);
        }
        if (lane == 0) wave_sum[wave] = mine;
        __syncthreads();
        int off = m.count, all = 0;
        for (int w = 0; w < THREADS / 64; ++w) {
            if (w < wave) off += wave_sum[w];
            all += wave_sum[w];
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int i = first + 64 * k;
            const int before = off + __popcll(ball[k] & ((1ull << lane) - 1ull));
            if (y[k] != s.ignore) {
                map[before] = i;
                if (tgt) tgt[before] = (y[k] >= 0 && y[k] < s.v) ? (int)y[k] : -1;
                if (s.row_grad) {
                    const float c = fabsf(s.row_grad[i]);
                    if (c < INFINITY) m.grad_max = fmaxf(m.grad_max, c);
                }
            } else if (i < s.n) {
                map[s.n - 1 - (i - before)] = i;
            }
            off += __popcll(ball[k]);
        }
        m.count += all;
        __syncthreads();
    }
    for (int off = 32; off > 0; off >>= 1) m.grad_max = nanmax(m.grad_max, __shfl_xor(m.grad_max, off, 64));
    if (lane == 0) wave_max[wave] = m.grad_max;
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) m.grad_max = nanmax(m.grad_max, wave_max[w]);
    return m;
}
constexpr int kRowsThreads = 1024;
__global__ __launch_bounds__(kRowsThreads) void k_rows(const Select s) {
    const Meta m = select_rows<kRowsThreads>(s, s.map, s.tgt);
    if (threadIdx.x != 0) return;
    if (s.again) s.meta->grad_max = m.grad_max;
    else *s.meta = m;
}

// x (scaled into half's range) as a half and what it leaves times kLowScale.
__device__ __forceinline__ void split_half(float x, uint16_t* hi, uint16_t* lo) {
    const f16_t h = from_f32<f16_t>(x);
    *hi = h.bits;
    // what is not finite has no remainder worth adding: inf - inf is NaN
    *lo = (h.bits & 0x7c00) == 0x7c00 ? 0 : from_f32<f16_t>((x - to_f32(h)) * kLowScale).bits;
}
// The same for what is finite or has no use for the low part (subnormal halves rounded as
// the conversion instruction does).
__device__ __forceinline__ uint16_t half_bits(float x) {
    const _Float16 h = (_Float16)x;
    uint16_t u;
    __builtin_memcpy(&u, &h, 2);
    return u;
}
__device__ __forceinline__ void split_half_fast(float x, uint16_t* hi, uint16_t* lo) {
    const _Float16 h = (_Float16)x;
    *hi = half_bits(x);
    *lo = half_bits((x - (float)h) * kLowScale);
}
__device__ __forceinline__ void split_bf16(float x, uint16_t* hi, uint16_t* lo) {
    const bf16_t h = from_f32<bf16_t>(x);
    *hi = h.bits;
    *lo = (h.bits & 0x7f80) == 0x7f80 ? 0 : from_f32<bf16_t>(x - to_f32(h)).bits;
}

// exp(l - m) in [0, 1] as 16 unsigned bits on its way to G: 5 exponent and 11 mantissa
// bits for a half G, 6 and 10 for a bf16 one, with subnormals.  The float's own exponent
// is brought down by a product with a power of two (subnormal results are rounded by the
// hardware), and the mantissa is rounded to nearest.  Relative error 2^-12 down to 2^-30 and
// 2^-42 absolute below (bf16: 2^-11 down to 2^-62, 2^-73 below): finer than a half G, which
// ends at 2^-39.  (With 4 and 12 bits a column 19 nats below the one that leads its slot
// was lost, and the target's entry, formed on its own, had nothing to balance it.)
// Two of them, low half first.
template <bool F16>
__device__ __forceinline__ uint32_t pack_exp2(float a, float b) {
    constexpr int drop = F16 ? 12 : 13;
    constexpr float down = F16 ? 0x1p-96f : 0x1p-64f;
    const uint32_t x = __float_as_uint(a * down) + (1u << (drop - 1));
    const uint32_t y = __float_as_uint(b * down) + (1u << (drop - 1));
    return (x >> drop & 0xffffu) | (y >> drop << 16);
}
template <bool F16>
__device__ __forceinline__ float unpack_exp(uint16_t x) {
    return __uint_as_float((uint32_t)x << (F16 ? 12 : 13)) * (F16 ? 0x1p96f : 0x1p64f);
}

// Packed pairs of 16-bit values of a lane's four rows of MFMA tiles i (a) and i + 1 (b),
// rearranged so that every lane has eight consecutive rows: those of tile i + (lane / 32)
// from 8 ((lane / 16) % 2).  Lanes exchange with lanes of the same column only.
__device__ __forceinline__ uint4 eight_rows(uint2 a, uint2 b) {
    typedef uint32_t pair __attribute__((ext_vector_type(2)));
    pair x = __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false);
    pair y = __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false);
    x = __builtin_amdgcn_permlane16_swap(x[0], x[1], false, false);
    y = __builtin_amdgcn_permlane16_swap(y[0], y[1], false, false);
    return make_uint4(x[0], y[0], x[1], y[1]);
}

// Exponent that brings a matrix's largest finite magnitude (its bits in `top`) to 2^14.
__device__ __forceinline__ int half_exponent(uint32_t top) {
    return top == 0 ? 0 : 14 - max((int)(top >> 23) - 127, -112);
}

// The gradient c of a row's loss, where each row has its own.  All are taken relative to 2^E,
// the largest finite one between 2^(E-1) and 2^E (bfloat16: its factor has to stay a float32,
// E is 127 at most), and a row that is 2^-s of it has its power of two taken apart, so that a
// half G, which ends at 2^-39 (two planes: 2^-50), keeps its precision in every row:
//   * G's row carries w = c 2^-E 2^rest, down to 2^-carry;
//   * dh's row is multiplied by 2^-rest at the end (exact);
//   * for dW the row of hidden is (k_shift): its planes keep 2^-28 of hidden's largest element
//     in full and end at 2^-49 (half: 2^-38).
// A bfloat16 G has the range to carry all of it.  A gradient that is not finite stays in its
// own row of G, and so in its row of dh, and in dW, which sums it.
constexpr int kCarryOne = 4, kCarryTwo = 8, kCarryAll = 1 << 20;
struct RowWeight {
    float w;
    int rest;
};
__device__ __forceinline__ int grad_exponent(float top, int carry) {
    return min(__builtin_amdgcn_frexp_expf(top), carry == kCarryAll ? 127 : 128);
}
__device__ __forceinline__ RowWeight row_weight(float c, float top, int carry) {
    if (c == 0.0f || !(fabsf(c) < INFINITY)) return {c, 0};
    const int e = grad_exponent(top, carry);
    const int rest = max(0, e - __builtin_amdgcn_frexp_expf(c) - carry);
    return {ldexpf(c, rest - e), rest};
}

// meta->top[which] = the largest finite magnitude of a float32 or half matrix, as the bits
// of a float32; with a map, of the rows that take part (rows: each one's own too).  Maxima
// of integers: any order gives the same.
struct Top {
    const void* src;
    int64_t row_stride, col_stride;
    int32_t n, d;
    const int32_t* map;
    Meta* meta;
    int32_t which, f16;
    uint32_t* rows;  // [n] (may be null)
};
constexpr int kTopThreads = 1024, kTopGrid = 256;
// the largest finite magnitude of up to eight columns of a row
template <typename T>
__device__ __forceinline__ uint32_t top_of_chunk(const T* s, int64_t col_stride, int cols) {
    uint32_t top = 0;
    auto see = [&](T x) {
        const uint32_t u = abs_key(to_f32(x));
        top = u < 0x7f800000u && u > top ? u : top;
    };
    if (col_stride == 1 && cols >= 8) {
        const AnyVec<T, 8> x = *reinterpret_cast<const AnyVec<T, 8>*>(s);
#pragma unroll
        for (int e = 0; e < 8; ++e) see(x.v[e]);
    } else {
        for (int e = 0; e < min(cols, 8); ++e) see(s[e * col_stride]);
    }
    return top;
}
__device__ __forceinline__ uint32_t top_of_chunk(const Top& t, int r, int c) {
    const int64_t at = (int64_t)(t.map ? t.map[r] : r) * t.row_stride + c * t.col_stride;
    return t.f16 ? top_of_chunk(static_cast<const f16_t*>(t.src) + at, t.col_stride, t.d - c)
                 : top_of_chunk(static_cast<const float*>(t.src) + at, t.col_stride, t.d - c);
}
__device__ __forceinline__ void top_block(const Top& t, int block, int blocks) {
    const int per = (t.d + 7) / 8;  // chunks of eight columns a row
    const int rows = t.map ? t.meta->count : t.n;
    uint32_t top = 0;
    if (t.rows) {  // a row per wave
        constexpr int kWaves = kTopThreads / 64;
        for (int r = block * kWaves + (threadIdx.x >> 6); r < rows; r += blocks * kWaves) {
            uint32_t own = 0;
            for (int c = threadIdx.x & 63; c < per; c += 64) own = max(own, top_of_chunk(t, r, c * 8));
            own = wave_group_max_u32(own, 64);
            if ((threadIdx.x & 63) == 0) t.rows[r] = own;
            top = max(top, own);
        }
    } else {
        const int64_t all = (int64_t)rows * per;
        for (int64_t q = (int64_t)block * kTopThreads + threadIdx.x; q < all; q += (int64_t)blocks * kTopThreads) {
            const int r = (int)(q / per);
            top = max(top, top_of_chunk(t, r, (int)(q - (int64_t)r * per) * 8));
        }
    }
    // one atomic per workgroup, and few of those: on one address each takes 12 ns
    __shared__ uint32_t part[kTopThreads / 64];
    top = wave_group_max_u32(top, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kTopThreads / 64; ++w) top = max(top, part[w]);
        if (top > 0) atomicMax(&t.meta->top[t.which], top);
    }
}
// Workgroups up to `first` take a, the others b.
__global__ __launch_bounds__(kTopThreads) void k_top(const Top a, const Top b, int first) {
    if ((int)blockIdx.x < first) top_block(a, blockIdx.x, first);
    else top_block(b, blockIdx.x - first, gridDim.x - first);
}

// Rows of a matrix of any strides as the products read them: dp = D rounded up to 64
// columns, zero-padded, one plane or those of a float32 operand, scaled: weight by its largest
// element, hidden row by row, so that no row's logits depend on the size of another (for dW,
// which sums rows, all by the largest: k_shift).  With a map: row r is src row map[r] for
// r < meta->count and zero up to the next multiple of kRowAlign, and the rows that take no
// part get a zero loss.  A thread moves eight columns of a row.
// Bound by HBM: 8192 x 4096 bf16 rows in 28 us (4.8 TB/s), 50257 x 768 float32 ones and
// their three planes in 60 (6.4), 8192 x 768 of them again for dW in 15.
constexpr int kPackPlanes = 3;  // of a float32 operand: high, low, high where finite
struct Pack {
    const void* src;
    int64_t row_stride, col_stride;
    int32_t n, d, dp;
    int32_t f32;
    uint16_t* dst;
    int64_t plane;
    int32_t rows;       // of dst
    const int32_t* map;
    const Meta* meta;
    int32_t which;      // float32: whose largest magnitude in meta->top
    float* zero_losses;  // [n] (may be null)
    const uint32_t* row_top;  // float32 hidden: largest magnitude of each row
    // SHIFT: rows [from, from + most) that take part again, scaled by the largest element of
    // all, times their gradients' powers of two (if they have their own)
    const float* row_grad;
    int32_t from, most, carry;
};
template <bool SHIFT = false>
__device__ __forceinline__ void pack_block(const Pack& p, const int32_t* map, int count, int block, int blocks) {
    const uint32_t per = (uint32_t)p.dp / 8;
    const int first = SHIFT ? p.from : 0;
    const int ends = SHIFT ? min(count, p.from + p.most)
                     : map ? (count + kRowAlign - 1) / kRowAlign * kRowAlign
                           : p.rows;
    const int64_t all = (int64_t)((SHIFT || ends > p.n ? ends : p.n) - first) * per;
    const int top = p.f32 || SHIFT ? half_exponent(p.meta->top[p.which]) : 0;
    for (int64_t q = (int64_t)block * 256 + threadIdx.x; q < all; q += (int64_t)blocks * 256) {
        const int up = (int)(q / per);
        const int r = first + up;
        const int c0 = (int)(q - (int64_t)up * per) * 8;
        const int64_t row = map && r < p.n ? map[r] : r;
        const bool live = r < count;
        int ex = top;
        if (SHIFT && p.row_grad) ex -= row_weight(p.row_grad[row], p.meta->grad_max, p.carry).rest;
        if (!SHIFT && p.row_top && live) ex = half_exponent(p.row_top[r]);
        if (map && !live && r < p.n && p.zero_losses && c0 == 0) p.zero_losses[row] = 0.0f;
        if (r >= ends) continue;
        Vec<uint16_t, 8> out[kPackPlanes] = {};
        if (live && p.f32) {
            const float* s = static_cast<const float*>(p.src) + row * p.row_stride + (int64_t)c0 * p.col_stride;
            AnyVec<float, 8> x = {};
            if (p.col_stride == 1 && c0 + 8 <= p.d) {
                x = *reinterpret_cast<const AnyVec<float, 8>*>(s);
            } else {
                for (int e = 0; e < 8; ++e)
                    if (c0 + e < p.d) x.v[e] = s[e * p.col_stride];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                split_half(ldexpf(x.v[e], ex), &out[0].v[e], &out[1].v[e]);
                out[2].v[e] = (out[0].v[e] & 0x7c00) == 0x7c00 ? 0 : out[0].v[e];
            }
        } else if (live) {
            const uint16_t* s = static_cast<const uint16_t*>(p.src) + row * p.row_stride + (int64_t)c0 * p.col_stride;
            if (p.col_stride == 1 && c0 + 8 <= p.d) {
                const AnyVec<uint16_t, 8> x = *reinterpret_cast<const AnyVec<uint16_t, 8>*>(s);
#pragma unroll
                for (int e = 0; e < 8; ++e) out[0].v[e] = x.v[e];
            } else {
                for (int e = 0; e < 8; ++e)
                    if (c0 + e < p.d) out[0].v[e] = s[e * p.col_stride];
            }
            if (SHIFT) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    out[0].v[e] = from_f32<f16_t>(ldexpf(to_f32(f16_t{out[0].v[e]}), ex)).bits;
            }
        }
        uint16_t* d = p.dst + (int64_t)r * p.dp + c0;
        vstore(d, 0, out[0]);
        if (p.f32) {
            vstore(d + p.plane, 0, out[1]);
            vstore(d + 2 * p.plane, 0, out[2]);
        }
    }
}

// hidden by the workgroups up to `first`, weight by the others (if there are any).
__global__ __launch_bounds__(256) void k_pack(const Pack x, const Pack w, int first) {
    if ((int)blockIdx.x < first) pack_block(x, x.map, x.meta->count, blockIdx.x, first);
    else pack_block(w, nullptr, w.n, blockIdx.x - first, gridDim.x - first);
}
// Hidden of half-precision products as dW reads it, where its rows are scaled one by one or
// have gradients of their own.
__global__ __launch_bounds__(256) void k_shift(const Pack x) {
    pack_block<true>(x, x.map, x.meta->count, blockIdx.x, gridDim.x);
}
// The same for few rows without k_rows: every workgroup of hidden selects them for itself
// (the first one for the kernels that follow), which saves a launch.
constexpr int kSelfRows = 1024;
__global__ __launch_bounds__(256) void k_select_pack(const Select s, const Pack x, const Pack w, int first) {
    __shared__ int32_t map[kSelfRows];
    if ((int)blockIdx.x >= first) {
        pack_block(w, nullptr, w.n, blockIdx.x - first, gridDim.x - first);
        return;
    }
    const Meta m = select_rows<256>(s, map, blockIdx.x == 0 ? s.tgt : nullptr);
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < s.n; i += 256) s.map[i] = map[i];
        if (threadIdx.x == 0) *s.meta = m;
    }
    pack_block(x, map, m.count, blockIdx.x, first);
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
    int32_t planes;
    const uint32_t* row_top;  // float32: largest magnitude of each row of hidden, over all pieces (or null)
};

// What a logits' product keeps for the gradients: nothing, 16 packed bits, two planes.
enum Keep { kKeepNone, kKeepPacked, kKeepPlanes };

// What becomes of a tile of logits.
template <typename C, int KEEP>
__device__ __forceinline__ void logits_tile(const Logits& a, int rows, int m0, int n0, int ex,
                                            f32x4 (&acc)[C::WI][C::WJ]) {
    constexpr int WI = C::WI, WJ = C::WJ;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = m0 + (wave / C::WAVES_N) * C::WM, wn = n0 + (wave % C::WAVES_N) * C::WN;
    const int hi = 4 * (lane >> 4);
    const int slot = wm / kSlot;
    static_assert(C::WM == kSlot, "a wave's columns are a slot");
    if (wm >= a.v && KEEP == kKeepNone) return;
    const bool f32 = KEEP != kKeepPacked && a.row_top;
    const bool part = wm + C::WM > a.v;  // the last columns end inside this wave's
    int target[WJ], down[WJ];  // loaded first: among the stores below each would wait for those before it
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        const int n = wn + j * 16 + (lane & 15);
        target[j] = n < rows ? a.tgt[a.from + n] - wm : -1;
        down[j] = f32 && n < rows ? ex - half_exponent(a.row_top[a.from + n]) : 0;
    }
#pragma unroll
    for (int j = 0; j < WJ; ++j) {
        const int n = wn + j * 16 + (lane & 15);
        float m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (f32) acc[i][j][r] = ldexpf(acc[i][j][r], down[j]);
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
        const int y = target[j];
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
                // the difference first: exact where it matters, however large the logits; the
                // product's rounding is 2^-24 |x| of exp(x) (the kept values' scale comes after
                // the exponential: as an offset of 64 in its argument it cost the sum 2^-18)
                acc[i][j][r] = __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * kLog2E);
                s += acc[i][j][r];
            }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (n < rows && lane < 16 && wm < a.v) {
            const int64_t at = (int64_t)n * a.slots + slot;
            a.stats[at] = make_float2(m, s);
            if (a.sums) a.sums[at] = sum;
        }
        if constexpr (KEEP == kKeepNone) continue;
        // rows past the piece's end stay inside the workspace (it holds whole tiles)
        uint16_t* row = a.g + (int64_t)n * a.ldg + wm + 16 * (lane >> 5) + 8 * (lane >> 4 & 1);
#pragma unroll
        for (int i = 0; i < WI; i += 2) {
            uint2 w[2][2];  // [plane][tile]
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 e = acc[i + t][j];
                if constexpr (KEEP == kKeepPacked) {
                    w[0][t] = make_uint2(pack_exp2<C::F16>(e[0], e[1]), pack_exp2<C::F16>(e[2], e[3]));
                } else {
                    uint16_t o[2][4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if constexpr (C::F16) split_half_fast(e[r] * kHalfScale, &o[0][r], &o[1][r]);
                        else split_bf16(e[r], &o[0][r], &o[1][r]);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        w[k][t] = make_uint2((uint32_t)o[k][0] | ((uint32_t)o[k][1] << 16),
                                             (uint32_t)o[k][2] | ((uint32_t)o[k][3] << 16));
                }
            }
            *reinterpret_cast<uint4*>(row + i * 16) = eight_rows(w[0][0], w[0][1]);
            if constexpr (KEEP == kKeepPlanes)
                *reinterpret_cast<uint4*>(row + i * 16 + a.g_plane) = eight_rows(w[1][0], w[1][1]);
        }
    }
}

template <typename C, int KEEP>
__global__ __launch_bounds__(C::TT, C::EU) void k_logits(const Logits a) {
    __shared__ __attribute__((aligned(1024))) uint16_t smem[C::NST * C::STAGE];
    const int rows = piece_rows(a.meta, a.from, a.most);
    const int tiles_n = (rows + C::TN - 1) / C::TN;
    const int live = tiles_n * a.tiles_m;
    if ((int)blockIdx.x >= live) return;
    const int ex = a.row_top ? -half_exponent(a.meta->top[1]) : 0;  // of weight
    auto unit_of = [&](int u) __attribute__((always_inline)) {
        int ti, tj;
        tile_of<C::GROUP_M>(logical_block(u, live), a.tiles_m, tiles_n, &ti, &tj);
        return Unit{ti * C::TM, tj * C::TN, 0, a.steps};
    };
    auto finish = [&](int, const Unit& unit, f32x4(&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        logits_tile<C, KEEP>(a, rows, unit.m0, unit.n0, ex, acc);
    };
    product_stream<C>(a.w, a.x, a.segs, blockIdx.x, live, gridDim.x, (lds_u16*)smem, unit_of, finish);
}

// Loss of each row from its slots, and (g) the row's values turned into G: one workgroup a
// row, or parts of one where the rows are few (each joins the row's slots for itself).
// Bound by HBM: 8192 x 128256 values read and written in 0.84 ms (5.0 TB/s); the losses alone
// in 48 us.
struct Rows {
    const float2* stats;
    const float* sums;
    const float* target_logit;
    const int32_t* tgt;
    const int32_t* map;
    Meta* meta;
    const float* row_grad;  // gradient of each row's loss (null: one for all)
    const float* grad;      // gradient of the loss (null: 1)
    int32_t mean, dtype, carry;
    float* losses;          // [n], original order
    uint16_t* g;
    int64_t ldg, g_plane;
    int32_t v, slots, from, most, planes;
    float smoothing;
    void* zero_rows;        // [n, zero_bytes]: dh, zero where a row takes no part (may be null)
    int64_t zero_bytes;     // of a row
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
    const float m = nanmax(a.x, b.x);
    const float ref = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * expf(a.x - ref) + b.y * expf(b.x - ref));
}

template <bool STREAM>
__device__ __forceinline__ Vec<uint16_t, 8> load8(const uint16_t* p) {
    using R = typename RawVec<16>::type;
    const R r = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const R*>(p)) : *reinterpret_cast<const R*>(p);
    Vec<uint16_t, 8> x;
    __builtin_memcpy(&x, &r, sizeof(x));
    return x;
}
template <bool STREAM>
__device__ __forceinline__ void store8(uint16_t* p, const Vec<uint16_t, 8>& x) {
    using R = typename RawVec<16>::type;
    R r;
    __builtin_memcpy(&r, &x, sizeof(r));
    if (STREAM) __builtin_nontemporal_store(r, reinterpret_cast<R*>(p));
    else *reinterpret_cast<R*>(p) = r;
}

constexpr int64_t kKeepBytes = 192 << 20;  // of a memory-side cache of 256 MB
constexpr int kGradThreads = 256;
// STREAM: G is larger than the memory-side cache holds, and its values go past the caches.
template <bool F16, bool STREAM>
__global__ __launch_bounds__(kGradThreads) void k_gradient_rows(const Rows a) {
    __shared__ float2 part[kGradThreads / 64];
    __shared__ float part_sum[kGradThreads / 64];
    const int r = blockIdx.x;
    const int rows = piece_rows(a.meta, a.from, a.most);
    const int chunks = (int)(a.ldg / 8);
    if (a.g && r == 0 && blockIdx.y == 0 && threadIdx.x < 2) {
        // of dW (whose other operand is hidden) and dh
        float f = a.dtype == GEFEN_BF16 ? 1.0f : 1.0f / kHalfScale;
        int ex = 0;
        if (a.dtype == GEFEN_F32 || (a.dtype == GEFEN_F16 && a.row_grad && threadIdx.x == 0))
            ex = -half_exponent(a.meta->top[threadIdx.x]);
        if (a.row_grad) {
            ex += grad_exponent(a.meta->grad_max, a.carry);
        } else {
            if (a.grad) f *= *a.grad;
            if (a.mean) f = a.meta->count ? f / (float)a.meta->count : 0.0f;
        }
        a.meta->factor[threadIdx.x] = ldexpf(f, ex);
    }
    if (r >= rows) {
        if (a.zero_rows && r < a.most) {
            uint16_t* z = static_cast<uint16_t*>(a.zero_rows) + (int64_t)a.map[a.from + r] * (a.zero_bytes / 2);
            for (int64_t c = blockIdx.y * kGradThreads + threadIdx.x; c < a.zero_bytes / 2; c += gridDim.y * kGradThreads)
                z[c] = 0;
        }
        // zero rows up to the end of the last K step of dW
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
    // lse = m + log s, kept apart: differences to m stay exact for large logits
    const float log_s = logf(st.y);
    const int y = a.tgt[a.from + r];
    const float tl = y >= 0 ? a.target_logit[a.from + r] : NAN;
    const float e = a.smoothing;
    const int64_t n = a.map[a.from + r];
    if (a.losses && blockIdx.y == 0 && threadIdx.x == 0) {
        float loss = (1.0f - e) * ((st.x - tl) + log_s);
        if (e > 0.0f) loss += e * ((st.x - sum / (float)a.v) + log_s);
        a.losses[n] = loss;
    }
    if (!a.g) return;
    float w = F16 ? kHalfScale : 1.0f;
    if (a.row_grad) w *= row_weight(a.row_grad[n], a.meta->grad_max, a.carry).w;
    const float unit = e > 0.0f ? e / (float)a.v : 0.0f;
    if (y < 0) w = NAN;
    // the target's entry from its own logit: p - 1 without cancellation in 16 bits
    const float at_target = expm1f((tl - st.x) - log_s) + e - unit;
    const float back = F16 && a.planes == 2 ? 1.0f / kHalfScale : 1.0f;
    constexpr int kBatch = 4;  // chunks in flight per thread
    const int stride = gridDim.y * kGradThreads;
    uint16_t* const row = a.g + (int64_t)r * a.ldg;
    for (int c0 = blockIdx.y * kGradThreads + threadIdx.x; c0 < chunks; c0 += kBatch * stride) {
        Vec<uint16_t, 8> x[kBatch][2];
        float top[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int c = min(c0 + i * stride, chunks - 1);
            top[i] = stats[min(c * 8, a.v - 1) / kSlot].x;
            x[i][0] = load8<STREAM>(row + (int64_t)c * 8);
            if (a.planes == 2) x[i][1] = load8<STREAM>(row + a.g_plane + (int64_t)c * 8);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int c = c0 + i * stride, v0 = c * 8;
            if (c >= chunks) break;
            const float f = expf((top[i] - st.x) - log_s) * back;
            Vec<uint16_t, 8>& hi = x[i][0];
            Vec<uint16_t, 8>& lo = x[i][1];
            const bool hit = y >= v0 && y < v0 + 8, part = v0 + 8 > a.v;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float q;
                if (a.planes == 1) q = unpack_exp<F16>(hi.v[e]);
                else if (F16) q = to_f32(f16_t{hi.v[e]}) + to_f32(f16_t{lo.v[e]}) * (1.0f / kLowScale);
                else q = to_f32(bf16_t{hi.v[e]}) + to_f32(bf16_t{lo.v[e]});
                q = q * f - unit;
                if (hit && v0 + e == y) q = at_target;
                q *= w;
                if (part && v0 + e >= a.v) q = 0.0f;
                if (a.planes == 1) hi.v[e] = F16 ? half_bits(q) : from_f32<bf16_t>(q).bits;
                else if (F16) split_half_fast(q, &hi.v[e], &lo.v[e]);
                else split_bf16(q, &hi.v[e], &lo.v[e]);
            }
            store8<STREAM>(row + (int64_t)c * 8, hi);
            if (a.planes == 2) store8<STREAM>(row + a.g_plane + (int64_t)c * 8, lo);
        }
    }
}

// The sum of the rows' losses in float64, over the count for a mean (0 / 0 = NaN
// where no row takes part, as the mean of nothing is).  One workgroup.
struct Loss {
    const float* losses;
    int32_t n, mean;
    const Meta* meta;
    float* out;  // null: no loss wanted
};
template <int THREADS>
__device__ __forceinline__ void sum_losses(const Loss& l) {
    __shared__ double part[THREADS / 64];
    double s = 0.0;
    for (int i = threadIdx.x; i < l.n; i += THREADS) s += (double)l.losses[i];
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; ++w) s += part[w];
        *l.out = (float)(l.mean ? s / (double)l.meta->count : s);
    }
}
__global__ __launch_bounds__(1024) void k_loss(const Loss l) { sum_losses<1024>(l); }

// A gradient's product: out[n, m] = factor * sum_k A[m, k] B[n, k] for m < D, rows n of
// the piece (dh, through the map) or of the vocabulary (dW).
struct Grad {
    Operand a, b;
    int32_t d, tiles_m, steps, segs;
    int32_t n;              // rows of the result (dW: V); dh: the piece's, from meta
    int32_t dh;             // dh: rows through the map, all of K; dW: K = the piece's rows
    int32_t from, most;
    const int32_t* map;
    const Meta* meta;
    int32_t slots;          // workgroups that fill the chip
    int32_t most_parts;     // partial tiles that `parts` holds
    float* parts;           // [cut][tile of the rest][TN][TM]
    float* sum;             // float32 sum over the pieces (null: one piece)
    int32_t first, last;    // pieces of the sum (last: it is the output, in float32)
    void* out;
    int32_t out_f32;
    const float* row_grad;  // dh: gradient of each row's loss (null: one for all)
    int32_t carry;
};
// What the sums of an output row are multiplied by.
template <typename C>
__device__ __forceinline__ float factor_of(const Grad& g, float factor, int64_t row) {
    if (C::BMN || !g.row_grad) return factor;  // dW; one gradient for all rows
    return ldexpf(factor, -row_weight(g.row_grad[row], g.meta->grad_max, g.carry).rest);
}

// How the tiles of a product meet the chip: whole rounds of it tile by tile, and the
// `rest` of the tiles with K cut into `cuts` equal parts, each left in float32 for k_join.
// All tiles of one part run together, so that they share what they read (dealing the rest's
// K steps out evenly instead, as one stretch per workgroup, balances better but left no
// two workgroups at the same K: dh of 2796 x 2048 over 128256 2.0 ms against 1.63 with two
// equal parts; with the number below 1.33).  The number of parts is the one of the least
// estimated time, in K steps of a full chip: rounds times the steps of a part and 4 for its
// ends, 0.06 for the traffic of each partial tile, and 4 and 0.1 a part for the launch that
// joins them.  The rows that take part are only known on the device, so this is worked out
// there; the host bounds it.
constexpr int kMostCuts = 128;
constexpr int kMostRounds = 4;
constexpr int kLeastSteps = 4;  // of a part
struct Deal {
    int n_all, tiles_n, steps, full, rest;
};
template <typename C>
__device__ __forceinline__ Deal deal_of(const Grad& g) {
    const int rows = piece_rows(g.meta, g.from, g.most);
    Deal d;
    d.n_all = g.dh ? rows : g.n;
    d.tiles_n = (d.n_all + C::TN - 1) / C::TN;
    d.steps = g.dh ? g.steps : (rows + C::BK - 1) / C::BK;
    const int tiles = d.tiles_n * g.tiles_m;
    d.rest = tiles & (g.slots - 1);  // slots: a power of two
    d.full = tiles - d.rest;
    return d;
}
__device__ __forceinline__ int cuts_of(const Grad& g, const Deal& d) {
    int cuts = 1;
    const float run = (float)(d.steps * g.segs);
    float best = run + 4.0f;
    for (int rounds = 1; rounds <= kMostRounds; ++rounds) {
        int c = min(rounds * g.slots, g.most_parts) / d.rest;
        c = min(min(c, kMostCuts), d.steps / kLeastSteps);
        if (c < 2) continue;
        const float cost = (float)((d.rest * c + g.slots - 1) / g.slots) * (run / (float)c + 4.0f) +
                           0.06f * (float)(d.rest * c) + 0.1f * (float)c + 4.0f;
        if (cost < best) {
            best = cost;
            cuts = c;
        }
    }
    return cuts;
}

// A result goes to the sum over the pieces (plain float32 up to the last one of a float32
// output), or times the factor to the output in its type.
enum Out { kOutSum, kOutF32, kOut16 };
// cnt (1 to 4) float32 results of output row `row`, from column m
template <int OUT>
__device__ __forceinline__ void finish_f32(const Grad& g, int64_t row, int m, int cnt, f32x4 v, float factor) {
    const int64_t at = row * g.d + m;
    if constexpr (OUT == kOutSum) {
        float* s = g.sum + at;
        for (int e = 0; e < cnt; ++e) {
            const float x = g.first ? v[e] : s[e] + v[e];
            s[e] = g.last ? x * factor : x;
        }
    } else {
        v *= factor;
        float* o = static_cast<float*>(g.out) + at;
        if (cnt == 4) {
            *reinterpret_cast<AnyVec<float, 4>*>(o) = AnyVec<float, 4>{{v[0], v[1], v[2], v[3]}};
        } else {
            for (int e = 0; e < cnt; ++e) o[e] = v[e];
        }
    }
}
template <bool F16>
__device__ __forceinline__ uint2 round16(f32x4 v, float factor) {
    uint16_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = F16 ? from_f32<f16_t>(v[e] * factor).bits : from_f32<bf16_t>(v[e] * factor).bits;
    return make_uint2((uint32_t)o[0] | ((uint32_t)o[1] << 16), (uint32_t)o[2] | ((uint32_t)o[3] << 16));
}
// cnt (1 to 8 of N) 16-bit results
template <int N>
__device__ __forceinline__ void store16(const Grad& g, int64_t row, int m, int cnt, const uint32_t (&w)[N / 2]) {
    uint16_t* o = static_cast<uint16_t*>(g.out) + row * g.d + m;
    AnyVec<uint16_t, N> x;
    __builtin_memcpy(&x, w, sizeof(x));
    if (cnt >= N) {
        *reinterpret_cast<AnyVec<uint16_t, N>*>(o) = x;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < cnt) o[e] = x.v[e];
    }
}
// The tile of this wave, from row m of the product and its column n.
template <typename C, int OUT>
__device__ __forceinline__ void finish_tile(const Grad& g, int n_all, int m0, int n0, float factor,
                                            const f32x4 (&acc)[C::WI][C::WJ]) {
    const int lane = threadIdx.x & 63;
    int rows[C::WJ];  // loaded before the first store
#pragma unroll
    for (int j = 0; j < C::WJ; ++j) {
        rows[j] = n0 + j * 16 + (lane & 15);
        if (g.dh && rows[j] < n_all) rows[j] = g.map[g.from + rows[j]];
    }
#pragma unroll
    for (int j = 0; j < C::WJ; ++j) {
        if (n0 + j * 16 + (lane & 15) >= n_all) continue;
        const int64_t row = rows[j];
        const float f = factor_of<C>(g, factor, row);
        if constexpr (OUT == kOut16) {
#pragma unroll
            for (int i = 0; i < C::WI; i += 2) {
                const uint4 v = eight_rows(round16<C::F16>(acc[i][j], f), round16<C::F16>(acc[i + 1][j], f));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                const int m = m0 + 16 * (i + (lane >> 5)) + 8 * (lane >> 4 & 1);
                if (m < g.d) store16<8>(g, row, m, g.d - m, w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < C::WI; ++i) {
                const int m = m0 + i * 16 + 4 * (lane >> 4);
                if (m < g.d) finish_f32<OUT>(g, row, m, min(4, g.d - m), acc[i][j], f);
            }
        }
    }
}

// Worker `b` of `workers` of a product.
template <typename C>
__device__ __forceinline__ void grad_block(const Grad& g, int b, int workers, lds_u16* smem) {
    const Deal deal = deal_of<C>(g);
    const int cuts = deal.rest ? cuts_of(g, deal) : 1;
    const int parts = deal.rest * cuts, total = deal.full + parts;
    const float factor = g.meta->factor[g.dh];
    auto unit_of = [&](int u) __attribute__((always_inline)) {
        int tile, cut = 0;
        const bool whole = u < deal.full;
        if (whole) {
            tile = logical_block(u, deal.full);
        } else {
            const int q = logical_block(u - deal.full, parts);
            cut = q / deal.rest;
            tile = deal.full + q - cut * deal.rest;
        }
        int ti, tj;
        tile_of<C::GROUP_M>(tile, g.tiles_m, deal.tiles_n, &ti, &tj);
        return Unit{ti * C::TM, tj * C::TN, whole ? 0 : deal.steps * cut / cuts,
                    whole ? deal.steps : deal.steps * (cut + 1) / cuts};
    };
    auto finish = [&](int u, const Unit& unit, f32x4(&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wm = (wave / C::WAVES_N) * C::WM, wn = (wave % C::WAVES_N) * C::WN;
        if (cuts > 1 && u >= deal.full) {
            float* p = g.parts + (int64_t)logical_block(u - deal.full, parts) * (C::TM * C::TN) +
                       (wn + (lane & 15)) * C::TM + wm + 4 * (lane >> 4);
#pragma unroll
            for (int j = 0; j < C::WJ; ++j)
#pragma unroll
                for (int i = 0; i < C::WI; ++i) *reinterpret_cast<f32x4*>(p + j * 16 * C::TM + i * 16) = acc[i][j];
        } else if (g.sum) {
            finish_tile<C, kOutSum>(g, deal.n_all, unit.m0 + wm, unit.n0 + wn, factor, acc);
        } else if (g.out_f32) {
            finish_tile<C, kOutF32>(g, deal.n_all, unit.m0 + wm, unit.n0 + wn, factor, acc);
        } else {
            finish_tile<C, kOut16>(g, deal.n_all, unit.m0 + wm, unit.n0 + wn, factor, acc);
        }
    };
    if (deal.steps == 0) {  // dW of no row at all
        for (int u = b; u < total; u += workers) {
            f32x4 none[C::WI][C::WJ] = {};
            finish(u, unit_of(u), none);
        }
    } else if (b < total) {
        product_stream<C>(g.a, g.b, g.segs, b, total, workers, smem, unit_of, finish);
    }
}

// One gradient's product; the last workgroup sums the losses where l.out is given, which
// saves a launch.
template <typename C>
__global__ __launch_bounds__(C::TT, C::EU) void k_grad(const Grad g, const Loss l) {
    __shared__ __attribute__((aligned(1024))) uint16_t smem[C::NST * C::STAGE];
    const int workers = gridDim.x - (l.out ? 1 : 0);
    if ((int)blockIdx.x == workers) return sum_losses<C::TT>(l);
    grad_block<C>(g, blockIdx.x, workers, (lds_u16*)smem);
}
// Both products, dh by the workers up to `first`.
template <typename H, typename W>
__global__ __launch_bounds__(H::TT, H::EU) void k_grads(const Grad h, const Grad w, const Loss l, int first) {
    static_assert(H::TT == W::TT && H::STAGE == W::STAGE && H::NST == W::NST, "one launch");
    __shared__ __attribute__((aligned(1024))) uint16_t smem[H::NST * H::STAGE];
    const int workers = gridDim.x - (l.out ? 1 : 0);
    if ((int)blockIdx.x == workers) return sum_losses<H::TT>(l);
    if ((int)blockIdx.x < first) grad_block<H>(h, blockIdx.x, first, (lds_u16*)smem);
    else grad_block<W>(w, blockIdx.x - first, workers - first, (lds_u16*)smem);
}

// The parts of the cut tiles added up, the same way each time: wave w of a workgroup adds
// parts w, w + 4, ... in order, and the four sums are added in order.  t: tile of the rest,
// blockIdx.y of kJoinBlocks: every kJoinBlocks-th 256 of its elements.
constexpr int kJoinBlocks = 64;
template <typename C>
__device__ __forceinline__ void join_block(const Grad& g, int t) {
    __shared__ f32x4 part[4][64];
    const Deal deal = deal_of<C>(g);
    if (t >= deal.rest) return;
    const int cuts = cuts_of(g, deal);
    if (cuts == 1) return;
    int ti, tj;
    tile_of<C::GROUP_M>(deal.full + t, g.tiles_m, deal.tiles_n, &ti, &tj);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float factor = g.meta->factor[g.dh];
    for (int chunk = blockIdx.y; chunk < C::TM * C::TN / 256; chunk += kJoinBlocks) {
        const int q = chunk * 256 + lane * 4;
        const int n = tj * C::TN + q / C::TM, m = ti * C::TM + q % C::TM;
        const bool in = n < deal.n_all && m < g.d;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (in) {
            const float* p = g.parts + ((int64_t)wave * deal.rest + t) * (C::TM * C::TN) + q;
#pragma unroll 4
            for (int c = wave; c < cuts; c += 4, p += (int64_t)4 * deal.rest * (C::TM * C::TN))
                v += *reinterpret_cast<const f32x4*>(p);
        }
        part[wave][lane] = v;
        __syncthreads();
        if (wave == 0 && in) {
            v = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
            const int64_t row = g.dh ? g.map[g.from + n] : n;
            const int cnt = min(4, g.d - m);
            const float f = factor_of<C>(g, factor, row);
            if (g.sum) {
                finish_f32<kOutSum>(g, row, m, cnt, v, f);
            } else if (g.out_f32) {
                finish_f32<kOutF32>(g, row, m, cnt, v, f);
            } else {
                const uint2 r = round16<C::F16>(v, f);
                const uint32_t w[2] = {r.x, r.y};
                store16<4>(g, row, m, cnt, w);
            }
        }
        __syncthreads();
    }
}
template <typename C>
__global__ __launch_bounds__(256) void k_join(const Grad g) {
    join_block<C>(g, blockIdx.x);
}
template <typename H, typename W>
__global__ __launch_bounds__(256) void k_joins(const Grad h, const Grad w, int first) {
    if ((int)blockIdx.x < first) join_block<H>(h, blockIdx.x);
    else join_block<W>(w, blockIdx.x - first);
}

// 16-bit dW from its float32 sum over the pieces.
template <bool F16>
__global__ __launch_bounds__(256) void k_convert(const Grad g) {
    const int64_t all = ((int64_t)g.n * g.d + 3) / 4, numel = (int64_t)g.n * g.d;
    const float factor = g.meta->factor[0];
    const float* sum = g.sum;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        const int cnt = (int)(numel - q * 4 < 4 ? numel - q * 4 : 4);
        for (int e = 0; e < cnt; ++e) v[e] = sum[q * 4 + e];
        for (int e = 0; e < cnt; ++e)
            static_cast<uint16_t*>(g.out)[q * 4 + e] =
                F16 ? from_f32<f16_t>(v[e] * factor).bits : from_f32<bf16_t>(v[e] * factor).bits;
    }
}

// ------------------------------------------------------------------ host side
namespace {

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

template <bool F16> using LogitsBig = Cfg<F16, 256, 256, 64, 128, 64, 2, false, false, 4>;
template <bool F16> using LogitsSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, false, false, 4>;
// For few rows the logits' product is one pass over W: one wave a tile and six stages keep
// 120 KB a CU in flight (525 MB for one row in 87 us, 6.0 TB/s; tiles of 128 columns in four
// stages 93 us, three stages 95 us).
template <bool F16> using LogitsRow = Cfg<F16, 64, 32, 64, 32, 64, 6, false, false, 4, true>;
template <bool F16> using HiddenBig = Cfg<F16, 256, 256, 64, 128, 64, 2, true, false, 8>;
template <bool F16> using HiddenSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, true, false, 8>;
template <bool F16> using WeightBig = Cfg<F16, 256, 256, 128, 64, 64, 2, true, true, 4>;
template <bool F16> using WeightSmall = Cfg<F16, 128, 128, 64, 64, 64, 2, true, true, 4>;

// Rows up to which G has two planes.  The gradients' products of so few rows wait for W to
// be read and dW to be written rather than for their operations: dW of 80 x 42438 x 3136,
// 266 MB, takes 121 us, and the 8 n V D operations of two planes 71 at 1.2 PFLOP/s.
constexpr int kTwoPlaneRows = 64;

enum LogitsTile { kRowTile, kSmallTile, kBigTile };

// How a call runs: fixed by its sizes, types, alignment and workspace.
struct Plan {
    int n, v, d, dtype;
    bool train, dh, dw, pack_w, smooth;
    bool forward, backward;  // the stages that this call runs
    int planes;         // of G
    bool halves;        // products of half-precision operands
    bool out_f32;       // gradients in float32
    int64_t dp, ldg;
    int rows, pieces;   // rows of a piece
    LogitsTile tile;
    int slots;
    bool dh_big, dw_big;
    bool pair;          // both gradients' products in one launch
    int dh_parts, dw_parts;
    // byte offsets into the workspace
    size_t o_meta, o_map, o_tgt, o_tlogit, o_losses, o_xtop, o_x, o_w, o_stats, o_sums, o_g, o_wsum, o_parts, o_dw_parts, bytes;
};

// Workgroups that fill the chip: one with a big tile or two with a small one per CU.
constexpr int kCus = 256;
constexpr int slots_of(bool big) { return big ? kCus : 2 * kCus; }

// Measured: a K step of 64 takes 1.7 us on a chip full of big tiles (256 of 256 x 256)
// and about 1.06 us on one full of small ones (512 of 128 x 128, half the products).  So
// big tiles win unless the edges leave more than a fifth of them empty, or there are not
// steps enough to give every workgroup a few.
// And unless the steps (of all segments) are few: with one workgroup per CU nothing runs
// beside the ends of a tile.  dW of 80 rows (two steps) x 42438 x 3136 142 us, with small
// tiles 121; of 512 rows (eight) x 32000 x 2048 107 and 108.
constexpr int kBigGradSteps = 9;
bool big_tile(int64_t m, int64_t n, int64_t steps, int segs) {
    if (steps * segs < kBigGradSteps) return false;
    const int64_t tb = up(m, 256) / 256 * (up(n, 256) / 256), ts = up(m, 128) / 128 * (up(n, 128) / 128);
    return tb * steps >= kCus * kLeastSteps && ts * 10 > tb * 32;
}
// K steps that are run in one piece whatever the tiles: joining costs a launch (5 us),
// what eight steps take where a CU has one small tile.
constexpr int kUncutSteps = 24;
// The same for the logits, whose tiles are whole, by an estimate: the times above, and what
// the ends of a tile take, 7 us a round of big ones and 4 of small ones (256 or fewer small
// ones, one per CU, run a step in 0.6 us).  Measured, big and small: 3740 x 80744 of width
// 128 240 us and 267, 2307 x 91309 of width 64 150 and 162, 309 x 110742 of width 256 63 and
// 48, 80 x 42438 of width 3136 96 and 88, 67 x 97809 of width 1536 115 and 89.  Where the
// two are within a tenth the estimate may miss: 507 x 16747 of width 4096 106 and 112, and
// it takes the small ones.
bool logits_big(int64_t v, int64_t n, int64_t steps) {
    const int64_t tb = up(v, 256) / 256 * (up(n, 256) / 256), ts = up(v, 128) / 128 * (up(n, 128) / 128);
    const double s = (double)steps;
    const double big = (double)((tb + kCus - 1) / kCus) * (1.7 * s + 7.0);
    const int64_t rest = ts % (2 * kCus);
    const double small = (double)(ts / (2 * kCus)) * (1.06 * s + 4.0) +
                         (rest > kCus ? 1.06 * s + 4.0 : rest > 0 ? 0.6 * s + 4.0 : 0.0);
    return big <= small;
}

// Partial tiles that a product of up to `tiles` tiles of `steps` K steps may leave: kMostRounds
// rounds of the chip at most.
int parts_of(int64_t tiles, int64_t steps, int segs, bool big) {
    if (steps * segs <= kUncutSteps) return 0;
    const int64_t cuts = steps / kLeastSteps < kMostCuts ? steps / kLeastSteps : kMostCuts;
    const int64_t rest = tiles < slots_of(big) ? tiles : slots_of(big) - 1;
    if (cuts < 2) return 0;
    return (int)(rest * cuts < kMostRounds * slots_of(big) ? rest * cuts : kMostRounds * slots_of(big));
}
int64_t tiles_of(int64_t m, int64_t n, bool big) {
    const int64_t t = big ? 256 : 128;
    return up(m, t) / t * (up(n, t) / t);
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
    const int stage = t.stage & ~GEFEN_LCE_GRADS_F32;
    if (stage < GEFEN_LCE_WHOLE || stage > GEFEN_LCE_BACKWARD) return fail_inval("%s: unknown stage %d", what, t.stage);
    if (stage == GEFEN_LCE_FORWARD && (t.grad_hidden || t.grad_weight))
        return fail_inval("%s: a forward stage forms no gradients", what);
    if (stage == GEFEN_LCE_BACKWARD && (t.losses || t.loss || (!t.grad_hidden && !t.grad_weight)))
        return fail_inval("%s: a backward stage forms gradients, and no loss", what);
    p->forward = stage != GEFEN_LCE_BACKWARD;
    p->n = (int)t.n;
    p->v = (int)t.v;
    p->d = (int)t.d;
    p->dtype = t.dtype;
    // a forward stage lays its workspace out for either gradient
    p->dh = t.grad_hidden || stage == GEFEN_LCE_FORWARD;
    p->dw = t.grad_weight || stage == GEFEN_LCE_FORWARD;
    p->train = p->dh || p->dw;
    p->backward = p->train && stage != GEFEN_LCE_FORWARD;
    p->smooth = t.label_smoothing > 0.0;
    p->planes = t.dtype == GEFEN_F32 || t.n <= kTwoPlaneRows ? 2 : 1;
    p->halves = t.dtype != GEFEN_BF16;
    p->out_f32 = t.dtype == GEFEN_F32 || (t.stage & GEFEN_LCE_GRADS_F32);
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
    if (stage && p->pieces > 1) return fail_inval("%s: stages of %d pieces of rows", what, p->pieces);
    const int64_t n = t.n < rows ? (t.n > 0 ? t.n : 1) : rows;
    const int64_t in_steps = p->dp / 64 * (t.dtype == GEFEN_F32 ? 3 : 1);
    p->tile = n <= 32 ? kRowTile : logits_big(t.v, n, in_steps) ? kBigTile : kSmallTile;
    p->slots = (int)(up(t.v, kSlot) / kSlot);
    const int segs = t.dtype == GEFEN_F32 ? 3 : p->planes;
    p->dh_big = big_tile(t.d, n, up(t.v, 64) / 64, segs);
    p->dw_big = big_tile(t.d, t.v, up(n, 64) / 64, segs);

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
    p->o_xtop = t.dtype == GEFEN_F32 ? take(n_up * 4) : at;
    p->o_x = take((size_t)in_planes * p->rows * p->pieces * p->dp * 2);
    p->o_w = p->pack_w ? take((size_t)in_planes * p->v * p->dp * 2) : at;
    p->o_stats = take((size_t)p->rows * p->slots * sizeof(float2));
    p->o_sums = p->smooth ? take((size_t)p->rows * p->slots * 4) : at;
    p->o_g = p->train ? take((size_t)p->planes * p->rows * p->ldg * 2) : at;
    // float32 gradients are their own sum over the pieces
    p->o_wsum = p->dw && p->pieces > 1 && !p->out_f32 ? take((size_t)p->v * p->d * 4) : at;
    p->dh_parts = p->dh ? parts_of(tiles_of(t.d, n, p->dh_big), up(t.v, 64) / 64, segs, p->dh_big) : 0;
    p->dw_parts = p->dw ? parts_of(tiles_of(t.d, t.v, p->dw_big), up(n, 64) / 64, segs, p->dw_big) : 0;
    const size_t dh_bytes = (size_t)p->dh_parts * (p->dh_big ? 256 * 256 : 128 * 128) * 4;
    const size_t dw_bytes = (size_t)p->dw_parts * (p->dw_big ? 256 * 256 : 128 * 128) * 4;
    p->pair = p->dh && p->dw && !p->dh_big && !p->dw_big && p->pieces == 1 && t.n > 0;
    p->o_parts = take(p->pair ? dh_bytes + dw_bytes : dh_bytes > dw_bytes ? dh_bytes : dw_bytes);
    p->o_dw_parts = p->o_parts + (p->pair ? dh_bytes : 0);
    p->bytes = at;
    return GEFEN_OK;
}

template <typename C>
void launch_logits(Logits a, int most, hipStream_t st) {
    a.tiles_m = (a.v + C::TM - 1) / C::TM;
    const int tiles = a.tiles_m * ((most + C::TN - 1) / C::TN), slots = kCus * C::WGS;
    const dim3 grid((unsigned)(tiles < slots ? tiles : slots)), wg(C::TT);
    if (!a.g) hipLaunchKernelGGL((k_logits<C, kKeepNone>), grid, wg, 0, st, a);
    else if (a.planes == 1) hipLaunchKernelGGL((k_logits<C, kKeepPacked>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((k_logits<C, kKeepPlanes>), grid, wg, 0, st, a);
}
template <bool F16>
void launch_logits_tile(const Plan& p, const Logits& a, int most, hipStream_t st) {
    if (p.tile == kBigTile) launch_logits<LogitsBig<F16>>(a, most, st);
    else if (p.tile == kSmallTile) launch_logits<LogitsSmall<F16>>(a, most, st);
    else launch_logits<LogitsRow<F16>>(a, most, st);
}
// Workers for g.n rows, the most that the device may find.
template <typename C>
int grad_grid(Grad* g, int* join) {
    g->tiles_m = (g->d + C::TM - 1) / C::TM;
    const int tiles = g->tiles_m * ((g->n + C::TN - 1) / C::TN);
    *join = g->most_parts == 0 ? 0 : tiles < g->slots ? tiles : g->slots - 1;
    const int units = tiles + g->most_parts;
    return units < g->slots ? units : g->slots;
}
template <typename C>
void launch_grad(Grad g, const Loss& l, hipStream_t st) {
    int join;
    const int grid = grad_grid<C>(&g, &join) + (l.out ? 1 : 0);
    hipLaunchKernelGGL(k_grad<C>, dim3((unsigned)grid), dim3(C::TT), 0, st, g, l);
    if (join) hipLaunchKernelGGL(k_join<C>, dim3((unsigned)join, kJoinBlocks), dim3(256), 0, st, g);
}
template <bool F16>
void launch_grad_tile(Grad g, bool big, const Loss& l, hipStream_t st) {
    if (g.dh) {
        if (big) launch_grad<HiddenBig<F16>>(g, l, st);
        else launch_grad<HiddenSmall<F16>>(g, l, st);
    } else {
        if (big) launch_grad<WeightBig<F16>>(g, l, st);
        else launch_grad<WeightSmall<F16>>(g, l, st);
    }
}
template <bool F16>
void launch_grad_pair(Grad h, Grad w, const Loss& l, hipStream_t st) {
    using H = HiddenSmall<F16>;
    using W = WeightSmall<F16>;
    int join_h, join_w;
    const int first = grad_grid<H>(&h, &join_h);
    const int grid = first + grad_grid<W>(&w, &join_w) + (l.out ? 1 : 0);
    hipLaunchKernelGGL((k_grads<H, W>), dim3((unsigned)grid), dim3(H::TT), 0, st, h, w, l, first);
    if (join_h + join_w)
        hipLaunchKernelGGL((k_joins<H, W>), dim3((unsigned)(join_h + join_w), kJoinBlocks), dim3(256), 0, st,
                           h, w, join_h);
}
unsigned grid_of(int64_t chunks, int64_t most) {
    const int64_t wg = (chunks + 255) / 256;
    return (unsigned)(wg < 1 ? 1 : wg > most ? most : wg);
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
    const int size = dtype_size(t.dtype), grad_size = p.out_f32 ? 4 : 2;
    if (!aligned(t.hidden, size) || !aligned(t.weight, size) || !aligned(t.grad_hidden, grad_size) ||
        !aligned(t.grad_weight, grad_size) || !aligned(t.targets, t.targets_int32 ? 4 : 8))
        return fail_inval("%s: an operand is not aligned to its elements", what);
    if (t.n && !t.losses && !t.loss && !p.train) return fail_inval("%s: nothing to compute", what);
    if (t.loss && t.reduction == GEFEN_REDUCE_NONE) return fail_inval("%s: no reduction for a loss", what);
    if (t.reduction == GEFEN_REDUCE_NONE && p.backward && t.n && !t.grad)
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
    uint32_t* x_top = t.dtype == GEFEN_F32 ? reinterpret_cast<uint32_t*>(ws + p.o_xtop) : nullptr;
    uint16_t* gbuf = reinterpret_cast<uint16_t*>(ws + p.o_g);
    const bool by_row = p.backward && t.reduction == GEFEN_REDUCE_NONE;
    const bool shift = p.backward && p.dw && (t.dtype == GEFEN_F32 || (by_row && t.dtype == GEFEN_F16));
    const int carry = !p.halves ? kCarryAll : p.planes == 2 ? kCarryTwo : kCarryOne;

    const Select sel{t.targets, t.targets_int32, p.n, p.v, t.ignore_index, by_row ? t.grad : nullptr, map, tgt, meta,
                     !p.forward};
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
    pk.rows = x_rows;
    pk.map = map;
    pk.meta = meta;
    pk.which = 0;
    pk.zero_losses = losses;
    pk.row_top = x_top;
    pk.row_grad = by_row ? t.grad : nullptr;
    pk.carry = carry;
    Pack pw{};
    pw.src = t.weight;
    pw.row_stride = t.weight_row_stride;
    pw.col_stride = t.weight_col_stride;
    pw.n = p.v;
    pw.d = p.d;
    pw.dp = (int)p.dp;
    pw.dst = wp;
    pw.f32 = pk.f32;
    pw.plane = (int64_t)p.v * p.dp;
    pw.rows = p.v;
    pw.meta = meta;
    pw.which = 1;
    const int pack_x = (int)grid_of(x_rows * (p.dp / 8), 8192);
    const int pack_w = p.pack_w ? (int)grid_of(p.v * (p.dp / 8), 8192) : 0;
    const int64_t per = (p.d + 7) / 8;
    const Top tx{t.hidden, t.hidden_row_stride, t.hidden_col_stride, p.n, p.d, map, meta, 0, t.dtype == GEFEN_F16, x_top};
    const int top_x = (int)grid_of(p.n * per / 4, kTopGrid);
    if (!p.forward) {
        if (by_row) hipLaunchKernelGGL(k_rows, dim3(1), dim3(kRowsThreads), 0, st, sel);
    } else if (p.n <= kSelfRows && !pk.f32) {
        hipLaunchKernelGGL(k_select_pack, dim3((unsigned)(pack_x + pack_w)), dim3(256), 0, st, sel, pk, pw, pack_x);
    } else {
        hipLaunchKernelGGL(k_rows, dim3(1), dim3(kRowsThreads), 0, st, sel);
        if (pk.f32) {
            const Top tw{t.weight, t.weight_row_stride, t.weight_col_stride, p.v, p.d, nullptr, meta, 1, 0, nullptr};
            const int top_w = (int)grid_of(p.v * per / 4, kTopGrid);
            hipLaunchKernelGGL(k_top, dim3((unsigned)(top_x + top_w)), dim3(kTopThreads), 0, st, tx, tw, top_x);
        }
        hipLaunchKernelGGL(k_pack, dim3((unsigned)(pack_x + pack_w)), dim3(256), 0, st, pk, pw, pack_x);
    }
    if (shift && !pk.f32)
        hipLaunchKernelGGL(k_top, dim3((unsigned)top_x), dim3(kTopThreads), 0, st, tx, tx, top_x);
    Operand w{};
    w.p = p.pack_w ? wp : static_cast<const uint16_t*>(t.weight);
    w.ld = p.pack_w ? p.dp : t.weight_row_stride;
    w.plane = (int64_t)p.v * p.dp;
    // segments of the logits' product: low x high, high x low, high x high
    w.planes = pk.f32 ? 1 | 2 << 2 | 0 << 4 : 0;
    w.rows = p.v;
    w.cols = (int)p.dp;

    Loss loss{losses, p.n, t.reduction == GEFEN_REDUCE_MEAN, meta, t.loss};
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
        l.row_top = x_top;
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
            if (p.forward) {
                if (f16) launch_logits_tile<true>(p, l, most, st);
                else launch_logits_tile<false>(p, l, most, st);
            }
            Rows r{};
            r.stats = l.stats;
            r.sums = l.sums;
            r.target_logit = l.target_logit;
            r.tgt = tgt;
            r.map = map;
            r.meta = meta;
            r.row_grad = by_row ? t.grad : nullptr;
            r.grad = by_row ? nullptr : t.grad;
            r.mean = t.reduction == GEFEN_REDUCE_MEAN;
            r.dtype = t.dtype;
            r.carry = carry;
            r.losses = losses;
            r.g = p.backward ? l.g : nullptr;
            r.ldg = p.ldg;
            r.g_plane = l.g_plane;
            r.v = p.v;
            r.slots = p.slots;
            r.from = from;
            r.most = most;
            r.planes = p.planes;
            r.smoothing = (float)t.label_smoothing;
            r.zero_rows = p.backward ? t.grad_hidden : nullptr;
            r.zero_bytes = (int64_t)p.d * grad_size;
            // a row per workgroup, or parts of it where the rows do not fill the chip
            const int64_t rows_up = p.backward ? up(most, 64) : most;
            int64_t parts = p.backward ? 2048 / rows_up : 1;
            const int64_t chunks = p.ldg / 8 / kGradThreads;
            if (parts > chunks) parts = chunks;
            if (parts < 1) parts = 1;
            const dim3 grid((unsigned)rows_up, (unsigned)parts);
            const bool stream_past = p.backward && (int64_t)p.planes * most * p.ldg * 2 > kKeepBytes;
            auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kGradThreads), 0, st, r); };
            if (f16) stream_past ? launch(k_gradient_rows<true, true>) : launch(k_gradient_rows<true, false>);
            else stream_past ? launch(k_gradient_rows<false, true>) : launch(k_gradient_rows<false, false>);
            if (shift) {
                pk.from = from;
                pk.most = most;
                hipLaunchKernelGGL(k_shift, dim3(grid_of(most * (p.dp / 8), 8192)), dim3(256), 0, st, pk);
            }
        }
        if (!p.backward) continue;
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
        g.out_f32 = p.out_f32;
        // the loss goes with the last launch of the last piece
        const bool last = piece == p.pieces - 1;
        Loss with{};
        if (last && (p.dw || most > 0)) std::swap(with, loss);
        g.b = go;
        Grad h = g, wg = g;
        h.parts = reinterpret_cast<float*>(ws + p.o_parts);
        h.most_parts = p.dh_parts;
        h.slots = slots_of(p.dh_big);
        h.a = w;
        h.dh = 1;
        h.n = most;
        h.steps = (p.v + 63) / 64;
        h.out = t.grad_hidden;
        h.row_grad = by_row ? t.grad : nullptr;
        h.carry = carry;
        wg.parts = reinterpret_cast<float*>(ws + p.o_dw_parts);
        wg.most_parts = p.dw_parts;
        wg.slots = slots_of(p.dw_big);
        wg.a = xo;
        wg.a.planes = w.planes;
        wg.dh = 0;
        wg.n = p.v;
        wg.sum = p.pieces == 1 ? nullptr
                 : p.out_f32   ? static_cast<float*>(t.grad_weight)
                               : reinterpret_cast<float*>(ws + p.o_wsum);
        wg.first = piece == 0;
        wg.last = last && p.out_f32;
        wg.out = t.grad_weight;
        if (p.pair) {
            if (f16) launch_grad_pair<true>(h, wg, with, st);
            else launch_grad_pair<false>(h, wg, with, st);
            continue;
        }
        if (p.dh && most > 0) {
            if (f16) launch_grad_tile<true>(h, p.dh_big, p.dw ? Loss{} : with, st);
            else launch_grad_tile<false>(h, p.dh_big, p.dw ? Loss{} : with, st);
        }
        if (p.dw) {
            if (f16) launch_grad_tile<true>(wg, p.dw_big, with, st);
            else launch_grad_tile<false>(wg, p.dw_big, with, st);
            if (wg.sum && last && !p.out_f32) {
                const dim3 grid(grid_of(((int64_t)p.v * p.d + 3) / 4, 8192));
                if (f16) hipLaunchKernelGGL(k_convert<true>, grid, dim3(256), 0, st, wg);
                else hipLaunchKernelGGL(k_convert<false>, grid, dim3(256), 0, st, wg);
            }
        }
    }
    if (loss.out) hipLaunchKernelGGL(k_loss, dim3(1), dim3(1024), 0, st, loss);
    return launch_status(what);
}
