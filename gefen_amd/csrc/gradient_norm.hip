// Global norm of many gradients and clipping to a bound.
//
//   t = (sum |g|^2)^(1/2), sum |g| or max |g| over every element of every tensor
//   c = min(1, max_norm / (t + 1e-6)),  dst = c * src
//
// Both passes are bound by HBM: the norm reads each gradient once, clipping reads
// and writes it once more.  Tensors are cut into chunks of kChunk elements; a launch
// takes up to kTable tensors (their table travels in the kernel arguments) and its
// workgroups walk the chunks in strides of the grid.  Each workgroup leaves one
// float64 partial in its own slot and the partials are added in a fixed order, so a
// norm does not depend on how the workgroups were scheduled.
//
// Squares are summed in float64: the square of a float32 is exact there, so a norm
// neither overflows for gradients above 1.8e19 nor loses those below 1e-23, and no
// order of summation matters within float32's precision.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "capi_internal.h"
#include "common.h"

namespace gefen {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384, kSmallChunk = 2048;
constexpr int kTable = 128;       // tensors per launch: the table fits the 4 KB of kernel arguments
constexpr int64_t kKeepBytes = 192 << 20;
constexpr int kGrid = 2048;         // workgroups of a launch (8 per CU)
constexpr int kMaxPartials = 8192;  // workgroups of all norm launches together, about
constexpr int kJoinInClip = 2048;   // partials that every scaling workgroup adds up itself

enum NormKind { kNormMax = 0, kNormAbs = 1, kNormSquare = 2 };

struct Table {
    const void* src[kTable];
    void* dst[kTable];
    int64_t numel[kTable];
    int32_t first[kTable];  // first chunk of each tensor
    uint8_t src_dtype[kTable], dst_dtype[kTable];
    int32_t count, chunks;
};

// The tensor that chunk c belongs to (c is uniform over the workgroup).
__device__ __forceinline__ int tensor_of(const Table& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <int KIND>
struct Acc {
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    float m = 0.0f;
    __device__ __forceinline__ void add(float x, int k) {
        if constexpr (KIND == kNormMax) m = nanmax(m, fabsf(x));
        else if constexpr (KIND == kNormAbs) v[k & 3] += (double)fabsf(x);
        else v[k & 3] = __builtin_fma((double)x, (double)x, v[k & 3]);
    }
    __device__ __forceinline__ double total() const {
        if constexpr (KIND == kNormMax) return (double)m;
        else return (v[0] + v[1]) + (v[2] + v[3]);
    }
};
template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (KIND == kNormMax) return (b > a || b != b) ? b : a;
    else return a + b;
}
template <int KIND>
__device__ __forceinline__ double block_join(double x) {
    __shared__ double part[kThreads / 64];
    for (int off = 32; off > 0; off >>= 1) x = join<KIND>(x, __shfl_xor(x, off, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
    for (int w = 1; w < kThreads / 64; ++w) x = join<KIND>(x, part[w]);
    __syncthreads();
    return x;
}

// W elements at any alignment; STREAM: with the non-temporal hint, for what is not read
// again before it has left every cache.
template <typename T, int W, bool STREAM>
__device__ __forceinline__ AnyVec<T, W> load_any(const T* p) {
    using R = typename RawAny<sizeof(T) * W, sizeof(T)>::type;
    const R* q = reinterpret_cast<const R*>(p);
    const typename RawVec<sizeof(T) * W>::type r = STREAM ? __builtin_nontemporal_load(q) : *q;
    AnyVec<T, W> x;
    __builtin_memcpy(&x, &r, sizeof(x));
    return x;
}
template <typename T, int W, bool STREAM>
__device__ __forceinline__ void store_any(T* p, const AnyVec<T, W>& x) {
    using R = typename RawAny<sizeof(T) * W, sizeof(T)>::type;
    typename RawVec<sizeof(T) * W>::type r;
    __builtin_memcpy(&r, &x, sizeof(r));
    if (STREAM) __builtin_nontemporal_store(r, reinterpret_cast<R*>(p));
    else *reinterpret_cast<R*>(p) = r;
}

// n elements (n <= kChunk) at p into the accumulator.
template <int KIND, bool STREAM, typename T>
__device__ __forceinline__ void norm_chunk(const T* __restrict__ p, int n, Acc<KIND>& acc) {
    constexpr int W = 16 / sizeof(T);  // one 16-byte load, at any alignment
    constexpr int kVecs = kChunk / W / kThreads;
    if (n == kChunk) {
        AnyVec<T, W> x[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
            x[i] = load_any<T, W, STREAM>(p + (i * kThreads + (int)threadIdx.x) * W);
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) acc.add(to_f32(x[i].v[e]), e);
    } else {
        const int whole = n / W;
        for (int i = threadIdx.x; i < whole; i += kThreads) {
            const AnyVec<T, W> x = load_any<T, W, STREAM>(p + i * W);
#pragma unroll
            for (int e = 0; e < W; ++e) acc.add(to_f32(x.v[e]), e);
        }
        const int e = whole * W + (int)threadIdx.x;
        if (e < n) acc.add(to_f32(p[e]), 0);
    }
}

template <int KIND>
__device__ __forceinline__ float norm_of(double joined) {
    return KIND == kNormSquare ? (float)sqrt(joined) : (float)joined;
}

// partial[blockIdx.x] of this launch; with norm set (a launch of one workgroup that
// is the only one) the norm itself.
template <int KIND, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_norm_part(const Table t, double* __restrict__ partial,
                                                        float* __restrict__ norm) {
    Acc<KIND> acc;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const int64_t at = (int64_t)(c - t.first[k]) * kChunk;
        const int64_t left = t.numel[k] - at;
        const int n = left < kChunk ? (int)left : kChunk;
        const int dt = t.src_dtype[k];
        if (dt == GEFEN_F32) norm_chunk<KIND, STREAM>(static_cast<const float*>(t.src[k]) + at, n, acc);
        else if (dt == GEFEN_BF16) norm_chunk<KIND, STREAM>(static_cast<const bf16_t*>(t.src[k]) + at, n, acc);
        else norm_chunk<KIND, STREAM>(static_cast<const f16_t*>(t.src[k]) + at, n, acc);
    }
    const double s = block_join<KIND>(acc.total());
    if (threadIdx.x == 0) {
        if (norm) *norm = norm_of<KIND>(s);
        else partial[blockIdx.x] = s;
    }
}

template <int KIND>
__device__ __forceinline__ float joined_norm(const double* __restrict__ partial, int count) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += kThreads) s = join<KIND>(s, partial[i]);
    return norm_of<KIND>(block_join<KIND>(s));
}

template <int KIND>
__global__ __launch_bounds__(kThreads) void k_norm_join(const double* __restrict__ partial, int count,
                                                        float* __restrict__ norm) {
    const float t = joined_norm<KIND>(partial, count);
    if (threadIdx.x == 0) *norm = t;
}

template <bool STREAM, typename S, typename D>
__device__ __forceinline__ void scale_chunk(const S* src, D* dst, int n, float c) {
    constexpr int W = 16 / (sizeof(S) > sizeof(D) ? sizeof(S) : sizeof(D));
    constexpr int kVecs = kChunk / W / kThreads;
    constexpr int kBatch = 8;  // loads in flight per thread
    auto scaled = [&](const AnyVec<S, W>& x) {
        AnyVec<D, W> y;
#pragma unroll
        for (int e = 0; e < W; ++e) y.v[e] = from_f32<D>(to_f32(x.v[e]) * c);
        return y;
    };
    if (n == kChunk) {
#pragma unroll
        for (int i0 = 0; i0 < kVecs; i0 += kBatch) {
            AnyVec<S, W> x[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                x[i] = load_any<S, W, STREAM>(src + ((i0 + i) * kThreads + (int)threadIdx.x) * W);
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                store_any<D, W, STREAM>(dst + ((i0 + i) * kThreads + (int)threadIdx.x) * W, scaled(x[i]));
        }
    } else {
        const int whole = n / W;
        for (int i = threadIdx.x; i < whole; i += kThreads)
            store_any<D, W, STREAM>(dst + i * W, scaled(load_any<S, W, STREAM>(src + i * W)));
        const int e = whole * W + (int)threadIdx.x;
        if (e < n) dst[e] = from_f32<D>(to_f32(src[e]) * c);
    }
}
template <bool STREAM, typename S>
__device__ __forceinline__ void scale_chunk_to(const S* src, void* dst, int dt, int64_t at, int n, float c) {
    if (dt == GEFEN_F32) scale_chunk<STREAM>(src + at, static_cast<float*>(dst) + at, n, c);
    else if (dt == GEFEN_BF16) scale_chunk<STREAM>(src + at, static_cast<bf16_t*>(dst) + at, n, c);
    else scale_chunk<STREAM>(src + at, static_cast<f16_t*>(dst) + at, n, c);
}

// Bound by HBM: 1.5e9 float32 gradients into bf16 ones 1.58 ms (5.7 TB/s), after a norm of
// 0.9 ms (6.8 TB/s).
// dst = c * src.  Every workgroup joins the partials itself (16 KB at most, from L2),
// which saves a launch between the two passes; partial == nullptr: *norm is given.
// Chunks are walked from the last to the first: the norm pass read those last, so
// what the memory-side cache still holds of them is read from there.  A coefficient
// of one leaves tensors that are scaled in place untouched.
template <int KIND, bool STREAM>
__global__ __launch_bounds__(kThreads) void k_clip(const Table t, const double* __restrict__ partial, int count,
                                                   float* norm, float max_norm) {
    float total;
    if (partial) {
        total = joined_norm<KIND>(partial, count);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    } else {
        total = *norm;
    }
    float c = max_norm / (total + 1e-6f);
    if (c > 1.0f) c = 1.0f;  // NaN stays NaN, as clamp(max=1) leaves it
    for (int b = blockIdx.x; b < t.chunks; b += gridDim.x) {
        const int ch = t.chunks - 1 - b;
        const int k = tensor_of(t, ch);
        if (c == 1.0f && t.src[k] == t.dst[k]) continue;
        const int64_t at = (int64_t)(ch - t.first[k]) * kChunk;
        const int64_t left = t.numel[k] - at;
        const int n = left < kChunk ? (int)left : kChunk;
        const int sd = t.src_dtype[k], dd = t.dst_dtype[k];
        if (sd == GEFEN_F32) scale_chunk_to<STREAM>(static_cast<const float*>(t.src[k]), t.dst[k], dd, at, n, c);
        else if (sd == GEFEN_BF16) scale_chunk_to<STREAM>(static_cast<const bf16_t*>(t.src[k]), t.dst[k], dd, at, n, c);
        else scale_chunk_to<STREAM>(static_cast<const f16_t*>(t.src[k]), t.dst[k], dd, at, n, c);
    }
}

// a and b times *factor (a loss's own gradient), in chunks over both.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_scale_by(T* a, int64_t na, T* b, int64_t nb,
                                                       const float* __restrict__ factor) {
    const float f = *factor;
    if (f == 1.0f) return;
    const int64_t ca = (na + kChunk - 1) / kChunk, cb = (nb + kChunk - 1) / kChunk;
    for (int64_t c = blockIdx.x; c < ca + cb; c += gridDim.x) {
        T* p = c < ca ? a + c * kChunk : b + (c - ca) * kChunk;
        const int64_t left = c < ca ? na - c * kChunk : nb - (c - ca) * kChunk;
        scale_chunk<true>(static_cast<const T*>(p), p, left < kChunk ? (int)left : kChunk, f);
    }
}

// Float32 a and b times *factor into a_out and b_out, in chunks of up to kChunk.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_scale_from(const float* a, T* a_out, int64_t na, const float* b, T* b_out,
                                                         int64_t nb, const float* __restrict__ factor, int chunk) {
    const float f = *factor;
    const int64_t ca = (na + chunk - 1) / chunk, cb = (nb + chunk - 1) / chunk;
    for (int64_t c = blockIdx.x; c < ca + cb; c += gridDim.x) {
        const bool first = c < ca;
        const int64_t at = (first ? c : c - ca) * chunk, left = (first ? na : nb) - at;
        scale_chunk<true>((first ? a : b) + at, (first ? a_out : b_out) + at, left < chunk ? (int)left : chunk, f);
    }
}

int64_t chunks_of(const gefen_gradient_task& t) { return (t.numel + kChunk - 1) / kChunk; }

// The launches of a call: tables of up to kTable tensors and 2^30 chunks, empty tensors left out.
struct Launches {
    const gefen_gradient_task* tasks;
    int num, next = 0;
    bool fill(Table* t) {
        t->count = 0;
        int64_t chunks = 0;
        for (; next < num && t->count < kTable; ++next) {
            const gefen_gradient_task& g = tasks[next];
            if (g.numel == 0) continue;
            if (t->count && chunks + chunks_of(g) > (1 << 30)) break;
            t->src[t->count] = g.src;
            t->dst[t->count] = g.dst;
            t->numel[t->count] = g.numel;
            t->first[t->count] = (int32_t)chunks;
            t->src_dtype[t->count] = (uint8_t)g.src_dtype;
            t->dst_dtype[t->count] = (uint8_t)g.dst_dtype;
            chunks += chunks_of(g);
            ++t->count;
        }
        t->chunks = (int32_t)chunks;
        return t->count > 0;
    }
};

int check_tasks(const gefen_gradient_task* tasks, int num, bool dst, const char* what) {
    if (num < 0 || (num && !tasks)) return fail_inval("%s: no tasks", what);
    for (int i = 0; i < num; ++i) {
        const gefen_gradient_task& g = tasks[i];
        if (g.numel < 0 || g.numel > ((int64_t)1 << 44)) return fail_inval("%s: task %d has %lld elements", what, i, (long long)g.numel);
        if (!valid_dtype(g.src_dtype) || (dst && !valid_dtype(g.dst_dtype)))
            return fail_inval("%s: task %d has an unknown dtype", what, i);
        if (g.numel && (!g.src || (dst && !g.dst))) return fail_inval("%s: task %d has a null pointer", what, i);
        if (!aligned(g.src, dtype_size(g.src_dtype)) || (dst && !aligned(g.dst, dtype_size(g.dst_dtype))))
            return fail_inval("%s: task %d is not aligned to its elements", what, i);
        if (dst && g.numel && g.src == g.dst && g.src_dtype != g.dst_dtype)
            return fail_inval("%s: task %d scales in place into another dtype", what, i);
    }
    return GEFEN_OK;
}

int norm_kind(double norm_type) {
    if (norm_type == 2.0) return kNormSquare;
    if (norm_type == 1.0) return kNormAbs;
    if (norm_type == INFINITY) return kNormMax;
    return -1;
}

// Workgroups of a norm launch: all launches of a call share about kMaxPartials by their chunks.
int norm_grid(int chunks, int64_t all) {
    const int64_t share = all <= kMaxPartials ? chunks : ((int64_t)chunks * kMaxPartials + all - 1) / all;
    return (int)(share < 1 ? 1 : share > kGrid ? kGrid : share);
}
int64_t all_chunks(const gefen_gradient_task* tasks, int num) {
    int64_t all = 0;
    for (int i = 0; i < num; ++i) all += chunks_of(tasks[i]);
    return all;
}

// Gradients that the memory-side cache (256 MB) holds between the norm and the scaling are
// better left to it; larger sets are streamed past the caches: a norm of 16 GB reads at
// 7.1 TB/s with the hint and at 6.3 without.
bool stream_past(const gefen_gradient_task* tasks, int num) {
    int64_t bytes = 0;
    for (int i = 0; i < num; ++i) bytes += tasks[i].numel * dtype_size(tasks[i].src_dtype);
    return bytes > kKeepBytes;
}

template <int KIND>
int run_norm(const gefen_gradient_task* tasks, int num, double* partial, float* norm, bool join, int* count,
             hipStream_t st) {
    const int64_t all = all_chunks(tasks, num);
    Launches ls{tasks, num};
    Table t;
    int at = 0;
    const bool single = join && all == 1;
    const bool stream = join || stream_past(tasks, num);  // a norm alone reads once
    while (ls.fill(&t)) {
        const int grid = norm_grid(t.chunks, all);
        float* out = single ? norm : nullptr;
        if (stream) hipLaunchKernelGGL((k_norm_part<KIND, true>), dim3(grid), dim3(kThreads), 0, st, t, partial + at, out);
        else hipLaunchKernelGGL((k_norm_part<KIND, false>), dim3(grid), dim3(kThreads), 0, st, t, partial + at, out);
        at += grid;
    }
    // a scaling that follows joins few partials itself
    if ((join && !single) || at > kJoinInClip)
        hipLaunchKernelGGL(k_norm_join<KIND>, dim3(1), dim3(kThreads), 0, st, partial, at, norm);
    *count = at;
    return launch_status("gefen_gradient_norm");
}

template <int KIND>
int run_clip(const gefen_gradient_task* tasks, int num, const double* partial, int count, float* norm, float max_norm,
             hipStream_t st) {
    // the launches of the norm in reverse, as the chunks inside each are
    int starts[64], n = 0;
    Launches ls{tasks, num};
    Table t;
    int from = 0;
    const bool stream = stream_past(tasks, num);
    // runs of up to 64 launches are reversed; more tensors than that go in runs
    while (from < num) {
        n = 0;
        ls.next = from;
        while (n < 64) {
            const int s = ls.next;
            if (!ls.fill(&t)) break;
            starts[n++] = s;
        }
        const int end = ls.next;
        for (int i = n - 1; i >= 0; --i) {
            ls.next = starts[i];
            ls.fill(&t);
            const int grid = t.chunks < kGrid ? t.chunks : kGrid;
            if (stream)
                hipLaunchKernelGGL((k_clip<KIND, true>), dim3(grid), dim3(kThreads), 0, st, t, partial, count, norm,
                                   max_norm);
            else
                hipLaunchKernelGGL((k_clip<KIND, false>), dim3(grid), dim3(kThreads), 0, st, t, partial, count, norm,
                                   max_norm);
        }
        if (n == 0) break;
        from = end;
    }
    return launch_status("gefen_clip_gradients");
}

}  // namespace
}  // namespace gefen

using namespace gefen;

extern "C" size_t gefen_gradient_norm_workspace_size(const gefen_gradient_task* tasks, int num_tasks) {
    if (num_tasks < 0 || (num_tasks && !tasks)) return 0;
    // one float64 per workgroup: the shares of kMaxPartials rounded up once per launch
    const int64_t all = all_chunks(tasks, num_tasks);
    const int64_t launches = num_tasks / kTable + 2 + (all >> 30);
    return (size_t)((all < kMaxPartials ? all : kMaxPartials) + launches) * sizeof(double);
}

extern "C" int gefen_gradient_norm(const gefen_gradient_task* tasks, int num_tasks, double norm_type, float* norm,
                                   void* workspace, gefen_stream_t stream) {
    const int bad = check_tasks(tasks, num_tasks, false, "gefen_gradient_norm");
    if (bad) return bad;
    const int kind = norm_kind(norm_type);
    if (kind < 0) return fail_inval("gefen_gradient_norm: norm_type must be 1, 2 or infinity, got %g", norm_type);
    if (!norm || !workspace) return fail_inval("gefen_gradient_norm: null output or workspace");
    double* partial = static_cast<double*>(workspace);
    int count = 0;
    if (kind == kNormSquare) return run_norm<kNormSquare>(tasks, num_tasks, partial, norm, true, &count, stream);
    if (kind == kNormAbs) return run_norm<kNormAbs>(tasks, num_tasks, partial, norm, true, &count, stream);
    return run_norm<kNormMax>(tasks, num_tasks, partial, norm, true, &count, stream);
}

extern "C" int gefen_clip_gradients(const gefen_gradient_task* tasks, int num_tasks, double norm_type, double max_norm,
                                    float* norm, void* workspace, gefen_stream_t stream) {
    const int bad = check_tasks(tasks, num_tasks, true, "gefen_clip_gradients");
    if (bad) return bad;
    const int kind = norm_kind(norm_type);
    if (kind < 0) return fail_inval("gefen_clip_gradients: norm_type must be 1, 2 or infinity, got %g", norm_type);
    if (!norm || !workspace) return fail_inval("gefen_clip_gradients: null norm or workspace");
    if (!(max_norm >= 0.0)) return fail_inval("gefen_clip_gradients: max_norm must not be negative, got %g", max_norm);
    double* partial = static_cast<double*>(workspace);
    int count = 0;
    auto run = [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        const bool none = all_chunks(tasks, num_tasks) == 0;  // no scaling launch to write the norm
        const int rc = run_norm<KIND>(tasks, num_tasks, partial, norm, none, &count, stream);
        if (rc) return rc;
        return run_clip<KIND>(tasks, num_tasks, count > kJoinInClip ? nullptr : partial, count, norm, (float)max_norm,
                              stream);
    };
    if (kind == kNormSquare) return run(std::integral_constant<int, kNormSquare>());
    if (kind == kNormAbs) return run(std::integral_constant<int, kNormAbs>());
    return run(std::integral_constant<int, kNormMax>());
}

extern "C" int gefen_scale_gradients(const gefen_gradient_task* tasks, int num_tasks, const float* norm,
                                     double max_norm, gefen_stream_t stream) {
    const int bad = check_tasks(tasks, num_tasks, true, "gefen_scale_gradients");
    if (bad) return bad;
    if (!norm) return fail_inval("gefen_scale_gradients: null norm");
    if (!(max_norm >= 0.0)) return fail_inval("gefen_scale_gradients: max_norm must not be negative, got %g", max_norm);
    return run_clip<kNormSquare>(tasks, num_tasks, nullptr, 0, const_cast<float*>(norm), (float)max_norm, stream);
}

extern "C" int gefen_scale_by(void* a, int64_t a_numel, void* b, int64_t b_numel, int dtype, const float* factor,
                              gefen_stream_t stream) {
    if (!valid_dtype(dtype)) return fail_inval("gefen_scale_by: unknown dtype %d", dtype);
    if (a_numel < 0 || b_numel < 0 || (a_numel && !a) || (b_numel && !b) || !factor)
        return fail_inval("gefen_scale_by: null pointer or negative size");
    const int size = dtype_size(dtype);
    if (!aligned(a, size) || !aligned(b, size)) return fail_inval("gefen_scale_by: not aligned to its elements");
    const int64_t chunks = (a_numel + kChunk - 1) / kChunk + (b_numel + kChunk - 1) / kChunk;
    if (!chunks) return GEFEN_OK;
    const dim3 grid((unsigned)(chunks < kGrid ? chunks : kGrid)), wg(kThreads);
    if (dtype == GEFEN_F32)
        hipLaunchKernelGGL(k_scale_by<float>, grid, wg, 0, stream, static_cast<float*>(a), a_numel,
                           static_cast<float*>(b), b_numel, factor);
    else if (dtype == GEFEN_BF16)
        hipLaunchKernelGGL(k_scale_by<bf16_t>, grid, wg, 0, stream, static_cast<bf16_t*>(a), a_numel,
                           static_cast<bf16_t*>(b), b_numel, factor);
    else
        hipLaunchKernelGGL(k_scale_by<f16_t>, grid, wg, 0, stream, static_cast<f16_t*>(a), a_numel,
                           static_cast<f16_t*>(b), b_numel, factor);
    return launch_status("gefen_scale_by");
}

extern "C" int gefen_scale_from_f32(const float* a, void* a_out, int64_t a_numel, const float* b, void* b_out,
                                    int64_t b_numel, int dtype, const float* factor, gefen_stream_t stream) {
    const char* what = "gefen_scale_from_f32";
    if (!valid_dtype(dtype)) return fail_inval("%s: unknown dtype %d", what, dtype);
    if (a_numel < 0 || b_numel < 0 || (a_numel && (!a || !a_out)) || (b_numel && (!b || !b_out)) || !factor)
        return fail_inval("%s: null pointer or negative size", what);
    const int size = dtype_size(dtype);
    if (!aligned(a, 4) || !aligned(b, 4) || !aligned(a_out, size) || !aligned(b_out, size))
        return fail_inval("%s: not aligned to its elements", what);
    // few elements are spread over the chip: 101e3 in 7 chunks took 6.2 us, in 50 3.2
    const int chunk = a_numel + b_numel <= (int64_t)kGrid * kSmallChunk ? kSmallChunk : kChunk;
    const int64_t chunks = (a_numel + chunk - 1) / chunk + (b_numel + chunk - 1) / chunk;
    if (!chunks) return GEFEN_OK;
    const dim3 grid((unsigned)(chunks < kGrid ? chunks : kGrid)), wg(kThreads);
    auto launch = [&](auto type) {
        using T = decltype(type);
        hipLaunchKernelGGL(k_scale_from<T>, grid, wg, 0, stream, a, static_cast<T*>(a_out), a_numel, b,
                           static_cast<T*>(b_out), b_numel, factor, chunk);
    };
    if (dtype == GEFEN_F32) launch(0.0f);
    else if (dtype == GEFEN_BF16) launch(bf16_t{});
    else launch(f16_t{});
    return launch_status(what);
}
