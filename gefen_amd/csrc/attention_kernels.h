// Softmax attention and its gradients: the kernels and their launches (attention.hip has the
// entry points, attention_inst_*.hip the instances of each dtype).
//
//   S_ij = scale q_i . k_j,  L_i = log sum_j exp S_ij,  P_ij = exp(S_ij - L_i),  O_i = sum_j P_ij v_j
//   D_i = dO_i . O_i,  dS_ij = P_ij (dO_i . v_j - D_i)
//   dV_j = sum_i P_ij dO_i,  dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i
//
// Neither S nor P is stored: the forward pass keeps a running maximum and sum per row, and
// the backward pass forms P again from L.  It takes two kernels, one that owns queries (dQ,
// and D on its way) and one that owns keys (dK, dV, in workgroups of their own): S and dO v are
// formed again, eight products in place of five, and in return every sum has one owner and one
// order, with no atomics.
//
// The heads that share a key head are rows of one problem: row u = query u / G of head
// u % G of the group (G = heads / kv_heads), so a tile of keys and values is loaded once for
// all of them, and a single new token still gives G rows.
//
// P and dS are rounded to the operands' 16 bits on their way into the second products, whose matrix
// instructions take no more, and D is formed of the rounded output; float32 rounds neither.  So dQ
// and dK of bfloat16 are off by 2.6e-3 (float16 3.1e-4) where their own rounding is 1.7e-3 (2.1e-4);
// 2.4e-3 of it are the rounding of dS and of the result.
//
// What bounds it: with many rows the matrix cores, and beside them the vector unit: a 32 x 32
// block of S takes a wave some 480 cycles of exponentials, maxima and conversions, and its two
// products of the forward pass 256 (heads of 64) or 512.  8192 causal tokens, 32 / 8 heads of
// 128, bf16: forward 547 us, dQ 725, dK and dV 1320, which is 1.00, 1.14 and 1.04 PFLOP/s on the
// 2, 3 and 5 products that they form (a large library product reaches 1.24 on that card; matrix
// cores busy 49%, 59% and 58%, no bank conflicts, 1.95 to 2.1 GHz; 600, 800 and 1440 us on one whose
// product reaches 1.18).  8 x 1024 tokens, 12 heads of 64, float32: 142, 219 and 310 us, matrix cores
// busy 74%, 66% and 78%.  With one row a sequence, HBM: one query in each of 16 sequences of up to
// 8192 keys, 392 MB of 8 heads of 128, takes 90 us with the join.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attention_tiles.h"
#include "capi_internal.h"
#include "common.h"

namespace gefen {
namespace attn {

constexpr int kThreads = 256;
constexpr int kCols = 128;   // rows u (or keys) that a workgroup owns, 32 a wave
constexpr int BN = 64;       // rows of a tile
constexpr int kRangeParts = 16;

// A tensor [batch, rows, heads, width] with strides in elements.
struct View {
    void* p;
    int64_t batch, row, head;
};

struct Params {
    View q, k, v, o, go, gq, gk, gv;
    float* lse;    // [batch, heads, queries], log2 of the sum of exp2(c S): 0 for a row without keys
    float* delta;  // [batch, heads, queries]
    float* range;  // half precision: [2][batch * kv_heads][kRangeParts] largest norms of rows of v and of go
    const void* key_lengths;
    const void* offsets;
    int32_t lengths64, offsets64, sequences;
    int32_t batch, queries, keys, kv_heads, group, width, causal;
    int32_t rows;       // U = queries * group
    uint32_t div_mul;   // u / group = u * div_mul >> div_shift for u < 2^31
    int32_t div_shift;
    float c, scale;     // c = scale * log2(e)
    // A workgroup's tiles are split into `parts`; with more than one, part k leaves its sums in
    // float32 at partial + k * partial_stride (dV: behind the parts of dK), laid out as the
    // result, and its lse (forward) at partial_lse + k * stats.
    int32_t parts;
    float *partial, *partial_lse;
    int64_t partial_stride, stats;
};

__device__ __forceinline__ int div_group(const Params& a, int u) {
    return (int)(((uint64_t)(uint32_t)u * a.div_mul) >> a.div_shift);
}
__device__ __forceinline__ int clamped(const void* p, int is64, int k, int most) {
    const int64_t v = is64 ? static_cast<const int64_t*>(p)[k] : (int64_t)static_cast<const int32_t*>(p)[k];
    return (int)max((int64_t)0, min(v, (int64_t)most));
}

struct Interval {
    int lo, hi;
};
// The packed sequence that token i belongs to; empty if none.
__device__ __forceinline__ Interval sequence_of(const Params& a, int i) {
    int lo = -1, hi = a.sequences;  // offsets[lo] <= i (or lo = -1), and offsets past hi are not
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (clamped(a.offsets, a.offsets64, mid, a.queries) <= i) lo = mid;
        else hi = mid - 1;
    }
    if (lo < 0 || lo >= a.sequences) return {0, 0};
    const Interval s = {clamped(a.offsets, a.offsets64, lo, a.queries), clamped(a.offsets, a.offsets64, lo + 1, a.queries)};
    return s.lo <= i && i < s.hi ? s : Interval{0, 0};
}
// The keys that query i of sequence b sees.
__device__ __forceinline__ Interval keys_of(const Params& a, int b, int i) {
    Interval r = {0, a.keys};
    if (a.offsets) r = sequence_of(a, i);
    if (a.key_lengths) r.hi = min(r.hi, clamped(a.key_lengths, a.lengths64, b, a.keys));
    if (a.causal) r.hi = min(r.hi, i + a.keys - a.queries + 1);
    return r.hi > r.lo ? r : Interval{0, 0};
}
// The queries that see key j.
__device__ __forceinline__ Interval queries_of(const Params& a, int b, int j) {
    Interval r = {0, a.queries};
    if (a.offsets) r = sequence_of(a, j);
    if (a.key_lengths && j >= clamped(a.key_lengths, a.lengths64, b, a.keys)) return {0, 0};
    if (a.causal) r.lo = max(r.lo, j - (a.keys - a.queries));
    return r.hi > r.lo ? r : Interval{0, 0};
}

// What a wave's columns see of the other side: nothing outside [lo, hi), everything inside
// [full_lo, full_hi).
struct Span {
    int lo, hi, full_lo, full_hi;
    __device__ __forceinline__ void of(Interval r) {
        const bool any = r.hi > r.lo;
        lo = wave_min(any ? r.lo : 0x7fffffff);
        hi = wave_max(r.hi);
        full_lo = wave_max(r.lo);
        full_hi = wave_min(r.hi);
    }
    // of the tile from r0 on
    __device__ __forceinline__ bool none(int r0) const { return r0 >= hi || r0 + BN <= lo; }
    __device__ __forceinline__ bool full(int r0) const { return full_lo <= r0 && r0 + BN <= full_hi; }
};
// The span of the workgroup's waves (lo, hi only).
__device__ __forceinline__ Interval block_span(const Span& s) {
    __shared__ int part[2][kThreads / 64];
    if ((threadIdx.x & 63) == 0) {
        part[0][threadIdx.x >> 6] = s.lo;
        part[1][threadIdx.x >> 6] = s.hi;
    }
    __syncthreads();
    Interval r = {part[0][0], part[1][0]};
    for (int w = 1; w < kThreads / 64; ++w) {
        r.lo = min(r.lo, part[0][w]);
        r.hi = max(r.hi, part[1][w]);
    }
    return {uniform(r.lo), uniform(r.hi)};
}

// Place of row u in lse and delta.
__device__ __forceinline__ int64_t stat_at(const Params& a, int bh, int u) {
    const int i = div_group(a, u);
    return ((int64_t)bh * a.group + u - i * a.group) * a.queries + i;
}

// Rows of a view: of keys, or (GROUPED) rows u of queries.
template <typename T, bool GROUPED>
struct Rows {
    const T* base;
    int64_t row, head;
    int count;
    __device__ __forceinline__ Rows(const Params& a, const View& v, int b, int hk)
        : base(static_cast<const T*>(v.p) + b * v.batch + (int64_t)hk * (GROUPED ? a.group : 1) * v.head),
          row(v.row),
          head(v.head),
          count(GROUPED ? a.rows : a.keys) {}
    __device__ __forceinline__ const T* at(const Params& a, int u) const {
        if constexpr (GROUPED) {
            const int i = div_group(a, u);
            return base + i * row + (u - i * a.group) * head;
        } else {
            return base + u * row;
        }
    }
};

// Fills two tiles, one behind the other, from rows r0 .. of two operands.  ASYNC: rows are
// 16-byte aligned and a width of whole chunks (what lies behind the width is cleared once);
// issue() starts LOADS loads of a wave, for which the caller waits, each lane at an offset of
// its own that stays the same from tile to tile.  What lies behind the last row is left as it
// is: no step takes a row that it does not see (zeros there cost heads of 128 8%).  Otherwise
// (ASYNC false) issue() takes the rows into registers, the last one again behind it, and land()
// writes them.
template <typename T, int ROWS, int DP, bool ASYNC, int THREADS>
struct Filler {
    using TileT = Tile<T, ROWS, DP>;
    static constexpr int CPR = TileT::CPR, CHUNKS = ROWS * CPR, EPC = Elem<T>::EPC, LOADS = 2 * CHUNKS / THREADS;
    static_assert(LOADS * THREADS == 2 * CHUNKS && CHUNKS % 64 == 0, "whole loads, whole waves a tile");
    static constexpr uint32_t kBehind = 0xffffffffu;  // the offset of a chunk behind the width
    const int64_t row_x, row_y;                       // elements (ASYNC: ROWS of them are less than 2^30 bytes)
    const int width, count;
    const uint32_t lds;
    uint32_t off[ASYNC ? LOADS : 1];
    u32x4 r[ASYNC ? 1 : LOADS];

    // base: of the first tile, in LDS
    __device__ __forceinline__ Filler(const View& x, const View& y, int width, int count, typename TileT::lds_t* base)
        : row_x(x.row),
          row_y(y.row),
          width(width),
          count(count),
          lds(uniform((int)(uint32_t)(uintptr_t)(base + ((int)threadIdx.x >> 6) * 64 * EPC))) {
        if constexpr (ASYNC) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int c = chunk(i, threadIdx.x) * EPC;
                off[i] = c < width
                             ? (uint32_t)((row(i, threadIdx.x) * (int)(second(i) ? row_y : row_x) + c) * (int)sizeof(T))
                             : kBehind;
            }
        }
    }
    // load i of thread t
    __device__ __forceinline__ static int id(int i, int t) { return t + THREADS * i; }
    // whether it belongs to y (the same for a wave)
    __device__ __forceinline__ static bool second(int i) {
        if (THREADS * (i + 1) <= CHUNKS) return false;
        if (THREADS * i >= CHUNKS) return true;
        return uniform(id(i, threadIdx.x)) >= CHUNKS;
    }
    __device__ __forceinline__ static int row(int i, int t) { return (unsigned)id(i, t) % CHUNKS / CPR; }
    __device__ __forceinline__ static int chunk(int i, int t) {
        return ((unsigned)id(i, t) % CPR) ^ (ASYNC ? chunk_xor(row(i, t), CPR) : 0);
    }
    // x, y: row 0 of the operands
    __device__ __forceinline__ void issue(const T* x, const T* y, int r0, uint32_t tile_bytes) {
        int t = threadIdx.x;
        if constexpr (ASYNC) {
            x += r0 * row_x;
            y += r0 * row_y;
            const uint32_t to = lds + tile_bytes;
            const bool tail = r0 + ROWS > count;
            asm volatile("" : "+v"(t));  // rows are not kept in registers for the last tile's sake
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                bool have = off[i] != kBehind;
                if (tail) have = have && r0 + row(i, t) < count;
                if (have) load_to_lds(second(i) ? y : x, off[i], to + i * THREADS * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int n = width - chunk(i, t) * EPC;
                const T* at = (second(i) ? y : x) + min(r0 + row(i, t), count - 1) * (second(i) ? row_y : row_x);
                r[i] = n > 0 ? load_chunk(at + chunk(i, t) * EPC, n) : u32x4{0u, 0u, 0u, 0u};
            }
        }
    }
    // t: the first tile
    __device__ __forceinline__ void land(const TileT& t) const {
        if constexpr (!ASYNC) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                TileT{t.p + (second(i) ? TileT::ELEMS : 0)}.put(row(i, threadIdx.x), chunk(i, threadIdx.x), r[i]);
        }
    }
};
// The tiles of two operands, twice: one pair is filled while the other is worked on.
template <typename T, int DP, bool ASYNC>
struct Pipe {
    using TileT = Tile<T, BN, DP>;
    static constexpr int BYTES = 4 * TileT::BYTES;
    typename TileT::lds_t* base;
    Filler<T, BN, DP, ASYNC, kThreads> fill;
    const T *x, *y;  // row 0 of the operands

    __device__ __forceinline__ Pipe(const View& vx, const View& vy, const T* x, const T* y, int width, int count, char* smem)
        : base((typename TileT::lds_t*)smem), fill(vx, vy, width, count, base), x(x), y(y) {
        if (ASYNC && width < DP) {  // zeros behind the rows' width, which the loads leave as they are
            typedef __attribute__((address_space(3))) u32x4 lds_chunk;
            lds_chunk* p = (lds_chunk*)base;
            for (int i = threadIdx.x; i < BYTES / 16; i += kThreads) p[i] = u32x4{0u, 0u, 0u, 0u};
        }
        __syncthreads();
    }
    __device__ __forceinline__ TileT tile(int buffer, int which) const {
        return TileT{base + (2 * buffer + which) * TileT::ELEMS};
    }
    // step(r0, first tile, second tile, buffer) for this part of the tiles of [all.lo, all.hi)
    // of `heads` heads, head_x and head_y elements apart; more(head, r0, buffer) loads what else
    // the step needs, and land(buffer) writes what of it is in registers.  The heads of a tile
    // follow each other, and the tiles (DOWN: from the last to the first): causal workgroups see
    // a common beginning of that order, and those that run side by side read the same rows at
    // about the same time, from their XCD's L2.
    template <bool DOWN, typename More, typename Land, typename Step>
    __device__ __forceinline__ void run(Interval all, int heads, int64_t head_x, int64_t head_y, int part, int parts,
                                        More more, Land land, Step step) {
        if (all.hi <= all.lo) return;
        const int start = all.lo / BN * BN, count = (all.hi - start + BN - 1) / BN;
        // parts share the heads out, and where there are more of them than heads the tiles too
        const int by_head = min(parts, heads), by_tile = parts / by_head;
        const int head0 = part % by_head * heads / by_head, heads_here = (part % by_head + 1) * heads / by_head - head0;
        const int tile0 = part / by_head * count / by_tile, tiles = (part / by_head + 1) * count / by_tile - tile0;
        int left = part < by_head * by_tile ? tiles * heads_here : 0;
        if (left <= 0) return;
        int head = head0, r0 = start + (DOWN ? count - 1 - tile0 : tile0) * BN;
        x += head * head_x;
        y += head * head_y;
        fill.issue(x, y, r0, 0);
        more(head, r0, 0);
        fill.land(tile(0, 0));
        land(0);
        auto one = [&](auto which) __attribute__((always_inline)) {
            constexpr int buffer = decltype(which)::value;
            // this buffer has landed, and every wave is done with the other one
            wait_loads_and_sync();
            const int now = r0;
            x += head_x;
            y += head_y;
            if (++head == head0 + heads_here) {
                head = head0;
                x -= heads_here * head_x;
                y -= heads_here * head_y;
                r0 += DOWN ? -BN : BN;
            }
            const bool next = --left > 0;
            if (next) {
                fill.issue(x, y, r0, (1 - buffer) * 2 * TileT::BYTES);
                more(head, r0, 1 - buffer);
            }
            step(now, tile(buffer, 0), tile(buffer, 1), buffer);
            if (next) {
                fill.land(tile(1 - buffer, 0));
                land(1 - buffer);
            }
            return next;
        };
        while (one(std::integral_constant<int, 0>{}) && one(std::integral_constant<int, 1>{})) {
        }
    }
};

// A lane's row as the right side of the rows products.
template <typename T, int DP>
struct Column {
    static constexpr int EPC = Elem<T>::EPC, STEPS = DP / (2 * EPC);
    u32x4 c[STEPS];
    __device__ __forceinline__ void load(const T* row, int width, int lane) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int at = (2 * s + (lane >> 5)) * EPC;
            c[s] = at < width ? load_chunk(row + at, width - at) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    // The row has arrived: without a use before the tiles' loop the compiler waits for it within,
    // each time, and so for the next tile's loads.
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) asm volatile("" : "+v"(c[s]));
    }
    // sum of this half's products with another row, float32
    __device__ __forceinline__ float dot(const Column& o) const {
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < EPC; ++i) sum = __builtin_fmaf(elem(c[s], i), elem(o.c[s], i), sum);
        return sum;
    }
    __device__ __forceinline__ static float elem(u32x4 v, int i) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
        else return Elem<T>::value((uint16_t)(v[i / 2] >> (16 * (i & 1))));
    }
};

template <typename T, int ROWS, int DP>
__device__ __forceinline__ f32x16 rows_product(const Tile<T, ROWS, DP>& t, int r0, const Column<T, DP>& x, int lane,
                                               f32x16 acc = {}) {
#pragma unroll
    for (int c = 0; c < Column<T, DP>::STEPS; ++c) acc = mma_rows<T>(t.row_chunk(r0, c, lane), x.c[c], acc);
    return acc;
}
// The row of a tile that register i of a rows product holds.
__device__ __forceinline__ int row_of(int r0, int i, int lane) { return r0 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4; }
__device__ __forceinline__ bool within(int r, Interval s) { return (uint32_t)(r - s.lo) < (uint32_t)(s.hi - s.lo); }

// acc[d, n] times f into a row of width elements.
template <typename T, int DT>
__device__ __forceinline__ void store_column(T* row, const f32x16 (&acc)[DT], float f, int width, int lane) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = row_of(32 * dt, i, lane);
            if (d < width)
                store4(row + d, acc[dt][i] * f, acc[dt][i + 1] * f, acc[dt][i + 2] * f, acc[dt][i + 3] * f, width - d);
        }
}

// LDS reads that are on their way before the matrix instruction of the first one, where stream()
// orders them: the forward pass (11 packed sequences of 16384 tokens, heads of 64: 515 us, and
// 535 as the compiler orders them) and dK and dV of wide heads (8192 tokens, heads of 128: 1477
// and 1590 us; heads of 64: 1126 and 1026).  dQ took 768 and 770, 608 and 564 us.
constexpr int kAhead = 4;

// How the forward pass takes a tile: all of it; what a wave's columns see of it (scores of -inf
// for the rest, so c must not be zero); or that, with what is not finite kept from the columns
// that do not see it (0 x inf is NaN), where the tile holds such elements at all, in rows that
// the wave sees or in others.  Looking first cost less than keeping them out always: packed
// sequences 530 us and 494.  Wider heads, whose registers it spills, gained 1%, dQ as much
// (570 and 564), and dK and dV, whose third wave on a SIMD has no registers to spare, lost (1013
// and 1164): they know the first and the last only.
enum : int { kFull, kMasked, kChecked };
template <int KIND>
using Kind = std::integral_constant<int, KIND>;

// Half precision keeps 2^-14 .. 65504 at full precision, so what is rounded to it is brought
// there by powers of two that are taken out again: probabilities by 2^14 in the backward pass
// and 2^6 in the forward one (whose running maximum may lag by 2^8), and dO v - D by the
// bound that the rows' norms give.
template <typename T>
constexpr bool kHalf = std::is_same<T, f16_t>::value;
constexpr float kLag = 8.0f;
constexpr float kAllInfinite = -3.4028235e38f;  // lse of a part whose keys all score -inf
template <typename T>
constexpr float kForwardShift = kHalf<T> ? 6.0f : 0.0f;
template <typename T>
constexpr float kBackwardShift = kHalf<T> ? 14.0f : 0.0f;

// Waves on a SIMD of the forward pass.  The third one of heads of up to 64 hides more than the
// registers that it spills cost (43 words; packed sequences, heads of 64: 511 us with two, 444 with
// three; 8192 causal tokens, 32 heads of 32: 265 and 227), if there are workgroups for it: up to
// kTwoEach it only spills (one query of 16 sequences, 32 / 8 heads of 64: 52 us with two, 58 with
// three; 777 queries over 1003 keys: 21.8 and 23.8).  Tiles that come through registers leave fewer:
// none is spilled up to 32 (heads of 17: 374 us with two, 288 with three), 89 words above (12 heads
// of 63 of 8 x 1024 tokens 107 us with two, 142 with three; 11 packed sequences, 32 heads of 64 off
// alignment, 260 and 403; only 8192 tokens of 32 heads of 63 lost with two, 1146 and 978).
template <typename T>
constexpr int forward_waves(int dp, bool async) {
    return sizeof(T) == 2 ? (dp <= (async ? 64 : 32) ? 3 : 2) : dp <= 64 ? 2 : 1;
}
constexpr int kTwoEach = 512;  // workgroups of four waves, two waves a SIMD

template <typename T, int DP, bool ASYNC, int WAVES>
__global__ void __launch_bounds__(kThreads, WAVES) k_forward(Params a) {
    using TileT = Tile<T, BN, DP>;
    using PipeT = Pipe<T, DP, ASYNC>;
    constexpr int DT = DP / 32;
    constexpr bool STREAM = sizeof(T) == 2;
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // PipeT::BYTES
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the rows that see most keys first
    const int heads = a.batch * a.kv_heads, tiles = (a.rows + kCols - 1) / kCols;
    const int bh = blockIdx.x % heads, part = blockIdx.x / heads % a.parts, tile = tiles - 1 - blockIdx.x / heads / a.parts;
    const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
    const int u = tile * kCols + wave * 32 + (lane & 31), uc = min(u, a.rows - 1);
    const Interval seen = keys_of(a, b, div_group(a, uc));
    Span span;
    span.of(seen);
    const Interval all = block_span(span);

    const Rows<T, true> queries(a, a.q, b, hk);
    const Rows<T, false> keys(a, a.k, b, hk), values(a, a.v, b, hk);
    PipeT pipe(a.k, a.v, keys.base, values.base, a.width, a.keys, smem);
    Column<T, DP> q;
    q.load(queries.at(a, uc), a.width, lane);
    q.arrived();
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
    float top = -INFINITY, sum = 0.0f;

    auto tile_step = [&](auto kind, int k0, const TileT& kt, const TileT& vt) __attribute__((always_inline)) {
        constexpr bool PARTIAL = decltype(kind)::value != kFull, CHECK = decltype(kind)::value == kChecked;
        f32x16 s[2] = {};
        if constexpr (STREAM && !CHECK) {
            constexpr int STEPS = Column<T, DP>::STEPS;
            stream<2 * STEPS, kAhead>([&](int i) { return kt.row_chunk(32 * (i / STEPS), i % STEPS, lane); },
                                      [&](int i, u32x4 f) { s[i / STEPS] = mma_rows<T>(f, q.c[i % STEPS], s[i / STEPS]); });
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = rows_product(kt, 32 * t, q, lane);
        }
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (PARTIAL && !within(row_of(k0 + 32 * t, i, lane), seen)) s[t][i] = -INFINITY;
                most = fmaxf(most, s[t][i]);
            }
        most = fmaxf(most, other_half(most)) * a.c;
        if (__any(most > top + kLag)) {
            const float next = fmaxf(top, most);
            const float f = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.0f : next));
            top = next;
            sum *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
        }
        const float shift = kForwardShift<T> - (top == -INFINITY ? 0.0f : top);
        const RowRange rows = {span.lo - k0, span.hi - k0};
        uint32_t bad = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.c, shift));
                if (CHECK && !within(row_of(k0 + 32 * t, i, lane), seen)) p = 0.0f;
                s[t][i] = p;
                sum += p;
            }
            if (STREAM && !CHECK) continue;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const PFrag<T> p = pack<T>(s[t], c);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = vt.template mma_columns<CHECK>(p, 32 * t + 16 * c, 32 * dt, lane, acc[dt], rows, &bad);
            }
        }
        if constexpr (STREAM && !CHECK) {
            PFrag<T> p[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = pack<T>(s[c / 2], c % 2);
            stream<4 * DT, kAhead>([&](int i) { return vt.column_chunk(16 * (i / DT), 32 * (i % DT), lane); },
                                   [&](int i, u32x4 f) { acc[i % DT] = mma_chunk<T>(f, p[i / DT], acc[i % DT]); });
        }
        if (CHECK && __any((bad & kBadBits<T>) != 0)) vt.template add_nonfinite<false>(acc, BN, seen.lo - k0, seen.hi - k0, lane);
    };

    auto step = [&](int k0, const TileT& kt, const TileT& vt, int) __attribute__((always_inline)) {
        if (span.none(k0)) return;
        if (span.full(k0)) return tile_step(Kind<kFull>{}, k0, kt, vt);
        if constexpr (sizeof(T) == 2 && DP <= (ASYNC ? 96 : 64))
            if (a.c >= 1.2e-38f && vt.all_finite(lane)) return tile_step(Kind<kMasked>{}, k0, kt, vt);
        tile_step(Kind<kChecked>{}, k0, kt, vt);
    };
    pipe.template run<false>(all, 1, 0, 0, part, a.parts, [](int, int, int) {}, [](int) {}, step);
    sum += other_half(sum);
    if (u >= a.rows) return;
    const bool empty = seen.hi <= seen.lo;
    const int i = div_group(a, u);
    const int64_t at = b * a.o.batch + i * a.o.row + (int64_t)(hk * a.group + u - i * a.group) * a.o.head;
    if (a.parts > 1) {
        // a part's own result; a part without keys, or whose scores are all -inf, weighs nothing
        store_column(a.partial + part * a.partial_stride + at, acc, sum == 0.0f ? 0.0f : 1.0f / sum, a.width, lane);
        if (lane < 32)
            a.partial_lse[part * a.stats + stat_at(a, bh, u)] =
                empty ? -INFINITY : sum == 0.0f ? kAllInfinite : top + __builtin_amdgcn_logf(sum) - kForwardShift<T>;
        return;
    }
    store_column(static_cast<T*>(a.o.p) + at, acc, empty ? 1.0f : 1.0f / sum, a.width, lane);
    if (a.lse && lane < 32)
        a.lse[stat_at(a, bh, u)] = empty ? 0.0f : top + __builtin_amdgcn_logf(sum) - kForwardShift<T>;
}

// The parts of a row of the output together: 32 lanes a row, four elements each.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_join_forward(Params a) {
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;  // [batch, query, head]
    const int heads = a.kv_heads * a.group;
    if (row >= (int64_t)a.batch * a.queries * heads) return;
    const int64_t bi = row / heads;
    const int h = (int)(row - bi * heads), b = (int)(bi / a.queries), i = (int)(bi - (int64_t)b * a.queries);
    const int64_t stat = ((int64_t)b * heads + h) * a.queries + i;
    float most = -INFINITY;
    for (int p = 0; p < a.parts; ++p) most = fmaxf(most, a.partial_lse[p * a.stats + stat]);
    const int d = (threadIdx.x & 31) * 4, have = a.width - d;
    float sum = 0.0f, out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = 0; p < a.parts; ++p) {
        const float lse = a.partial_lse[p * a.stats + stat];
        u32x4 x = {0u, 0u, 0u, 0u};
        if (have > 0) x = load_chunk(a.partial + p * a.partial_stride + row * a.width + d, have);
        if (lse == -INFINITY) continue;  // no keys
        const float w = __builtin_amdgcn_exp2f(lse - most);
        sum += w;
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = __builtin_fmaf(w, __uint_as_float(x[k]), out[k]);
    }
    const bool empty = sum == 0.0f;
    // keys, but none of a finite score
    const float f = empty ? 1.0f : most == kAllInfinite ? __uint_as_float(0x7fc00000u) : 1.0f / sum;
    if (have > 0) store4(static_cast<T*>(a.o.p) + row * a.width + d, out[0] * f, out[1] * f, out[2] * f, out[3] * f, have);
    if (a.lse && d == 0) a.lse[stat] = empty ? 0.0f : (most + __builtin_amdgcn_logf(sum)) + (f != f ? f : 0.0f);
}

// The sums of the parts, in their order: of dQ, or of dK and (blockIdx.y = 1) dV.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_join_sums(const float* partial, int parts, int64_t stride, int64_t numel,
                                                        T* first, T* second) {
    const int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
    if (e >= numel) return;
    const int have = (int)min((int64_t)4, numel - e);
    partial += blockIdx.y * parts * stride + e;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        const u32x4 x = load_chunk(partial + p * stride, have);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += __uint_as_float(x[k]);
    }
    store4((blockIdx.y ? second : first) + e, sum[0], sum[1], sum[2], sum[3], have);
}

// The power of two that brings values of up to `most` into [-1, 1].
__device__ __forceinline__ float into_one(float most) {
    if (!(most > 0.0f) || most > 3.0e38f) return 1.0f;
    int e;
    frexpf(most, &e);
    return ldexpf(1.0f, min(max(-e, -120), 120));
}
// The largest row norm of v (which = 0) or of go (1) in (batch, key head) bh.
__device__ __forceinline__ float largest_norm(const Params& a, int which, int bh) {
    const float* r = a.range + ((int64_t)which * a.batch * a.kv_heads + bh) * kRangeParts;
    float m = 0.0f;
    for (int k = 0; k < kRangeParts; ++k) m = fmaxf(m, r[k]);
    return m;
}

// Largest norms of the rows of v and of go that take part (what the others hold must not reach
// the scale either), for half precision; 16 lanes a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_range(Params a) {
    const int heads = a.batch * a.kv_heads, bh = blockIdx.x, part = blockIdx.y, which = blockIdx.z;
    const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
    const Rows<T, true> grads(a, a.go, b, hk);
    const Rows<T, false> values(a, a.v, b, hk);
    Interval in = {0, which ? a.queries : a.keys};
    if (a.offsets) {
        in = {clamped(a.offsets, a.offsets64, 0, a.queries), clamped(a.offsets, a.offsets64, a.sequences, a.queries)};
    } else {
        const int seen = a.key_lengths ? clamped(a.key_lengths, a.lengths64, b, a.keys) : a.keys;
        if (!which || seen == 0) in.hi = min(in.hi, seen);
        if (which && a.causal) in.lo = max(0, a.queries - a.keys);
    }
    const int lo = in.lo * (which ? a.group : 1), rows = in.hi * (which ? a.group : 1);
    const int c = (threadIdx.x & 15) * Elem<T>::EPC;
    float most = 0.0f;
    for (int r = lo + part * (kThreads / 16) + (threadIdx.x >> 4); r < rows; r += kRangeParts * (kThreads / 16)) {
        const T* row = which ? grads.at(a, r) : values.at(a, r);
        float sq = 0.0f;
        if (c < a.width) {
            const u32x4 x = load_chunk(row + c, a.width - c);
#pragma unroll
            for (int i = 0; i < Elem<T>::EPC; ++i) {
                const float e = Column<T, 128>::elem(x, i);
                sq = __builtin_fmaf(e, e, sq);
            }
        }
        for (int off = 8; off > 0; off >>= 1) sq += __shfl_xor(sq, off, 64);
        if (sq < INFINITY) most = fmaxf(most, sq);  // what is not finite reaches its results anyway
    }
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64));
    __shared__ float part_most[kThreads / 64];
    if ((threadIdx.x & 63) == 0) part_most[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; ++w) most = fmaxf(most, part_most[w]);
        a.range[((int64_t)which * heads + bh) * kRangeParts + part] = sqrtf(most);
    }
}

// dQ, and D for the other kernel.
template <typename T, int DP, bool ASYNC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) k_backward_queries(Params a) {
    using TileT = Tile<T, BN, DP>;
    using PipeT = Pipe<T, DP, ASYNC>;
    constexpr int DT = DP / 32;
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // PipeT::BYTES
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int heads = a.batch * a.kv_heads, tiles = (a.rows + kCols - 1) / kCols;
    const int bh = blockIdx.x % heads, part = blockIdx.x / heads % a.parts, tile = tiles - 1 - blockIdx.x / heads / a.parts;
    const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
    const int u = tile * kCols + wave * 32 + (lane & 31), uc = min(u, a.rows - 1);
    const Interval seen = keys_of(a, b, div_group(a, uc));
    Span span;
    span.of(seen);
    const Interval all = block_span(span);

    const Rows<T, false> keys(a, a.k, b, hk), values(a, a.v, b, hk);
    PipeT pipe(a.k, a.v, keys.base, values.base, a.width, a.keys, smem);
    Column<T, DP> q, go;
    go.load(Rows<T, true>(a, a.go, b, hk).at(a, uc), a.width, lane);
    q.load(Rows<T, true>(a, a.o, b, hk).at(a, uc), a.width, lane);
    float delta = go.dot(q);
    delta += other_half(delta);
    if (lane < 32 && u < a.rows && part == 0) a.delta[stat_at(a, bh, u)] = delta;
    q.load(Rows<T, true>(a, a.q, b, hk).at(a, uc), a.width, lane);
    q.arrived();
    const float shift = kBackwardShift<T> - a.lse[stat_at(a, bh, uc)];
    float unit = 1.0f;
    if constexpr (kHalf<T>) {
        float norm = go.dot(go);
        norm = sqrtf(norm + other_half(norm));
        unit = into_one(2.0f * norm * largest_norm(a, 0, bh));
    }
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};

    auto tile_step = [&](auto partial, int k0, const TileT& kt, const TileT& vt) __attribute__((always_inline)) {
        constexpr bool PARTIAL = decltype(partial)::value;
        const RowRange rows = {span.lo - k0, span.hi - k0};
        uint32_t bad = 0;
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
            f32x16 s = {}, dp = {};
            if constexpr (DP <= 64) {  // wide heads took 7% longer this way
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = -delta;
            }
            s = rows_product(kt, 32 * t, q, lane);
            dp = rows_product(vt, 32 * t, go, lane, dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, shift));
                const float d = DP <= 64 ? dp[i] : dp[i] - delta;
                float ds = p * (kHalf<T> ? d * unit : d);
                if (PARTIAL && !within(row_of(k0 + 32 * t, i, lane), seen)) ds = 0.0f;
                s[i] = ds;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const PFrag<T> ds = pack<T>(s, c);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = kt.template mma_columns<PARTIAL>(ds, 32 * t + 16 * c, 32 * dt, lane, acc[dt], rows, &bad);
            }
        }
        if (PARTIAL && __any((bad & kBadBits<T>) != 0)) kt.template add_nonfinite<true>(acc, BN, seen.lo - k0, seen.hi - k0, lane);
    };

    auto step = [&](int k0, const TileT& kt, const TileT& vt, int) __attribute__((always_inline)) {
        if (span.none(k0)) return;
        if (span.full(k0)) tile_step(std::false_type{}, k0, kt, vt);
        else tile_step(std::true_type{}, k0, kt, vt);
    };
    pipe.template run<false>(all, 1, 0, 0, part, a.parts, [](int, int, int) {}, [](int) {}, step);
    if (u >= a.rows) return;
    const int i = div_group(a, u);
    const int64_t at = b * a.gq.batch + i * a.gq.row + (int64_t)(hk * a.group + u - i * a.group) * a.gq.head;
    const float f = kHalf<T> ? a.scale * (1.0f / 16384.0f) / unit : a.scale;
    if (a.parts > 1) store_column(a.partial + part * a.partial_stride + at, acc, f, a.width, lane);
    else store_column(static_cast<T*>(a.gq.p) + at, acc, f, a.width, lane);
}

// dK, or (VALUES) dV.  Together they would need 4 products instead of 5, but their accumulators
// beside a lane's key and value leave no room for a second wave on a SIMD: one kernel for both took
// 2022 us at 8192 causal tokens of 32 / 8 heads of 128 (bf16), where this one takes 1320 to 1440.  As
// pairs of waves that share 32 keys, one of which hands P over through LDS (rounded, so that dK's dS
// had a rounding more), both took 1369 us when this one took 1636.  Since then this one takes the rows
// from the last one on (1423) and orders its LDS reads (1530 to 1394 on another card); pairs without
// that order took 1541 beside the 1530, and 296 us beside 330 for float32 heads of 64.  With both they
// have not been measured.
template <typename T, int DP, bool ASYNC, bool VALUES>
__device__ __forceinline__ void backward_keys(const Params& a, int bh, int tile, int part, char* smem) {
    using TileT = Tile<T, BN, DP>;
    constexpr int DT = DP / 32;
    constexpr bool STREAM = sizeof(T) == 2 && DP > 64;
    // L / c and D of each buffer's rows, which the products subtract as terms of their own; float32:
    // -L and -D as numbers.  dP starts from -D.  S starts from zero and meets L as S c - L: terms that
    // are added to -L / c lose what is below its spacing, up to 300 x 2^-24 of P at L = log 64 (a
    // hundredth of what bfloat16 is rounded by, a fourteenth of float16), and made float32's dK and dV
    // 1.6 to 2.5 times as inexact as dQ.  It costs 1% (heads of 64: 336 and 342 us) and gained 4% at 128.
    constexpr bool TERMS = sizeof(T) == 2;
    __shared__ u32x4 row_terms[TERMS ? 2 : 1][2][TERMS ? BN : 1];
    __shared__ __attribute__((aligned(16))) float row_numbers[TERMS ? 1 : 2][2][TERMS ? 1 : BN];
    constexpr int UNROLL = VALUES || DP <= 64 ? 2 : 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = bh / a.kv_heads, hk = bh % a.kv_heads;
    const int j = tile * kCols + wave * 32 + (lane & 31), jc = min(j, a.keys - 1);
    const Interval seen = queries_of(a, b, jc);
    Span span;
    span.of(seen);
    const Interval all = block_span(span);

    const Rows<T, true> queries(a, a.q, b, hk), grads(a, a.go, b, hk);
    Pipe<T, DP, ASYNC> pipe(a.q, a.go, queries.base, grads.base, a.width, a.queries, smem);
    Column<T, DP> k, v;
    k.load(Rows<T, false>(a, a.k, b, hk).at(a, jc), a.width, lane);
    if (!VALUES) v.load(Rows<T, false>(a, a.v, b, hk).at(a, jc), a.width, lane);
    k.arrived();
    if (!VALUES) v.arrived();
    // 16 bits: S - L / c is formed, and c applied after; with a c that is as good as zero, -L with a key of zeros
    float c = a.c, over = 1.0f / a.c;
    if (TERMS && !(a.c > 5.4e-20f)) {
        c = over = 1.0f;
#pragma unroll
        for (int i = 0; i < Column<T, DP>::STEPS; ++i) k.c[i] = u32x4{0u, 0u, 0u, 0u};
    }
    float unit = 1.0f;
    if constexpr (kHalf<T> && !VALUES) unit = into_one(2.0f * largest_norm(a, 0, bh) * largest_norm(a, 1, bh));
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};

    auto tile_step = [&](auto partial, int i0, const TileT& qt, const TileT& gt, int buffer) __attribute__((always_inline)) {
        constexpr bool PARTIAL = decltype(partial)::value;
        const TileT& into = VALUES ? gt : qt;
        const RowRange rows = {span.lo - i0, span.hi - i0};
        uint32_t bad = 0;
#pragma unroll UNROLL
        for (int t = 0; t < BN / 32; ++t) {
            f32x16 s = {}, dp = {};
            auto numbers = [&](int which) __attribute__((always_inline)) {  // -L or -D of this lane's 16 rows
                f32x16 x = {};
                if constexpr (!TERMS) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 v = *(const f32x4*)&row_numbers[buffer][which][row_of(32 * t, i, lane)];
                        for (int k = 0; k < 4; ++k) x[i + k] = v[k];
                    }
                }
                return x;
            };
            if constexpr (TERMS) {
                s = RowTerm{(RowTerm::lds_chunk*)row_terms[buffer][0]}.subtract(32 * t, lane, s);
                if (!VALUES) dp = RowTerm{(RowTerm::lds_chunk*)row_terms[buffer][1]}.subtract(32 * t, lane, dp);
            } else {
                if (!VALUES) dp = numbers(1);
            }
            if constexpr (STREAM && !PARTIAL) {
                constexpr int STEPS = Column<T, DP>::STEPS;
                stream<STEPS * (VALUES ? 1 : 2), kAhead>(
                    [&](int i) { return (i < STEPS ? qt : gt).row_chunk(32 * t, i % STEPS, lane); },
                    [&](int i, u32x4 f) {
                        if (i < STEPS) s = mma_rows<T>(f, k.c[i], s);
                        else dp = mma_rows<T>(f, v.c[i - STEPS], dp);
                    });
            } else {
                s = rows_product(qt, 32 * t, k, lane, s);
                if (!VALUES) dp = rows_product(gt, 32 * t, v, lane, dp);
            }
            const f32x16 minus_l = numbers(0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = row_of(32 * t, i, lane);
                float p;
                if constexpr (!TERMS) p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, minus_l[i]));
                else p = __builtin_amdgcn_exp2f(kHalf<T> ? __builtin_fmaf(s[i], c, kBackwardShift<T>) : s[i] * c);
                if (!VALUES) p *= kHalf<T> ? dp[i] * unit : dp[i];
                s[i] = PARTIAL && !within(i0 + r, seen) ? 0.0f : p;
            }
            if constexpr (STREAM && !PARTIAL) {
                const PFrag<T> p[2] = {pack<T>(s, 0), pack<T>(s, 1)};
                stream<2 * DT, kAhead>([&](int i) { return into.column_chunk(32 * t + 16 * (i / DT), 32 * (i % DT), lane); },
                                       [&](int i, u32x4 f) { acc[i % DT] = mma_chunk<T>(f, p[i / DT], acc[i % DT]); });
                continue;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const PFrag<T> p = pack<T>(s, c);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = into.template mma_columns<PARTIAL>(p, 32 * t + 16 * c, 32 * dt, lane, acc[dt], rows, &bad);
            }
        }
        if (PARTIAL && __any((bad & kBadBits<T>) != 0))
            into.template add_nonfinite<!VALUES>(acc, BN, seen.lo - i0, seen.hi - i0, lane);
    };
    auto step = [&](int i0, const TileT& qt, const TileT& gt, int buffer) __attribute__((always_inline)) {
        if (span.none(i0)) return;
        if (span.full(i0)) tile_step(std::false_type{}, i0, qt, gt, buffer);
        else tile_step(std::true_type{}, i0, qt, gt, buffer);
    };
    // a wave's 64 lanes take the rows' L along, another one's D
    const float* const stats = (wave & 1 ? a.delta : a.lse) + (int64_t)bh * a.group * a.queries + lane;
    const bool takes = wave < (VALUES ? 1 : 2);
    float taken = 0.0f;
    auto more = [&](int head, int i0, int) __attribute__((always_inline)) {
        if (takes && i0 + lane < a.queries) taken = stats[(int64_t)head * a.queries + i0];
    };
    auto land = [&](int buffer) __attribute__((always_inline)) {
        if (!takes) return;
        if constexpr (TERMS) row_terms[buffer][wave][lane] = RowTerm::split(wave ? taken : taken * over);
        else row_numbers[buffer][wave][lane] = -taken;
    };
    pipe.template run<true>(all, a.group, a.q.head, a.go.head, part, a.parts, more, land, step);
    if (j >= a.keys) return;
    const View& out = VALUES ? a.gv : a.gk;
    const int64_t at = b * out.batch + j * out.row + hk * out.head;
    const float down = kHalf<T> ? 1.0f / 16384.0f : 1.0f, f = VALUES ? down : a.scale * down / unit;
    if (a.parts > 1)
        store_column(a.partial + (part + (VALUES ? a.parts : 0)) * a.partial_stride + at, acc, f, a.width, lane);
    else store_column(static_cast<T*>(out.p) + at, acc, f, a.width, lane);
}
// The workgroups of dK (the longer ones), then those of dV; of each the keys first that most
// rows see.
template <typename T, int DP, bool ASYNC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 || DP <= 64 ? 2 : 1) k_backward_keys(Params a) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // Pipe::BYTES
    const int heads = a.batch * a.kv_heads, block = blockIdx.x;
    const int bh = block % heads, part = block / heads % a.parts, tile = block / heads / a.parts;
    if (blockIdx.y) backward_keys<T, DP, ASYNC, true>(a, bh, tile, part, smem);
    else backward_keys<T, DP, ASYNC, false>(a, bh, tile, part, smem);
}

// ------------------------------------------------------------------ launches

enum Pass { kForwardPass, kQueriesPass, kKeysPass };

template <typename T, int DP, bool ASYNC>
int launch(Pass pass, const Params& a, hipStream_t st) {
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    const int64_t tiles = ((pass == kKeysPass ? a.keys : a.rows) + kCols - 1) / kCols;
    const uint32_t grid = (uint32_t)(heads * tiles * a.parts);
    constexpr int lds = Pipe<T, DP, ASYNC>::BYTES;
    constexpr int waves = forward_waves<T>(DP, ASYNC), few = DP > 32 ? std::min(waves, 2) : waves;
    constexpr auto forward = k_forward<T, DP, ASYNC, waves>, forward_few = k_forward<T, DP, ASYNC, few>;
    if (pass == kForwardPass) (grid <= kTwoEach ? forward_few : forward)<<<grid, kThreads, lds, st>>>(a);
    else if (pass == kQueriesPass) k_backward_queries<T, DP, ASYNC><<<grid, kThreads, lds, st>>>(a);
    else k_backward_keys<T, DP, ASYNC><<<dim3(grid, 2), kThreads, lds, st>>>(a);
    if (int rc = launch_status("attention")) return rc;
    if (a.parts == 1) return GEFEN_OK;
    if (pass == kForwardPass) {
        const int64_t rows = (int64_t)a.batch * a.queries * a.kv_heads * a.group;
        k_join_forward<T><<<(uint32_t)((rows + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(a);
    } else {
        const bool keys = pass == kKeysPass;
        const View& out = keys ? a.gk : a.gq;
        const int64_t numel = out.batch * a.batch;
        k_join_sums<T><<<dim3((uint32_t)((numel + 4 * kThreads - 1) / (4 * kThreads)), keys ? 2 : 1), kThreads, 0, st>>>(
            a.partial, a.parts, a.partial_stride, numel, static_cast<T*>(out.p), static_cast<T*>(a.gv.p));
    }
    return launch_status("attention");
}
// Whether a tensor's rows are whole 16-byte chunks at distances that a tile's offsets hold.
inline bool chunked(const Params& a, const View& v, int rows, int heads, int size) {
    auto apart = [&](int64_t stride, int count) { return count <= 1 || stride * size % 16 == 0; };
    return aligned(v.p, 16) && a.width * size % 16 == 0 && apart(v.batch, a.batch) && apart(v.row, rows) &&
           apart(v.head, heads) && (rows <= 1 || (v.row >= 0 && v.row < (int64_t)1 << 22));
}
template <typename T, int DP>
int launch_filler(Pass pass, const Params& a, hipStream_t st) {
    const bool keys = pass == kKeysPass;
    const int rows = keys ? a.queries : a.keys, heads = keys ? a.kv_heads * a.group : a.kv_heads;
    const bool async = chunked(a, keys ? a.q : a.k, rows, heads, sizeof(T)) &&
                       chunked(a, keys ? a.go : a.v, rows, heads, sizeof(T));
    return async ? launch<T, DP, true>(pass, a, st) : launch<T, DP, false>(pass, a, st);
}
template <typename T>
int launch_width(Pass pass, const Params& a, hipStream_t st) {
    if (a.width <= 32) return launch_filler<T, 32>(pass, a, st);
    if (a.width <= 64) return launch_filler<T, 64>(pass, a, st);
    if (a.width <= 96) return launch_filler<T, 96>(pass, a, st);
    return launch_filler<T, 128>(pass, a, st);
}
// The norms that half precision's backward passes scale by.
template <typename T>
int launch_range(const Params& a, hipStream_t st) {
    k_range<T><<<dim3((uint32_t)a.batch * (uint32_t)a.kv_heads, kRangeParts, 2), kThreads, 0, st>>>(a);
    return launch_status("attention");
}

}  // namespace attn
}  // namespace gefen
