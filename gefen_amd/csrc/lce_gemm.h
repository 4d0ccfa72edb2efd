// MFMA products of the linear cross entropy (linear_cross_entropy.hip), gfx950.
//
//   acc[m, n] = sum_k A[m, k] * B[n, k]     (16-bit operands, float32 accumulation)
//
// A workgroup owns a TM x TN tile; its waves own WM x WN of it as v_mfma_f32_16x16x32
// tiles (of the two MFMA shapes this one moves the accumulators half as often per
// operation: at full load the clock is set by power, and 16x16x32 ran 8% faster than
// 32x32x16 on the logits' product).  Each operand is either K-major (a row of it is
// contiguous along k) or MN-major (stored as its transpose: a row holds one k).
// A workgroup stays on its CU and takes tile after tile (product_stream).
// K advances BK at a time through NST LDS stages that are filled straight from
// global memory (buffer loads with the LDS destination), NST - 1 steps ahead, so an
// operand takes no registers on its way and one barrier ends a step.
//
// A lane's 16 bytes land at its own place of a wave's 1024 contiguous LDS bytes, so
// rows cannot be padded apart; instead the 16-byte chunks of a row are permuted by
// an XOR with bits of the row, and a lane fetches the chunk that belongs at its
// place.  K-major fragments are 16-byte reads of 16 rows at four k chunks, MN-major ones
// come out of the transposing ds_read_b64_tr_b16; the XOR spreads both over all banks
// (no conflicts counted).
//
// Bound by the matrix cores and the power they draw: the products of 8192 x 128256 x 4096
// (8.6e12 bf16 operations each) take 6.8 to 7.0 ms for the logits with all that is kept of
// them (1.23 to 1.26 PFLOP/s), 6.4 to 6.6 ms for dh (1.30 to 1.35) and 7.1 to 7.3 ms for dW
// (1.18 to 1.21), from card to card, MFMA busy 65, 69 and 61% of the cycles at a clock of 1.82
// to 1.9 GHz; the vendor's library reaches 1.29, 1.24 and 1.05 on the bare products.  Waves of 128 x 128 (half the waves, a third less LDS traffic) were 20%
// slower: one wave per SIMD has nothing to cover its waits with.  Steps of 32 in four or
// five stages lose to steps of 64 in two (twice the barriers).
//
// Operands of more than 16 bits are planes, and a product of them is several segments
// of one K loop, the small ones first: a float32 value is a half-precision high part and
// a low part of what the high one leaves, 22 bits together, and low x high, high x low
// and high x high hold the product to 2^-22 of it.  Half-precision low parts are stored
// times 2^11, in the range of the high ones, and the accumulators are scaled back
// (exactly) before the last segment.  An infinite element would meet the other side's
// low parts, whose signs are their own, and leave NaN: the low segments read a third
// plane, the high parts with zeros in place of what is not finite.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "capi_internal.h"
#include "common.h"

namespace gefen {
namespace lce {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Operand of a product: `rows` rows of `ld` elements.  K-major: rows are m (or n) and
// k < K <= ld; MN-major: rows are k and m (or n) runs along a row of `cols` elements.
// Tiles that reach past the rows or columns read the last ones again (their results
// are never stored, and past the end of K the other operand holds zeros), so every
// access is in bounds whatever the values.
struct Operand {
    const uint16_t* p;
    int64_t ld;
    int64_t plane;  // elements between planes
    int32_t rows, cols;
    uint32_t planes;  // plane of each segment, two bits each
};

constexpr float kLowScale = 2048.0f;  // of half-precision low parts

template <bool F16_, int TM_, int TN_, int WM_, int WN_, int BK_, int NST_, bool AMN_, bool BMN_, int GROUP_M_,
          bool STREAM_A_ = false>
struct Cfg {
    static constexpr bool F16 = F16_, AMN = AMN_, BMN = BMN_;
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, BK = BK_, NST = NST_;
    static constexpr int WI = WM / 16, WJ = WN / 16;
    static constexpr int WAVES_M = TM / WM, WAVES_N = TN / WN;
    static constexpr bool STREAM_A = STREAM_A_;  // A is read once by the whole launch
    static constexpr int GROUP_M = GROUP_M_;  // tile rows per band of the tile order
    static constexpr int TT = 64 * WAVES_M * WAVES_N;
    static constexpr int A_ELEMS = TM * BK, B_ELEMS = TN * BK, STAGE = A_ELEMS + B_ELEMS;
    static constexpr int A_LOADS = A_ELEMS / 8 / TT, B_LOADS = B_ELEMS / 8 / TT;
    static constexpr int LDS_BYTES = NST * STAGE * 2;
    static constexpr int WGS = (160 << 10) / LDS_BYTES;                 // workgroups per CU
    static constexpr int EU = WGS * TT / 256 > 2 ? 2 : WGS * TT / 256;  // waves per SIMD to allocate for
    static_assert(A_LOADS * TT * 8 == A_ELEMS && B_LOADS * TT * 8 == B_ELEMS, "whole loads per thread");
    static_assert(BK == 64, "swizzle_k, two slices of 32");
};

// Place of 16-byte chunk c of row r of a K-major tile (eight chunks a row).
__device__ __forceinline__ int swizzle_k(int r, int c) { return c ^ ((r >> 1) & 7); }
// Place of chunk c of k row r of an MN-major tile (sixteen or more chunks a row): 32-byte
// units by bits 0, 1 and 3 of the row, the rows that one transposing read covers.
__device__ __forceinline__ int swizzle_mn(int r, int c) { return c ^ (((r & 3) | ((r >> 3) & 1) << 2) << 1); }

typedef int i32x4 __attribute__((ext_vector_type(4)));
// LDS pointers keep their address space: no check for null on the way to an offset.
typedef __attribute__((address_space(3))) uint16_t lds_u16;

// 64 lanes' 16 bytes at base + voff to the 1024 LDS bytes at lds.  Written as assembly
// because the compiler otherwise holds every transposing LDS read back until all such
// loads in flight have landed; it has no register result, and wait_loads_and_sync
// waits for it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the compiler sets it before each use of its own
template <bool STREAM>
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, int voff, uint32_t lds) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds), "v"(voff), "s"(rsrc)
                     : "m0");
    else asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "m0");
}
#pragma clang diagnostic pop

// One operand's side of the K loop.
template <int ROWS, int BK, int LOADS, int TT, bool MN, bool STREAM>
struct Loader {
    static constexpr int CPR = MN ? ROWS / 8 : BK / 8;  // 16-byte chunks of a tile row
    static_assert(!MN || CPR >= 16, "swizzle_mn");
    int voff[LOADS];     // byte offset of this thread's chunk of each load
    const uint16_t* base;
    int64_t step;        // elements that a K step advances

    // t0: first m (or n) of the tile
    __device__ __forceinline__ void init(const Operand& o, int t0) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int q = (int)threadIdx.x + TT * i;
            const int r = q / CPR, s = q % CPR;
            if constexpr (MN) {
                const int c = min(t0 + swizzle_mn(r, s) * 8, o.cols - 8);
                voff[i] = (int)(((int64_t)r * o.ld + c) * 2);
            } else {
                const int row = min(t0 + r, o.rows - 1) - t0;
                voff[i] = (int)(((int64_t)row * o.ld + swizzle_k(r, s) * 8) * 2);
            }
        }
        base = MN ? o.p : o.p + (int64_t)t0 * o.ld;
        step = MN ? (int64_t)BK * o.ld : BK;
    }
    // the loads of K step k; MN-major rows past the operand's are read as its last one
    __device__ __forceinline__ void issue(const Operand& o, int64_t plane_off, int k, lds_u16* lds) const {
        const uint64_t at = reinterpret_cast<uint64_t>(base + plane_off + (int64_t)k * step);
        // raw buffer: every offset below is in bounds, the range covers any of them
        const i32x4 rsrc = {(int)(uint32_t)at, (int)((at >> 32) & 0xffff), 0x7ffffff0, 0x00020000};
        const uint32_t l0 =
            __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds + ((int)threadIdx.x >> 6) * 512));
        if (MN && (k + 1) * BK > o.rows) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = ((int)threadIdx.x + TT * i) / CPR;
                const int back = max(k * BK + r - (o.rows - 1), 0);
                load_to_lds<STREAM>(rsrc, (int)(voff[i] - (int64_t)back * o.ld * 2), l0 + TT * i * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) load_to_lds<STREAM>(rsrc, voff[i], l0 + TT * i * 16);
        }
    }
};

template <bool F16>
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Fragment of a K-major tile: rows row0 + lane % 16, k = 32 s + 8 (lane / 16) + 0..7.
template <int BK>
__device__ __forceinline__ bf16x8 frag_k(const lds_u16* tile, int row0, int s, int lane) {
    const int r = lane & 15;
    typedef __attribute__((address_space(3))) bf16x8 lds_v8;
    return *(const lds_v8*)(tile + (row0 + r) * BK + swizzle_k(r, 4 * s + (lane >> 4)) * 8);
}
// Fragment of an MN-major tile of ROWS elements a k: two transposing reads.  In each
// group of 16 lanes, lane 4 j + q points at k row j, elements 4 q .. 4 q + 3 of a 4 x 16
// block, and lane i receives element i of the rows 0 .. 3.
template <int ROWS>
__device__ __forceinline__ bf16x8 frag_mn(const lds_u16* tile, int row0, int s, int lane) {
    typedef __attribute__((address_space(3))) bf16x4 lds_v4;
    const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);  // within the slice of 32
    const int e = row0 + 4 * (lane & 3);
    const lds_u16* p = tile + (32 * s + k) * ROWS + swizzle_mn(k, e >> 3) * 8 + (e & 7);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)(p + 4 * ROWS));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

constexpr int kXcds = 8;    // workgroups go round-robin to the 8 XCDs

// Logical tile of workgroup b of nwg: consecutive tiles run on one XCD (one L2).
__device__ __forceinline__ int logical_block(int b, int nwg) {
    const int q = nwg / kXcds, r = nwg % kXcds;
    const int x = b % kXcds, k = b / kXcds;
    return x < r ? x * (q + 1) + k : r * (q + 1) + (x - r) * q + k;
}
// Tile (ti, tj) of tiles_m x tiles_n: bands of GROUP_M tile rows, column by column.
template <int GROUP_M>
__device__ __forceinline__ void tile_of(int t, int tiles_m, int tiles_n, int* ti, int* tj) {
    const int band = t / (GROUP_M * tiles_n);
    const int rows_in = min(GROUP_M, tiles_m - band * GROUP_M);
    const int w = t - band * GROUP_M * tiles_n;
    *ti = band * GROUP_M + w % rows_in;
    *tj = w / rows_in;
}

template <int N>
__device__ __forceinline__ void wait_loads_and_sync() {
    // this wave's LDS reads are done and at most N of its loads are in flight, then the barrier
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A unit of work: the tile at (m0, n0) over K steps [k0, k1) of each segment.
struct Unit {
    int m0, n0, k0, k1;
};

// The units first, first + stride, ... below `total` of this workgroup as one stream of K
// steps: the loads run ahead across the end of a unit, so that the next one's operands
// arrive while this one's results are written.  unit_of(u) names unit u; finish(u, unit,
// acc) takes its sums: acc[i][j][r] is m = m0 + (wave's) + 16 i + 4 (lane / 16) + r, n =
// n0 + (wave's) + 16 j + lane % 16.  Every unit has a K step at least.
template <typename C, typename UnitOf, typename Finish>
__device__ __forceinline__ void product_stream(const Operand& A, const Operand& B, int segs, int first, int total,
                                               int stride, lds_u16* smem, UnitOf unit_of, Finish finish) {
    constexpr int WI = C::WI, WJ = C::WJ, NST = C::NST, NS = C::BK / 32;
    constexpr int LOADS = C::A_LOADS + C::B_LOADS;
    constexpr int READS = WI * (C::AMN ? 2 : 1) + WJ * (C::BMN ? 2 : 1);   // LDS reads of a slice
    constexpr int PER = (2 * READS + WI * WJ - 1) / (WI * WJ);             // of them after each MFMA
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / C::WAVES_N) * C::WM, wn = (wave % C::WAVES_N) * C::WN;
    Loader<C::TM, C::BK, C::A_LOADS, C::TT, C::AMN, C::STREAM_A> la;
    Loader<C::TN, C::BK, C::B_LOADS, C::TT, C::BMN, false> lb;
    // the next step to load (past the last one: the last again)
    int lu = first, lk, lseg = 0;
    Unit load = unit_of(first);
    la.init(A, load.m0);
    lb.init(B, load.n0);
    lk = load.k0;
    auto issue = [&](int stage) __attribute__((always_inline)) {
        lds_u16* s = smem + stage * C::STAGE;
        la.issue(A, (int64_t)(A.planes >> (2 * lseg) & 3u) * A.plane, lk, s);
        lb.issue(B, (int64_t)(B.planes >> (2 * lseg) & 3u) * B.plane, lk, s + C::A_ELEMS);
        if (lk + 1 < load.k1) {
            ++lk;
        } else if (lseg + 1 < segs) {
            lk = load.k0;
            ++lseg;
        } else if (lu + stride < total) {
            lu += stride;
            load = unit_of(lu);
            la.init(A, load.m0);
            lb.init(B, load.n0);
            lk = load.k0;
            lseg = 0;
        }
    };
    bf16x8 af[2][WI], bf[2][WJ];
    auto read = [&](int stage, int s) __attribute__((always_inline)) {
        const lds_u16* as = smem + stage * C::STAGE;
        const lds_u16* bs = as + C::A_ELEMS;
#pragma unroll
        for (int i = 0; i < WI; ++i)
            af[s & 1][i] = C::AMN ? frag_mn<C::TM>(as, wm + i * 16, s, lane) : frag_k<C::BK>(as, wm + i * 16, s, lane);
#pragma unroll
        for (int j = 0; j < WJ; ++j)
            bf[s & 1][j] = C::BMN ? frag_mn<C::TN>(bs, wn + j * 16, s, lane) : frag_k<C::BK>(bs, wn + j * 16, s, lane);
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(s);
    int stage = 0;
    for (int u = first; u < total; u += stride) {
        const Unit unit = unit_of(u);
        const int per = unit.k1 - unit.k0, steps = per * segs;
        f32x4 acc[WI][WJ];
#pragma unroll
        for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int j = 0; j < WJ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < steps; ++k) {
            if (C::F16 && k == steps - per && segs > 1) {
#pragma unroll
                for (int i = 0; i < WI; ++i)
#pragma unroll
                    for (int j = 0; j < WJ; ++j) acc[i][j] *= 1.0f / kLowScale;
            }
            // this step's stage has landed, and every wave is done with the one to fill next
            wait_loads_and_sync<(NST - 2) * LOADS>();
            __builtin_amdgcn_sched_barrier(0);
            issue(stage == 0 ? NST - 1 : stage - 1);
            read(stage, 0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (s + 1 < NS) read(stage, s + 1);
#pragma unroll
                for (int i = 0; i < WI; ++i)
#pragma unroll
                    for (int j = 0; j < WJ; ++j) acc[i][j] = mfma<C::F16>(af[s & 1][i], bf[s & 1][j], acc[i][j]);
            }
            // the next slice's LDS reads between this slice's MFMAs (0x008 MFMA, 0x100 LDS read)
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int t = 0; t < WI * WJ; ++t) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (s + 1 < NS && t * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
            stage = stage + 1 == NST ? 0 : stage + 1;
        }
        finish(u, unit, acc);
    }
    // the last loads (repeats) must have landed before the workgroup gives its LDS back
    wait_loads_and_sync<0>();
}

}  // namespace lce
}  // namespace gefen
