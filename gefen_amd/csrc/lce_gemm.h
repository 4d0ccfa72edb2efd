// MFMA products of the linear cross entropy (linear_cross_entropy.hip), gfx950.
//
//   acc[m, n] = sum_k A[m, k] * B[n, k]     (16-bit operands, float32 accumulation)
//
// A workgroup owns a TM x TN tile; its waves own (32 WI) x (32 WJ) of it as
// v_mfma_f32_32x32x16 tiles.  Each operand is either K-major (a row of it is
// contiguous along k) or MN-major (stored as its transpose: a row holds one k).
// K advances BK at a time through NST LDS stages that are filled straight from
// global memory (buffer loads with the LDS destination), NST - 1 steps ahead, so an
// operand takes no registers on its way and one barrier ends a step.
//
// A lane's 16 bytes land at its own place of a wave's 1024 contiguous LDS bytes, so
// rows cannot be padded apart; instead the 16-byte chunks of a row are permuted by
// an XOR with bits of the row, and a lane fetches the chunk that belongs at its
// place.  K-major fragments are 16-byte reads of 32 rows at one k, MN-major ones come
// out of the transposing ds_read_b64_tr_b16, four rows at a time; the XOR spreads
// both over the banks.
//
// float32 operands are three bf16 planes (high, middle, low: 24 bits together), and
// the product is the sum of the six plane products above 2^-24 of it, run as six
// segments of one K loop.  An infinite element would meet the other side's middle and
// low parts, whose signs are their own, and leave NaN; a fourth plane holds the high
// part with zeros in place of what is not finite, and only high x high reads the other.
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
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Operand of a product: `rows` rows of `ld` elements.  K-major: rows are m (or n) and
// k < K <= ld; MN-major: rows are k and m (or n) runs along a row of `cols` elements.
// Tiles that reach past the rows or columns read the last ones again (their results
// are never stored, and past the end of K the other operand holds zeros), so every
// access is in bounds whatever the values.
struct Operand {
    const uint16_t* p;
    int64_t ld;
    int64_t plane;  // elements between the planes of a float32 operand
    int32_t rows, cols;
    int32_t finite;  // plane of the high parts without infinities (0: it has none)
};

template <bool F16_, int TM_, int TN_, int WI_, int WJ_, int BK_, int NST_, bool AMN_, bool BMN_>
struct Cfg {
    static constexpr bool F16 = F16_, AMN = AMN_, BMN = BMN_;
    static constexpr int TM = TM_, TN = TN_, WI = WI_, WJ = WJ_, BK = BK_, NST = NST_;
    static constexpr int WAVES_M = TM / (32 * WI), WAVES_N = TN / (32 * WJ);
    static constexpr int TT = 64 * WAVES_M * WAVES_N;
    static constexpr int A_ELEMS = TM * BK, B_ELEMS = TN * BK, STAGE = A_ELEMS + B_ELEMS;
    static constexpr int A_LOADS = A_ELEMS / 8 / TT, B_LOADS = B_ELEMS / 8 / TT;
    static constexpr int LDS_BYTES = NST * STAGE * 2;
    static constexpr int WGS = (160 << 10) / LDS_BYTES;                        // workgroups per CU
    static constexpr int EU = WGS * TT / 256 > 2 ? 2 : WGS * TT / 256;         // waves per SIMD to allocate for
    static_assert(A_LOADS * TT * 8 == A_ELEMS && B_LOADS * TT * 8 == B_ELEMS, "whole loads per thread");
};

// Place of chunk c of row r of a K-major tile of CPR chunks a row.
template <int CPR>
__device__ __forceinline__ int swz_k(int r, int c) {
    return c ^ (CPR == 8 ? (r & 7) : ((r >> 2) & 3));
}
// Place of chunk c of row r of an MN-major tile: 64-byte units by the row's low bits.
template <int CPR>
__device__ __forceinline__ int swz_mn(int r, int c) {
    return CPR >= 16 ? c ^ ((r & 3) << 2) : c;
}

// One operand's side of the K loop.
template <int ROWS, int BK, int LOADS, int TT, bool MN>
struct Loader {
    static constexpr int CPR = MN ? ROWS / 8 : BK / 8;  // 16-byte chunks of a tile row
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
                const int c = min(t0 + swz_mn<CPR>(r, s) * 8, o.cols - 8);
                voff[i] = (int)(((int64_t)r * o.ld + c) * 2);
            } else {
                const int row = min(t0 + r, o.rows - 1) - t0;
                voff[i] = (int)(((int64_t)row * o.ld + swz_k<CPR>(r, s) * 8) * 2);
            }
        }
        base = MN ? o.p : o.p + (int64_t)t0 * o.ld;
        step = MN ? (int64_t)BK * o.ld : BK;
    }
    // the loads of K step k (row k * BK on for MN: rows past the operand's are read as its last)
    __device__ __forceinline__ void issue(const Operand& o, int64_t plane_off, int k, uint16_t* lds) const {
        const uint16_t* at = base + plane_off + (int64_t)k * step;
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), (short)0, 0x7ffffff0, 0x00020000);
        const int wave = (int)threadIdx.x >> 6;
        bool tail = false;
        if constexpr (MN) tail = (k + 1) * BK > o.rows;
        if (!MN || !tail) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(lds + (wave * 64 + TT * i) * 8), 16, voff[i], 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int q = (int)threadIdx.x + TT * i;
                const int r = q / CPR;
                const int back = max(k * BK + r - (o.rows - 1), 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(lds + (wave * 64 + TT * i) * 8), 16,
                    (int)(voff[i] - (int64_t)back * o.ld * 2), 0, 0, 0);
            }
        }
    }
};

template <bool F16>
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Fragment of a K-major tile: rows row0 + lane % 32, k = 16 s + 8 (lane / 32) + 0..7.
template <int BK>
__device__ __forceinline__ bf16x8 frag_k(const uint16_t* tile, int row0, int s, int lane) {
    constexpr int CPR = BK / 8;
    const int r = lane & 31;
    const int c = swz_k<CPR>(r, 2 * s + (lane >> 5));
    return *reinterpret_cast<const bf16x8*>(tile + (row0 + r) * BK + c * 8);
}
// Fragment of an MN-major tile of ROWS elements a k: two transposing reads.  In each
// group of 16 lanes, lane 4 j + q points at k row j, elements 4 q .. 4 q + 3 of a 4 x 16
// block, and lane i receives element i of the rows 0 .. 3.
template <int ROWS>
__device__ __forceinline__ bf16x8 frag_mn(const uint16_t* tile, int row0, int s, int lane) {
    typedef __attribute__((address_space(3))) bf16x4 lds_v4;
    const int g = lane >> 4, j = (lane & 15) >> 2;
    const int k = 16 * s + 8 * (g >> 1) + j;
    const int e = row0 + 16 * (g & 1) + 4 * (lane & 3);  // element within the k row
    const int c = swz_mn<ROWS / 8>(j, e >> 3);
    const auto* p = (const __attribute__((address_space(3))) uint16_t*)(tile + k * ROWS + c * 8 + (e & 7));
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)(p + 4 * ROWS));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// The six plane products of float32 operands, smallest first (planes 0 high, 1
// middle, 2 low): low x high, high x low, middle x middle, middle x high, high x
// middle, high x high.
__device__ __forceinline__ int seg_plane(int code, int s, const Operand& o) {
    const int p = code >> (2 * s) & 3;
    return p == 0 && s != 5 ? o.finite : p;
}
constexpr int kSegA = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10;
constexpr int kSegB = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;

constexpr int kXcds = 8;    // workgroups go round-robin to the 8 XCDs
constexpr int kGroupM = 8;  // tile rows per band of the tile order

// Logical tile of workgroup b of nwg: consecutive tiles run on one XCD (one L2).
__device__ __forceinline__ int logical_block(int b, int nwg) {
    const int q = nwg / kXcds, r = nwg % kXcds;
    const int x = b % kXcds, k = b / kXcds;
    return x < r ? x * (q + 1) + k : r * (q + 1) + (x - r) * q + k;
}
// Tile (ti, tj) of tiles_m x tiles_n: bands of kGroupM tile rows, column by column.
__device__ __forceinline__ void tile_of(int t, int tiles_m, int tiles_n, int* ti, int* tj) {
    const int band = t / (kGroupM * tiles_n);
    const int rows_in = min(kGroupM, tiles_m - band * kGroupM);
    const int w = t - band * kGroupM * tiles_n;
    *ti = band * kGroupM + w % rows_in;
    *tj = w / rows_in;
}

template <int N>
__device__ __forceinline__ void wait_loads_and_sync() {
    // this wave's LDS reads are done and at most N of its loads are in flight, then the barrier
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// acc of the tile at (m0, n0) over K steps [k_from, k_to) of each of `segs` segments.
template <typename C>
__device__ __forceinline__ void product_tile(const Operand& A, const Operand& B, int m0, int n0, int k_from, int k_to,
                                             int segs, uint16_t* smem, f32x16 (&acc)[C::WI][C::WJ]) {
    constexpr int WI = C::WI, WJ = C::WJ, NST = C::NST;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / C::WAVES_N) * (32 * WI), wn = (wave % C::WAVES_N) * (32 * WJ);
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int j = 0; j < WJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    const int per = k_to - k_from, steps = per * segs;
    if (steps <= 0) return;
    Loader<C::TM, C::BK, C::A_LOADS, C::TT, C::AMN> la;
    Loader<C::TN, C::BK, C::B_LOADS, C::TT, C::BMN> lb;
    la.init(A, m0);
    lb.init(B, n0);
    int lk = k_from, lseg = 0;  // the next step to load (past the last one: the last again)
    auto issue = [&](int stage) {
        uint16_t* s = smem + stage * C::STAGE;
        la.issue(A, (segs > 1 ? seg_plane(kSegA, lseg, A) : 0) * A.plane, lk, s);
        lb.issue(B, (segs > 1 ? seg_plane(kSegB, lseg, B) : 0) * B.plane, lk, s + C::A_ELEMS);
        if (lk + 1 < k_to) ++lk;
        else if (lseg + 1 < segs) {
            lk = k_from;
            ++lseg;
        }
    };
    auto compute = [&](int stage) {
        const uint16_t* as = smem + stage * C::STAGE;
        const uint16_t* bs = as + C::A_ELEMS;
#pragma unroll
        for (int s = 0; s < C::BK / 16; ++s) {
            bf16x8 af[WI], bf[WJ];
#pragma unroll
            for (int i = 0; i < WI; ++i)
                af[i] = C::AMN ? frag_mn<C::TM>(as, wm + i * 32, s, lane) : frag_k<C::BK>(as, wm + i * 32, s, lane);
#pragma unroll
            for (int j = 0; j < WJ; ++j)
                bf[j] = C::BMN ? frag_mn<C::TN>(bs, wn + j * 32, s, lane) : frag_k<C::BK>(bs, wn + j * 32, s, lane);
#pragma unroll
            for (int i = 0; i < WI; ++i)
#pragma unroll
                for (int j = 0; j < WJ; ++j) acc[i][j] = mfma<C::F16>(af[i], bf[j], acc[i][j]);
        }
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(s);
    int stage = 0;
    for (int k = 0; k < steps; ++k) {
        wait_loads_and_sync<(NST - 2) * (C::A_LOADS + C::B_LOADS)>();
        issue(stage == 0 ? NST - 1 : stage - 1);
        compute(stage);
        stage = stage + 1 == NST ? 0 : stage + 1;
    }
    // the last loads (repeats) must have landed before LDS is used again
    wait_loads_and_sync<0>();
}

}  // namespace lce
}  // namespace gefen
