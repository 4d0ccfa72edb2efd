// Tiles of the attention kernels (attention.hip), gfx950.
//
// Every product of attention and of its gradients is taken with one side in registers and
// the other in LDS, 32 x 32 at a time (v_mfma_f32_32x32x16 of 16-bit operands,
// v_mfma_f32_32x32x2_f32 of float32 ones):
//
//   rows:     acc[m, n] += sum_k tile[m, k] x[n, k]      k along the head's width
//   columns:  acc[d, n] += sum_m tile[m, d] p[m, n]      m along the tile's rows
//
// A lane owns one n (lane % 32) throughout: a query in the forward pass and in dQ, a key in
// dK and dV.  The accumulator of a rows product holds p[m, n] for m = 8 (i / 4) + 4 h + i % 4
// (i = 0..15, h = lane / 32), and the columns product takes it as it lies: the order of m
// within a matrix instruction is free as long as both sides agree, so the tile's side is read
// in that order (16-bit: two transposing ds_read_b64_tr_b16, four rows each) and p never
// moves between lanes.  The softmax's maximum and sum need one exchange, between the halves.
//
// A tile is BN rows of DP elements, DP the head's width rounded up to 32 with zeros.  It is
// filled straight from global memory (loads with the LDS destination: no registers on the
// way), where a wave's 64 lanes write 1024 contiguous bytes; so rows are not padded, but the
// 16-byte chunks of a row are permuted by an XOR with bits of the row, and a lane fetches the
// chunk that belongs at its place.  The XOR spreads what one read takes at a time over all 64
// banks: 16 rows of one chunk, and 4 rows of four neighbouring ones (the transposing read).
// Heads whose rows are no whole aligned chunks come through registers (ASYNC false).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace gefen {
namespace attn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem {
    static constexpr int EPC = 16 / sizeof(T);     // elements of a 16-byte chunk
    using Raw = typename RawVec<sizeof(T)>::type;  // what LDS holds
    __device__ __forceinline__ static float value(Raw r) {
        T t;
        __builtin_memcpy(&t, &r, sizeof(T));
        return to_f32(t);
    }
};

// A rows product's step: 2 x EPC elements of k, lane half h holding k = 2 EPC c + EPC h + 0..
template <typename T>
__device__ __forceinline__ f32x16 mma_rows(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(f32x4, a)[i], __builtin_bit_cast(f32x4, b)[i], c,
                                                     0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, f16_t)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    }
}

// acc[m, n] - x[m], x float32: a product over three bfloat16 parts of x, which hold 24 bits of
// it.  A number of each row costs one read of a lane's chunk this way, where a lane's sixteen
// float32 numbers are four.
struct RowTerm {
    typedef __attribute__((address_space(3))) u32x4 lds_chunk;
    lds_chunk* p;  // a chunk a row: three parts and zeros
    __device__ __forceinline__ static u32x4 split(float x) {
        const __bf16 hi = (__bf16)x;
        const float r1 = x - (float)hi;
        const __bf16 mid = (__bf16)r1;
        const __bf16 lo = (__bf16)(r1 - (float)mid);
        return __builtin_bit_cast(u32x4, bf16x8{hi, mid, lo, (__bf16)0.0f, (__bf16)0.0f, (__bf16)0.0f, (__bf16)0.0f,
                                                (__bf16)0.0f});
    }
    __device__ __forceinline__ f32x16 subtract(int r0, int lane, f32x16 acc) const {
        const uint32_t one = lane < 32 ? 0xbf80bf80u : 0u;  // -1, -1, -1, 0 for k = 0 .. 3, zeros for the others
        const u32x4 b = {one, one & 0xffffu, 0u, 0u};
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p[r0 + (lane & 31)]),
                                                       __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    }
};

// Sixteen rows of p as the columns product takes them.
template <typename T>
struct PFrag {
    u32x4 v;
};
template <>
struct PFrag<float> {
    float v[8];
};
template <typename T>
__device__ __forceinline__ PFrag<T> pack(const f32x16& p, int chunk) {
    PFrag<T> out;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out.v[i] = p[8 * chunk + i];
    } else if constexpr (__is_same(T, f16_t)) {
        f16x8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (_Float16)p[8 * chunk + i];
        out.v = __builtin_bit_cast(u32x4, t);
    } else {
        bf16x8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (__bf16)p[8 * chunk + i];
        out.v = __builtin_bit_cast(u32x4, t);
    }
    return out;
}

// A columns product's step of 16-bit elements: a tile's chunk and sixteen rows of p.
template <typename T>
__device__ __forceinline__ f32x16 mma_chunk(u32x4 a, const PFrag<T>& p, f32x16 acc) {
    if constexpr (sizeof(T) == 2) acc = mma_rows<T>(a, p.v, acc);
    return acc;
}

// Zeros in place of what is not finite; *bad gets bits of kBadBits where there was any.  The
// largest exponent plus its lowest bit carries into the sign's place.
template <typename T>
constexpr uint32_t kBadBits = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
template <typename T>
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t x, uint32_t* bad) {
    constexpr uint32_t e = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, f16_t) ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t one = sizeof(T) == 4 ? 0x00800000u : __is_same(T, f16_t) ? 0x04000400u : 0x00800080u;
    const uint32_t t = ((x & e) + one) & kBadBits<T>;
    *bad |= t;
    if constexpr (sizeof(T) == 4) return x & ~(uint32_t)((int32_t)t >> 31);
    const uint32_t m = t >> 15;
    return x & ~((m << 16) - m);
}

// The XOR of row r's chunks, `chunks` a row.
constexpr __device__ __forceinline__ int chunk_xor(int r, int chunks) {
    return chunks % 16 == 0  ? (r & 3) << 2 | ((r >> 2) & 3)
           : chunks % 8 == 0 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3)
                             : (r >> 2) & 3;
}

// Rows of a tile that a wave sees.
struct RowRange {
    int lo, hi;
    __device__ __forceinline__ bool has(int r) const { return (uint32_t)(r - lo) < (uint32_t)(hi - lo); }
};

template <typename T, int BN, int DP>
struct Tile {
    static constexpr int EPC = Elem<T>::EPC, LD = DP;
    static constexpr int ELEMS = BN * LD, BYTES = ELEMS * (int)sizeof(T);
    static constexpr int CPR = DP / EPC;  // chunks of a row
    // LDS pointers keep their address space
    typedef __attribute__((address_space(3))) typename Elem<T>::Raw lds_t;
    typedef __attribute__((address_space(3))) u32x4 lds_chunk;
    lds_t* p;

    // element d of row r
    __device__ __forceinline__ static int place(int r, int d) {
        return r * LD + ((d / EPC) ^ chunk_xor(r, CPR)) * EPC + d % EPC;
    }
    __device__ __forceinline__ void put(int row, int c, u32x4 v) const { *(lds_chunk*)(p + place(row, c * EPC)) = v; }

    // chunk c of the rows product's left side: row r0 + lane % 32 (r0 a multiple of 32)
    __device__ __forceinline__ u32x4 row_chunk(int r0, int c, int lane) const {
        return *(const lds_chunk*)(p + r0 * LD + place(lane & 31, (2 * c + (lane >> 5)) * EPC));
    }
    // Whether every element of the tile is finite: two operations a word, where keeping what is
    // not out of the columns product takes five and a half.
    __device__ __forceinline__ bool all_finite(int lane) const {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < BYTES / (16 * 64); ++i) {
            const u32x4 w = ((const lds_chunk*)p)[64 * i + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4)
                    most = max(most, w[j] & 0x7fffffffu);
                else
                    most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most),
                                                                                  __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu)));
            }
        }
        if constexpr (sizeof(T) == 4) return !__any(most >= 0x7f800000u);
        constexpr uint32_t inf = __is_same(T, f16_t) ? 0x7c00u : 0x7f80u;
        return !__any((most & 0xffffu) >= inf || most >> 16 >= inf);
    }
    // The columns product's left side (16-bit elements): rows r0 .. r0 + 15 of columns d0 .. d0 + 31.
    // In each group of 16 lanes, lane 4 j + q points at row j, elements 4 q .. 4 q + 3.
    __device__ __forceinline__ u32x4 column_chunk(int r0, int d0, int lane) const {
        typedef __attribute__((address_space(3))) bf16x4 lds_v4;
        const int row = 4 * (lane >> 5) + ((lane & 15) >> 2);
        const int col = d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)(p + r0 * LD + place(row, col)));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_v4*)(p + r0 * LD + place(row + 8, col)));
        return __builtin_bit_cast(u32x4, bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    }
    // acc[d0 + .., n] += sum over rows r0 .. r0 + 15 (r0 a multiple of 16).  CHECK: rows
    // outside `rows` count as zeros whatever LDS holds there; of the others, what is not finite
    // does, and *bad tells (kBadBits).
    template <bool CHECK>
    __device__ __forceinline__ f32x16 mma_columns(const PFrag<T>& b, int r0, int d0, int lane, f32x16 acc,
                                                  RowRange rows, uint32_t* bad) const {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t a = p[r0 * LD + place(8 * (i / 4) + 4 * h + i % 4, d0 + (lane & 31))];
                if (CHECK) a = drop_nonfinite<T>(rows.has(r0 + 8 * (i / 4) + 4 * h + i % 4) ? a : 0u, bad);
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a), b.v[i], acc, 0, 0, 0);
            }
            return acc;
        } else {
            u32x4 a = column_chunk(r0, d0, lane);
            if (CHECK) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = r0 + 4 * h + 2 * (i & 1) + 8 * (i >> 1);
                    a[i] &= (rows.has(r) ? 0x0000ffffu : 0u) | (rows.has(r + 1) ? 0xffff0000u : 0u);
                    a[i] = drop_nonfinite<T>(a[i], bad);
                }
            }
            return mma_rows<T>(a, b.v, acc);
        }
    }
    // What the checked product has left out, for the rows in [lo, hi) that this lane's column
    // sees: infinities as they are, or (AS_NAN) NaN for any.
    template <bool AS_NAN, int DT>
    __device__ __forceinline__ void add_nonfinite(f32x16 (&acc)[DT], int rows, int lo, int hi, int lane) const {
        const int h = lane >> 5;
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
            const bool seen = r >= lo && r < hi;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float v = Elem<T>::value(p[place(r, 32 * dt + 8 * (i / 4) + 4 * h + i % 4)]);
                    const bool bad = (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
                    if (bad && seen) acc[dt][i] += AS_NAN ? __uint_as_float(0x7fc00000u) : v;
                }
        }
    }
};

// 16 bytes from each active lane's address, base (wave-uniform) + offset bytes, to its place
// after lds (wave-uniform): lane * 16.
// Written as assembly because the compiler otherwise holds every transposing LDS read back
// until all such loads in flight have landed; it has no register result, and
// wait_loads_and_sync waits for it.  The compiler counts no wait states into or inside the block,
// so it brings those that the load needs: one behind the write of m0, and five behind a vector
// instruction that wrote its base (which may be the last one before the block), the write of m0
// and s_nop 3 together.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the compiler sets it before each use of its own
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint64_t s = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                     __builtin_amdgcn_readfirstlane((int)lds)),
                 "v"(offset), "s"(s)
                 : "m0");
}
#pragma clang diagnostic pop
// This wave's loads to LDS have landed and its LDS reads are done, then the barrier.
__device__ __forceinline__ void wait_loads_and_sync() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// use(i, read(i)) for i < N, the reads DEPTH ahead of their uses.  Left alone the compiler puts an
// LDS read right before the matrix instruction that takes it and waits its latency out each time;
// the barriers let nothing but vector and scalar arithmetic across.
template <int N, int DEPTH, typename Read, typename Use>
__device__ __forceinline__ void stream(Read read, Use use) {
    u32x4 f[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH && i < N; ++i) f[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_barrier(0x6);
        use(i, f[i % DEPTH]);
        if (i + DEPTH < N) f[i % DEPTH] = read(i + DEPTH);
    }
}

// EPC elements from p, of which the first `n` exist (n >= 1); zeros for the others.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p, int n) {
    constexpr int EPC = Elem<T>::EPC;
    if (n >= EPC) return *reinterpret_cast<const typename RawAny<16, sizeof(T)>::type*>(p);
    u32x4 out = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
        if (i < n) {
            if constexpr (sizeof(T) == 4) out[i] = __float_as_uint(p[i]);
            else out[i / 2] |= (uint32_t)p[i].bits << (16 * (i & 1));
        }
    }
    return out;
}

// Four consecutive elements of which the first `n` exist.
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d, int n) {
    const AnyVec<T, 4> v = {{from_f32<T>(a), from_f32<T>(b), from_f32<T>(c), from_f32<T>(d)}};
    if (n >= 4) {
        using R = typename RawAny<sizeof(T) * 4, sizeof(T)>::type;
        typename RawVec<sizeof(T) * 4>::type r;
        __builtin_memcpy(&r, &v, sizeof(r));
        *reinterpret_cast<R*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = v.v[i];
    }
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int wave_min(int v) {
    for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
    return v;
}
__device__ __forceinline__ int wave_max(int v) {
    for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
    return v;
}

}  // namespace attn
}  // namespace gefen
