// dit_cross_device.hpp — fragments, LDS tiles and reductions of the attention kernels of dit_train.h.
//
// All products are 16 x 16 x 32 with eight values of the summed axis a lane: lane 16 g + i holds values
// 8 g .. 8 g + 7 of row (column) i.  For bf16 that is one matrix instruction; for fp32 it is eight of
// 16 x 16 x 4, the j-th on the lanes' j-th values.  A result's lane 16 g + i holds rows 4 g .. 4 g + 3 of
// column i.  So where 32 rows of a result (two blocks of 16) are the summed axis of the next product, a lane
// already holds eight of them, {4 g + j, 16 + 4 g + j}, and the other operand is read in that order.
#pragma once

#include <type_traits>

#include "dit_device.hpp"
#include "dit_train_internal.hpp"

namespace awa {
namespace cross {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) bf16x4 lbf16x4_t;

struct Bf16 {
    static constexpr int SIZE = 2;
    static constexpr bool WHOLE = false;
    using Frag = bf16x8;
    static __device__ inline Frag zero() { return (bf16x8)(__bf16)0.f; }
    static __device__ inline f32x4 mma(const Frag& a, const Frag& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // two blocks of a result as the next product's operand (rounded: see Bf16Whole), and that product
    using Packed = Frag;
    static __device__ inline Packed pack(const f32x4& lo, const f32x4& hi) {
        const f32x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_convertvector(v, bf16x8);
    }
    static __device__ inline f32x4 mma_packed(const Frag& a, const Packed& b, const f32x4& c) { return mma(a, b, c); }
    static __device__ inline float dot(const Frag& a, const Frag& b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) s = __builtin_fmaf((float)a[i], (float)b[i], s);
        return s;
    }
    static __device__ inline Frag load(const char* p) { return __builtin_bit_cast(Frag, *reinterpret_cast<const u32x4*>(p)); }
    // four consecutive channels
    static __device__ inline void store4(char* p, const f32x4& v) {
        *reinterpret_cast<uint2*>(p) = make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
    }
    // Two neighbouring blocks of 16 channels of a row whose lane 16 g + i holds channels 4 g .. 4 g + 3 of both: neighbouring
    // lane groups exchange halves, so that each stores 16 bytes and the four 64 in a row (one after the other at 8 bytes
    // a lane, 16384 queries x 128 keys x 20 heads take 52 us, so 44).
    static __device__ inline void store_blocks(char* row, int db, int g, int d, const f32x4& a, const f32x4& b) {
        const auto x = __builtin_amdgcn_permlane16_swap(bf16x2_rne(a[0], a[1]), bf16x2_rne(b[0], b[1]), false, false);
        const auto y = __builtin_amdgcn_permlane16_swap(bf16x2_rne(a[2], a[3]), bf16x2_rne(b[2], b[3]), false, false);
        const int ch = 16 * (db + (g & 1)) + 8 * (g >> 1);
        if (ch < d) *reinterpret_cast<u32x4*>(row + 2 * ch) = (u32x4){x[0], y[0], x[1], y[1]};
    }
};
// bf16 tensors whose probabilities (and dS) keep 16 bits, as the sum of two bf16 values and in two products (an infinity,
// whose rest is none, becomes NaN).  Rounded to one value they cost a result as much again as its own rounding, at three
// quarters of the time, so that a caller chooses.  2-norm of the error over the result's, heads of 128: results 2.32e-3 in one
// product and 1.66e-3 (their rounding) in two, dq 2.37e-3 and 1.68e-3.  27200 queries x 1024 keys x 20 heads: forward 306 to
// 311 us and 382 to 404; 16384 x 384 83 and 105 to 108, gradients 316 and 370; 5440 x 58 15.3 and 15.6, 56 and 61.
struct Bf16Whole : Bf16 {
    static constexpr bool WHOLE = true;
    struct Packed {
        Frag top, rest;
    };
    static __device__ inline Packed pack(const f32x4& lo, const f32x4& hi) {
        const f32x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        const bf16x8 top = __builtin_convertvector(v, bf16x8);
        return {top, __builtin_convertvector(v - __builtin_convertvector(top, f32x8), bf16x8)};
    }
    static __device__ inline f32x4 mma_packed(const Frag& a, const Packed& b, const f32x4& c) {
        return mma(a, b.top, mma(a, b.rest, c));
    }
};
struct F32 {
    static constexpr int SIZE = 4;
    static constexpr bool WHOLE = false;
    using Frag = f32x8;
    static __device__ inline Frag zero() { return (f32x8)0.f; }
    static __device__ inline f32x4 mma(const Frag& a, const Frag& b, const f32x4& c) {
        f32x4 r = c;
#pragma unroll
        for (int j = 0; j < 8; j++) r = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], r, 0, 0, 0);
        return r;
    }
    using Packed = Frag;
    static __device__ inline Packed pack(const f32x4& lo, const f32x4& hi) {
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ inline f32x4 mma_packed(const Frag& a, const Packed& b, const f32x4& c) { return mma(a, b, c); }
    static __device__ inline float dot(const Frag& a, const Frag& b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) s = __builtin_fmaf(a[i], b[i], s);
        return s;
    }
    static __device__ inline Frag load(const char* p) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 16);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ inline void store4(char* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
    static __device__ inline void store_blocks(char* row, int db, int g, int d, const f32x4& a, const f32x4& b) {
        const int ch = 16 * db + 4 * g;
        if (ch < d) store4(row + 4 * ch, a);
        if (ch + 16 < d) store4(row + 4 * (ch + 16), b);
    }
};

// How T's tensors are stored
template <typename T>
using Rows = std::conditional_t<T::SIZE == 4, F32, Bf16>;

// One LDS DMA instruction, 16 (4) bytes a lane to LDS at `to` + 16 (4) x lane from byte offset `at` of the resource.  From
// asm, because the compiler lets every transposed read wait for all DMA that it knows of; the kernels wait by themselves
// (wait_vmem_lds and a barrier) before anything reads the tile.  M0, the LDS address, is not used otherwise here.
__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(size_t)(const __attribute__((address_space(3))) char*)p);
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void dma16(const void* to, __amdgpu_buffer_rsrc_t from, uint32_t at) {
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 0\n\tbuffer_load_dwordx4 %[v], %[r], 0 offen lds"
                 :
                 : [v] "v"(at), [r] "s"(from), [m] "s"(lds_address(to))
                 : "memory", "m0");
}
__device__ inline void dma4(const void* to, __amdgpu_buffer_rsrc_t from, uint32_t at) {
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 0\n\tbuffer_load_dword %[v], %[r], 0 offen lds"
                 :
                 : [v] "v"(at), [r] "s"(from), [m] "s"(lds_address(to))
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Eight channels at byte offset `at` of a resource (zeros past it)
template <typename T>
__device__ inline typename T::Frag buffer_frag(__amdgpu_buffer_rsrc_t from, uint32_t at) {
    const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
    if constexpr (T::SIZE == 2) {
        return __builtin_bit_cast(typename T::Frag, lo);
    } else {
        const u32x4 hi = __builtin_amdgcn_raw_buffer_load_b128(from, at + 16, 0, 0);
        return __builtin_shufflevector(__builtin_bit_cast(f32x4, lo), __builtin_bit_cast(f32x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// An LDS tile: rows of 64 or 128 channels (DP = 96 has rows of 128, whose last channels nothing reads), 16-byte
// chunk c of row r at chunk c ^ swizzle(r).  LDS answers 256 bytes a cycle from 64 banks, so the 16 rows that read one
// chunk together, and the eight rows that 32 lanes of a transposed read (four rows that 64 lanes of fp32 columns) take two
// (four) neighbouring chunks of, have to begin at different ones.
template <typename T, int DP>
struct Tile {
    static constexpr int ROW = (DP == 64 ? 64 : 128) * T::SIZE, CHUNKS = ROW / 16, PER = 1024 / ROW;  // PER: rows of an instruction
    static __device__ inline int swizzle(int r) {
        if constexpr (T::SIZE == 4) return r & 15;
        if constexpr (DP == 64) r >>= 1;  // rows of half the banks
        return DP == 64 ? ((r & 3) << 1) | ((r >> 2) & 1) : ((r & 7) << 1) | ((r >> 3) & 1);
    }
    // eight channels 32 ks + 8 g .. of row `row`
    static __device__ inline typename T::Frag row_frag(const char* t, int row, int ks, int g) {
        const char* at = t + row * ROW;
        const int s = swizzle(row);
        if constexpr (T::SIZE == 2) {
            return __builtin_bit_cast(typename T::Frag, *reinterpret_cast<const u32x4*>(at + (((4 * ks + g) ^ s) << 4)));
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(at + (((8 * ks + 2 * g) ^ s) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(at + (((8 * ks + 2 * g + 1) ^ s) << 4));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // channel 16 db + lane % 16 of rows base + {4 g + j, 16 + 4 g + j}; base a multiple of 16
    static __device__ inline typename T::Frag column_frag(const char* t, int base, int db, int lane) {
        const int g = lane >> 4;
        if constexpr (T::SIZE == 2) {
            // lane 16 g + 4 i + a of a transposed read addresses row 4 g + i, channels 4 a .. 4 a + 3, and receives its
            // own channel's rows 4 g .. 4 g + 3
            const int r = 4 * g + ((lane >> 2) & 3), a = lane & 3;
            const char* at = t + (base + r) * ROW + (((2 * db + (a >> 1)) ^ swizzle(r)) << 4) + ((a & 1) << 3);
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lbf16x4_t*)at);
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lbf16x4_t*)(at + 16 * ROW));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            typename T::Frag f;
            const int c = 4 * db + ((lane >> 2) & 3);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = 4 * g + j;
                const char* at = t + (base + r) * ROW + ((c ^ swizzle(r)) << 4) + ((lane & 3) << 2);
                f[j] = *reinterpret_cast<const float*>(at);
                f[4 + j] = *reinterpret_cast<const float*>(at + 16 * ROW);
            }
            return f;
        }
    }
    // DMA instruction i of a tile: rows PER i .. of it, one 16-byte chunk a lane.  Rows that are not in `valid` (a bit
    // per row) and channels past head_d lie past the resource and become zeros.
    static __device__ inline void dma(char* t, int i, __amdgpu_buffer_rsrc_t from, int64_t row_bytes, uint64_t valid, int width,
                                      int lane) {
        const int row = i * PER + lane / CHUNKS, c = ((lane % CHUNKS) ^ swizzle(row)) << 4;
        const bool in = ((valid >> row) & 1) && c < width;
        const uint32_t at = in ? (uint32_t)(row * (uint32_t)row_bytes + c) : 0x80000000u;
        dma16(t + i * 1024, from, at);
    }
};

// An entry of a plan's table by the scalar cache (read-only memory at a wave-uniform index: as a vector load it would be
// waited for together with the tiles on their way)
template <typename S>
__device__ inline S table_entry(const S* table, int i) {
    constexpr int N = sizeof(S) / 4;
    typedef const __attribute__((address_space(4))) uint32_t* constant_t;
    const constant_t from = (constant_t)table + (size_t)__builtin_amdgcn_readfirstlane(i) * N;
    uint32_t w[N];
#pragma unroll
    for (int k = 0; k < N; k++) w[k] = from[k];
    S s;
    __builtin_memcpy(&s, w, sizeof(S));
    return s;
}

// Over the four lanes l % 16 + 16 i
__device__ inline float sum4(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// A row's results from its maximum and sum.  A row without keys, or with scores of -infinity alone, keeps the maximum and the sum
// that it starts with; a NaN leaves no mark on the maximum (fmaxf takes the other operand), but the sum is one; and a sum
// of 0 beside a maximum means that this passed fp32 on the way to a power of two.
__device__ inline bool no_score(float top, float sum) { return top == -INFINITY && sum == 0.f; }
__device__ inline float inverse_of(float top, float sum) { return no_score(top, sum) ? 0.f : 1.f / sum; }
__device__ inline float lse_of(float top, float sum, float scale) {
    if (no_score(top, sum)) return -INFINITY;
    return sum > 0.f ? top * scale + LN2 * __builtin_amdgcn_logf(sum) : NAN;
}

}  // namespace cross
}  // namespace awa
