// dit_fp8_quant.hip — rows and weights to e4m3 with a power-of-two scale per block.
//
// A block's scale is 2^e, e the smallest integer (>= -127) with its largest finite
// magnitude a <= 448 2^e: with a = 1.f 2^x, e = x - 8 where 1.f <= 1.75 (448 =
// 1.75 2^8) and x - 7 where it is larger, integer arithmetic on a's bits.  The
// product x 2^-e is exact (or below e4m3's range), so the one rounding is the
// conversion's, to nearest even.
//
// HBM-bound: each value is read once (2 or 4 bytes) and a byte written.  Rows of 27258 x
// 2560 bf16 take 36 us (5.85 TB/s), 5498 x 6912 fp32 28 (6.8, in part from the memory-side
// cache), weights of 13824 x 2560 bf16 17.6 (6.0) and 2560 x 6912 fp32 15.0 (5.9), where
// device copies of 50 to 100 MiB reach 4.8 to 5.1 TB/s; rows of 58 x 2560 2.5 us, of 679 x
// 2560 3.1.
#include "dit_ops_internal.hpp"

namespace awa {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows are only known to be aligned to their elements
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

// 8 values of a block per lane, 16 lanes a block: bf16 columns 8 c .. 8 c + 7 of
// lane c in one 16-byte piece, fp32 columns 4 c .. and 64 + 4 c .. in two (so that
// the lanes of a block read and write neighbouring bytes).
template <typename T> struct Piece;
template <> struct Piece<uint16_t> {
    static constexpr int N = 1, W = 8;  // pieces, values in each
    static __device__ inline u32x4 load(const uint16_t* p) { return *reinterpret_cast<const u32x4_2*>(p); }
    static __device__ inline float value(const u32x4& r, int i) {
        return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
    }
    static __device__ inline u32x4 load_some(const uint16_t* p, int n) {
        u32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) r[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
        return r;
    }
};
template <> struct Piece<float> {
    static constexpr int N = 2, W = 4;
    static __device__ inline u32x4 load(const float* p) { return *reinterpret_cast<const u32x4_4*>(p); }
    static __device__ inline float value(const u32x4& r, int i) { return __uint_as_float(r[i]); }
    static __device__ inline u32x4 load_some(const float* p, int n) {
        u32x4 r = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < n) r[i] = __float_as_uint(p[i]);
        return r;
    }
};

// the largest finite magnitude's bits (0 if there is none)
__device__ inline uint32_t finite_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
template <typename T>
__device__ inline uint32_t top_of(const u32x4 (&r)[Piece<T>::N]) {
    uint32_t t = 0;
#pragma unroll
    for (int k = 0; k < Piece<T>::N; k++)
#pragma unroll
        for (int i = 0; i < Piece<T>::W; i++) t = max(t, finite_bits(Piece<T>::value(r[k], i)));
    return t;
}
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, false);
}
__device__ inline uint32_t max16(uint32_t v) {  // over 16 neighbouring lanes
    v = max(v, dpp<0xB1>(v));   // lane ^ 1
    v = max(v, dpp<0x4E>(v));   // lane ^ 2
    v = max(v, dpp<0x141>(v));  // mirrored in 8: the other four
    return max(v, dpp<0x140>(v));
}
// the scale's byte (e + 127) of a block with this largest magnitude
__device__ inline int scale_byte(uint32_t top) {
    return max((int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}
__device__ inline float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// the block's values to e4m3 at q (columns of the lane's first value)
template <typename T>
__device__ inline void store(const u32x4 (&r)[Piece<T>::N], float inv, uint8_t* q) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = 4 * h + i;
            v[i] = Piece<T>::value(r[j / Piece<T>::W], j % Piece<T>::W) * inv;
        }
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], p, true);
    }
    // past the caches: 5498 x 6912 bf16 24 -> 20 us (the product reads it from memory
    // either way where it is large)
    if constexpr (Piece<T>::N == 1) {
        __builtin_nontemporal_store((u32x2){w[0], w[1]}, reinterpret_cast<u32x2*>(q));
    } else {
        __builtin_nontemporal_store(w[0], reinterpret_cast<uint32_t*>(q));
        __builtin_nontemporal_store(w[1], reinterpret_cast<uint32_t*>(q + 64));
    }
}
// column of the lane's piece k inside its block
template <typename T>
__device__ inline int piece_col(int c, int k) { return Piece<T>::N == 1 ? 8 * c : 64 * k + 4 * c; }

template <typename T>
__device__ inline void load_block(u32x4 (&r)[Piece<T>::N], const T* row, int col0, int K, int c) {
#pragma unroll
    for (int k = 0; k < Piece<T>::N; k++) {
        const int col = col0 + piece_col<T>(c, k);
        if (col + Piece<T>::W <= K) r[k] = Piece<T>::load(row + col);
        else r[k] = Piece<T>::load_some(row + col, K - col);
    }
}

// A wave takes R rows of one group (512 columns, a scale word a row), the four waves of
// a workgroup neighbouring rows, whose words are neighbours too, and workgroups one
// after another the groups of the same rows.
template <typename T, int R>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane & 15, groups = (a.K + 511) >> 9;
    const int64_t pieces = ((int64_t)a.M + 4 * R - 1) / (4 * R) * groups;
    for (int64_t at = blockIdx.x; at < pieces; at += gridDim.x) {
        const int g = (int)(at % groups), row0 = ((int)(at / groups) * 4 + wave) * R;
        const int col0 = g * 512 + (lane >> 4) * 128;
        const bool in = col0 < a.kp;  // the last group may have fewer blocks
        u32x4 r[R][Piece<T>::N];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const T* row = reinterpret_cast<const T*>(a.x) + (int64_t)min(row0 + i, a.M - 1) * a.ldx;
            load_block<T>(r[i], row, col0, in ? a.K : 0, c);
        }
        uint32_t word = 0;  // lane i: the word of row row0 + i
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int byte = scale_byte(max16(top_of<T>(r[i])));
            uint32_t w = 0;
#pragma unroll
            for (int b = 0; b < 4; b++) w |= (uint32_t)__builtin_amdgcn_readlane(byte, 16 * b) << (8 * b);
            if (lane == i) word = w;
            if (in && row0 + i < a.M)
                store<T>(r[i], inverse_scale(byte), a.q + (int64_t)(row0 + i) * a.kp + col0 + piece_col<T>(c, 0));
        }
        if (lane < R && row0 + lane < a.M) a.scale[g * a.ld_scale + row0 + lane] = word;
    }
}

// A workgroup takes a block of 128 x 128: 16 rows a pass, all of it in registers.
template <typename T>
__global__ __launch_bounds__(256) void quant_blocks_kernel(QuantArgs a) {
    __shared__ uint32_t tops[4];
    const int kbs = (a.K + 511) / 512 * 4;
    const int kb = blockIdx.x % kbs, nb = blockIdx.x / kbs, tid = threadIdx.x;
    uint8_t* byte_at = reinterpret_cast<uint8_t*>(a.scale + (kb >> 2) * a.ld_scale + nb) + (kb & 3);
    if (kb * 128 >= a.kp) {  // a byte of the last word without a block
        if (tid == 0) *byte_at = 0;
        return;
    }
    const int c = tid & 15, r0 = nb * 128 + (tid >> 4);
    u32x4 r[8][Piece<T>::N];
#pragma unroll
    for (int i = 0; i < 8; i++) {  // rows past the end repeat the last one, which moves no maximum
        const T* row = reinterpret_cast<const T*>(a.x) + (int64_t)min(r0 + 16 * i, a.M - 1) * a.ldx;
        load_block<T>(r[i], row, kb * 128, a.K, c);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, top_of<T>(r[i]));
    top = max16(top);
    top = max(max((uint32_t)__builtin_amdgcn_readlane((int)top, 0), (uint32_t)__builtin_amdgcn_readlane((int)top, 16)),
              max((uint32_t)__builtin_amdgcn_readlane((int)top, 32), (uint32_t)__builtin_amdgcn_readlane((int)top, 48)));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const int byte = scale_byte(top);
    if (tid == 0) *byte_at = (uint8_t)byte;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = r0 + 16 * i;
        if (row < a.M)
            store<T>(r[i], inverse_scale(byte), a.q + (int64_t)row * a.kp + kb * 128 + piece_col<T>(c, 0));
    }
}

template <typename T, int R>
void rows_launch(const QuantArgs& a, hipStream_t s) {
    const int64_t pieces = ((int64_t)a.M + 4 * R - 1) / (4 * R) * ((a.K + 511) / 512);
    const unsigned blocks = (unsigned)(pieces < (1 << 22) ? pieces : 1 << 22);
    hipLaunchKernelGGL((quant_rows_kernel<T, R>), dim3(blocks), dim3(256), 0, s, a);
}
// two rows a wave once that leaves 8 workgroups per CU (27258 x 2560 bf16 36.5 us; one row
// 38.0, four 37.6)
template <typename T>
void rows(const QuantArgs& a, hipStream_t s) {
    if ((int64_t)a.M * ((a.K + 511) / 512) >= 16384) rows_launch<T, 2>(a, s);
    else rows_launch<T, 1>(a, s);
}

}  // namespace

hipError_t launch_quant_rows(int dtype, const QuantArgs& a, hipStream_t s) {
    if (dtype == AWA_F32) rows<float>(a, s);
    else rows<uint16_t>(a, s);
    return hipGetLastError();
}

hipError_t launch_quant_blocks(int dtype, const QuantArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.M + 127) / 128 * ((a.K + 511) / 512 * 4)));
    if (dtype == AWA_F32) hipLaunchKernelGGL((quant_blocks_kernel<float>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((quant_blocks_kernel<uint16_t>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace awa
