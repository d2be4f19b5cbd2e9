// dit_fp8_gemm.hip — products of e4m3 rows with power-of-two block scales.
//
// C = A W^T with A [M][K] (a scale per row and 128 columns) and W [N][K] (a scale
// per 128 x 128).  As the bf16 GEMM (dit_gemm.hip) the kernels form the transposed
// product, W's rows as the matrix instruction's rows and A's as its columns, so
// that a lane ends with four consecutive output features of one activation row.
// Which columns of a block a lane holds does not matter as long as both operands
// agree.
//
// Precision.  The 8-bit matrix instructions sum their products in groups of eight
// consecutive columns, aligned to the group's largest product with 13 bits below
// its leading one (measured; further additions keep fp32's 24 bits): the sum of a
// block is off by 1.5e-5 of its size.  bf16 holds every e4m3 value, times any
// power of two, and the bf16 instructions keep fp32's bits, at half the rate.
#include "dit_ops_internal.hpp"

namespace awa {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// scale byte b to 2^(b - 127)
__device__ inline float scale_of(int b) { return __uint_as_float(b ? (uint32_t)b << 23 : 0x400000u); }

// eight e4m3 values times a power of two as bf16
__device__ inline bf16x8 widen(int lo, int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 16 features x 16 rows per workgroup, K in parts over its waves.
constexpr int WAVES = 4;
__global__ __launch_bounds__(64 * WAVES) void gemm_fp8_few_kernel(Fp8Gemm p) {
    __shared__ f32x4 part[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int n0 = (blockIdx.x % p.n_tiles) * 16, m0 = (blockIdx.x / p.n_tiles) * 16;
    const int wr = min(n0 + r, p.N - 1), ar = min(m0 + r, p.M - 1);  // rows past the end repeat the last
    const uint8_t* wp = p.W + (int64_t)wr * p.K + 16 * q;
    const uint8_t* ap = p.A + (int64_t)ar * p.K + 16 * q;
    const uint8_t* wsp = reinterpret_cast<const uint8_t*>(p.ws + (n0 >> 7));
    const uint8_t* asp = reinterpret_cast<const uint8_t*>(p.as + ar);
    const int nk = p.K >> 7, k0 = nk * wave / WAVES, k1 = nk * (wave + 1) / WAVES;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int kb = k0; kb < k1; kb++) {
        const int64_t g = kb >> 2;
        const float sw = scale_of(wsp[4 * g * p.ld_ws + (kb & 3)]), sa = scale_of(asp[4 * g * p.ld_as + (kb & 3)]);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const i32x4 w = *reinterpret_cast<const i32x4*>(wp + kb * 128 + 64 * h);
            const i32x4 a = *reinterpret_cast<const i32x4*>(ap + kb * 128 + 64 * h);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[0], w[1], sw), widen(a[0], a[1], sa), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[2], w[3], sw), widen(a[2], a[3], sa), acc, 0, 0, 0);
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; w++) acc += part[w][lane];
    const int m = m0 + r, n = n0 + 4 * q;
    if (m >= p.M) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < p.N) {
            const float v = acc[i] + (p.bias ? p.bias[n + i] : 0.f);
            if (p.c_f32) reinterpret_cast<float*>(p.C)[m * p.ldc + n + i] = v;
            else reinterpret_cast<uint16_t*>(p.C)[m * p.ldc + n + i] = (uint16_t)bf16x2_rne(v, v);
        }
}

}  // namespace

hipError_t launch_gemm_fp8(Fp8Gemm& p, hipStream_t s) {
    p.n_tiles = (p.N + 15) / 16;
    p.m_tiles = (p.M + 15) / 16;
    hipLaunchKernelGGL(gemm_fp8_few_kernel, dim3(p.n_tiles * p.m_tiles), dim3(64 * WAVES), 0, s, p);
    return hipGetLastError();
}

}  // namespace awa
