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
// its leading one (measured; further additions keep fp32's 24 bits).  A product has
// 8 bits, so it is whole up to 6 binades under the largest and loses less than 2^-13 of
// that below: at most 7 2^-13 of the sum of the groups' largest, with signs that follow
// the products'.  Root mean square before C's rounding, of the sums': 1.5e-5 for normal
// data (K = 2560 and 6912, all forms), 4.5e-5 with one column in eight 16 times the
// others, 8.4e-5 and 8.9e-5 with 256 and 2048 times: a 260th to a 43rd of bf16's step,
// and taken for bf16 C.  bf16 holds every e4m3 value, times any power of two, and the
// bf16 instructions keep fp32's bits, at half the rate.
#include "dit_device.hpp"
#include "dit_ops_internal.hpp"

namespace awa {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lptr_t;

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

// ---- few rows ---------------------------------------------------------------
//
// Up to 16 rows: 16 NI features per workgroup, the blocks of K in turn over its waves,
// whose sums meet in LDS (in the waves' order).  Bound by W, which is read once,
// straight into registers; A comes from the L2 again for every workgroup.  One row of
// 7680 x 2560 takes 5.4 us (19.7 MB of W: 3.6 TB/s), of 2560 x 6912 6.4, of 4096 x 11008 10.2
// (4.4 TB/s), 16 rows of 7680 x 2560 6.0, of which a launch and the fill of the chip are 2 to
// 3.  Widened to bf16: an 8-bit instruction would save nothing where W's bytes bound.
template <int NI, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void gemm_fp8_few_kernel(Fp8Gemm p) {
    __shared__ f32x4 part[WAVES][NI][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * (16 * NI);
    // rows past the end repeat the last
    const int row = min(r, p.M - 1);
    const uint8_t* ap = p.A + (int64_t)row * p.K + 16 * q;
    const uint8_t* asp = reinterpret_cast<const uint8_t*>(p.as + row);
    const uint8_t* wp[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) wp[i] = p.W + (int64_t)min(n0 + 16 * i + r, p.N - 1) * p.K + 16 * q;
    const uint8_t* wsp = reinterpret_cast<const uint8_t*>(p.ws + (n0 >> 7));
    const int nk = p.K >> 7;
    struct Block {
        i32x4 a[2], w[NI][2];
        int sw, sa;
    };
    auto load = [&](Block& b, int kb) __attribute__((always_inline)) {
        const int64_t g = kb >> 2;
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) b.w[i][h] = *reinterpret_cast<const i32x4*>(wp[i] + kb * 128 + 64 * h);
#pragma unroll
        for (int h = 0; h < 2; h++) b.a[h] = *reinterpret_cast<const i32x4*>(ap + kb * 128 + 64 * h);
        b.sw = wsp[4 * g * p.ld_ws + (kb & 3)];
        b.sa = asp[4 * g * p.ld_as + (kb & 3)];
    };
    f32x4 acc[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto sum = [&](const Block& b) __attribute__((always_inline)) {
        const float sw = scale_of(b.sw), sa = scale_of(b.sa);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bf16x8 a0 = widen(b.a[h][0], b.a[h][1], sa), a1 = widen(b.a[h][2], b.a[h][3], sa);
#pragma unroll
            for (int i = 0; i < NI; i++) {
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(b.w[i][h][0], b.w[i][h][1], sw), a0, acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(b.w[i][h][2], b.w[i][h][3], sw), a1, acc[i], 0, 0, 0);
            }
        }
    };
    // two blocks in flight
    Block b0, b1;
    if (wave < nk) load(b0, wave);
    for (int kb = wave; kb < nk; kb += 2 * WAVES) {
        if (kb + WAVES < nk) load(b1, kb + WAVES);
        sum(b0);
        if (kb + 2 * WAVES < nk) load(b0, kb + 2 * WAVES);
        if (kb + WAVES < nk) sum(b1);
    }
#pragma unroll
    for (int i = 0; i < NI; i++) part[wave][i][lane] = acc[i];
    __syncthreads();
    // wave i finishes feature block i
    if (wave >= NI) return;
    f32x4 c = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; w++) c += part[w][wave][lane];
    const int n = n0 + 16 * wave + 4 * q;
    if (r >= p.M) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < p.N) {
            const float v = c[i] + (p.bias ? p.bias[n + i] : 0.f);
            if (p.c_f32) reinterpret_cast<float*>(p.C)[r * p.ldc + n + i] = v;
            else reinterpret_cast<uint16_t*>(p.C)[r * p.ldc + n + i] = (uint16_t)bf16x2_rne(v, v);
        }
}

// ---- tiles ------------------------------------------------------------------
//
// Workgroup tile 32 NW NI (n) x 64 MJ (m), a block of K per stage, wave64 in a
// NW x 2 grid, NI x MJ accumulators of 32 x 32 per wave.  As in the bf16 GEMM the
// operands' 128-byte rows reach LDS by direct DMA into NS stages, 16-byte chunks at
// chunk ^ ((row >> 1) & 7), and each half block (64 columns, one instruction per
// accumulator) runs with the next half's fragment reads and, in the half that
// refills the freed stage, the DMA pieces between its instructions.  A row's scale
// word travels with its stage, and W's, which are the same for a whole wave.
//
// EXACT (fp32 C, and bf16 C where the caller asks for whole products): the fragments are
// widened to bf16 with their scales and take four 32x32x16 bf16 instructions in place of
// one 8-bit one.
//
// Bound by what a tile's operands take from the L2 where the tiles are small, and by the
// chip's power where they are large (a loop of 8-bit instructions alone reaches 4.0 to 4.1
// PFLOP/s, at 1.9 GHz).  bf16 C: 58 x 7680 x 2560 6.3 us, 679 x 2560 x 6912 19 to 21 (1.2
// PFLOP/s), 1237 x 1999 x 2816 14.6 to 15.1, 1400 x 13824 x 2560 52 (1.9).  fp32 C: 679 x
// 2560 x 6912 32 to 34 us (0.73), 5498 x 13824 x 2560 294 to 322 (1.2 to 1.3), 8192^3 728 to
// 752 (1.5; the library's bf16 product 1.31).  bf16 C of whole products: 58 x 7680 x 2560
// 7.4 us, 1237 x 1999 x 2816 22 to 24, 679 x 2560 x 6912 32, 5498 x 13824 x 2560 278 to 305.
constexpr int ROW = 128;  // bytes of a block's row

// Where tile t of the walk begins: four m-tiles per group, n advancing across the group
template <int BN, int BM>
__device__ inline void place(const Fp8Gemm& p, int t, int& m0, int& n0) {
    constexpr int GM = 4;
    const int group = t / (GM * p.n_tiles), first_m = group * GM, gm = min(p.m_tiles - first_m, GM);
    const int in_group = t - group * (GM * p.n_tiles);
    m0 = (first_m + in_group % gm) * BM;
    n0 = in_group / gm * BN;
}

// Lane (c = lane % 32, g = lane / 32) of accumulator (i, j): row 32 j + c, features
// 32 i + 8 t + 4 g + e in register 4 t + e.  Pieces of 32 rows go through the wave's
// 4 KiB of LDS so that global memory sees 128 bytes of a row at once (chunk k of
// staged row r at k ^ (r's low bits)).
constexpr int STG = 4096;
template <bool F32, bool BIAS, int NI, int MJ>
__device__ inline void epilogue(const Fp8Gemm& p, const f32x16 (&acc)[NI][MJ], int n_base, int m_base, int lane, uint8_t* stg) {
    constexpr int SZ = F32 ? 4 : 2, EPC = 16 / SZ;   // elements per 16-byte chunk
    constexpr int FW = F32 || NI == 1 ? 1 : 2;       // accumulators side by side in a piece
    constexpr int NC = 2 * FW * SZ, RPI = 64 / NC;   // chunks per staged row, rows per read
    constexpr int STEPS = 32 / RPI;
    auto at = [&](int r, int k) __attribute__((always_inline)) {
        return stg + r * (16 * NC) + ((k ^ (NC == 8 ? (r >> 1) & 7 : (r >> 2) & 3)) << 4);
    };
    const int c = lane & 31, g = lane >> 5;
    const int k = lane % NC, r0 = lane / NC;
    const bool vec = p.c_vec && p.N % EPC == 0;
    // a resource that ends at row M
    const int rows = min(max(p.M - m_base, 0), 32 * MJ);
    const uint32_t row_bytes = (uint32_t)p.ldc * SZ;
    uint8_t* crow = reinterpret_cast<uint8_t*>(p.C) + (int64_t)m_base * p.ldc * SZ;
    const __amdgpu_buffer_rsrc_t cres = uniform_rsrc(crow, (uint32_t)rows * row_bytes);
#pragma unroll
    for (int i0 = 0; i0 < NI; i0 += FW) {
        f32x4 b[FW][4];
        if constexpr (BIAS) {
            const __amdgpu_buffer_rsrc_t bres = uniform_rsrc(p.bias, p.N * 4);
#pragma unroll
            for (int f = 0; f < FW; f++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    b[f][t] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                            bres, 4u * (n_base + 32 * (i0 + f) + 8 * t + 4 * g), 0, 0));
        }
        const int n = n_base + 32 * i0 + k * EPC;
        // an offset past the resource for chunks past N
        const uint32_t ofs0 = n < p.N ? r0 * row_bytes + n * SZ : 0x80000000u;
#pragma unroll
        for (int j = 0; j < MJ; j++) {
#pragma unroll
            for (int f = 0; f < FW; f++) {
                f32x16 x = acc[i0 + f][j];
                asm volatile("" : "+a"(x));  // read here, not all of them ahead of the branches
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    f32x4 v = {x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
                    if constexpr (BIAS) v += b[f][t];
                    if constexpr (F32) {
                        *reinterpret_cast<f32x4*>(at(c, 2 * t + g)) = v;
                    } else {
                        *reinterpret_cast<uint2*>(at(c, 4 * f + t) + 8 * g) =
                            make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
                    }
                }
            }
            u32x4 v[STEPS];
#pragma unroll
            for (int u = 0; u < STEPS; u++) v[u] = *reinterpret_cast<const u32x4*>(at(RPI * u + r0, k));
            if (vec) {
#pragma unroll
                for (int u = 0; u < STEPS; u++)
                    __builtin_amdgcn_raw_buffer_store_b128(v[u], cres, ofs0 + (32 * j + RPI * u) * row_bytes, 0, 0);
            } else {
                // rows at any alignment: whole chunks as they are, the last one of a row in elements
                typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
                uint8_t* to = crow + ((32 * j + r0) * p.ldc + n) * SZ;
                const bool whole = n + EPC <= p.N;
#pragma unroll
                for (int u = 0; u < STEPS; u++, to += RPI * p.ldc * SZ)
                    if (whole && 32 * j + RPI * u + r0 < rows) *reinterpret_cast<u32x4_u*>(to) = v[u];
                if (!whole && n < p.N) {
                    to = crow + ((32 * j + r0) * p.ldc + n) * SZ;
#pragma unroll 1
                    for (int e = 0; e < (p.N - n) * (SZ / 2); e++) {
                        uint16_t h[STEPS];
#pragma unroll
                        for (int u = 0; u < STEPS; u++) h[u] = reinterpret_cast<const uint16_t*>(at(RPI * u + r0, k))[e];
#pragma unroll
                        for (int u = 0; u < STEPS; u++)
                            if (32 * j + RPI * u + r0 < rows) reinterpret_cast<uint16_t*>(to + RPI * u * p.ldc * SZ)[e] = h[u];
                    }
                }
            }
        }
    }
}

// A group of 2 NW waves (NW over n, two over m) makes the tile; KG of them take the blocks of
// K in turn, each with stages of its own, for products of few tiles; their sums meet in LDS at
// the end, in the groups' order.
template <bool EXACT, bool F32, int NI, int MJ, int NS, int KG, int NW>
__global__ __launch_bounds__(128 * NW * KG, 1) void gemm_fp8_kernel(Fp8Gemm p) {
    constexpr int BN = 32 * NW * NI, BM = 64 * MJ;
    constexpr int GW = 2 * NW, GT = 64 * GW;  // waves and threads of a group
    constexpr int PA = 4 * MJ / NW;           // a wave's DMA instructions for A (2 NI for W)
    constexpr int SCALES = (BN + BM) * ROW;
    // a stage's scale words: A's rows', then W's.  Each wave has one instruction for them (so
    // that all wait for one count): 256 rows take one of 16 bytes a lane (waves 0 and 2, W's
    // 1 and 3), fewer one of 4 (a wave for each 64 rows, W's the others).  NW = 1: MJ = 1.
    constexpr int WORD_B = MJ == 4 ? 16 : 4, W_WORDS = MJ == 4 ? 256 : 64 * MJ;
    constexpr int STAGE = SCALES + 4 * W_WORDS + 64 * WORD_B;
    // two-stage forms walk several tiles: the next tile's first stages land during this
    // one's epilogue, which therefore has LDS of its own
    constexpr bool WALK = NS == 2 && KG == 1;
    __shared__ __align__(16) uint8_t lds[KG * NS * STAGE + (WALK ? 4 * STG : 0)];
    static_assert(sizeof(lds) <= 160 * 1024 && 4 * STG + (KG - 1) * NI * MJ * GT * 64 <= (int)sizeof(lds), "LDS");
    const int total = p.n_tiles * p.m_tiles;
    // tiles lid, lid + stride, .. of the XCD's contiguous range up to `end`
    const int per = (total + 7) >> 3, stride = gridDim.x >> 3;
    const int end = min(((int)blockIdx.x & 7) * per + per, total);
    int tile = ((int)blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (tile >= end) return;

    const int tid = threadIdx.x, lane = tid & 63;
    const int kg = __builtin_amdgcn_readfirstlane(tid / GT), wave = __builtin_amdgcn_readfirstlane((tid >> 6) % GW);
    const int wn = wave >> 1, wm = wave & 1;
    const int c = lane & 31, g = lane >> 5;
    const int nk = p.K >> 7, ns = (nk + KG - 1) / KG;  // blocks, and stages of every group
    int ns_wrap = ns;
    asm("" : "+s"(ns_wrap));  // so that no last stage is peeled off the loop for its one comparison
    uint8_t* const ring = lds + kg * (NS * STAGE);

    // DMA: one instruction of a wave fills 8 rows; lane l lands in row l / 8, chunk
    // l % 8, so it fetches the chunk that the swizzle maps there.  Rows past N or M
    // lie past their resource and read zeros.
    const int lrow = lane >> 3;
    int woff[2 * NI], aoff[PA];
#pragma unroll
    for (int i = 0; i < 2 * NI; i++) {
        const int row = (wave * 2 * NI + i) * 8 + lrow;
        woff[i] = row * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < PA; i++) {
        const int row = (wave * PA + i) * 8 + lrow;
        aoff[i] = row * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
    constexpr int NP = 2 * NI + PA + 1;  // DMA instructions of a wave per stage
    const bool w_words = MJ == 4 ? wave & 1 : wave >= MJ;
    const int words0 = MJ == 4 || w_words ? 0 : 64 * wave;  // the first of the wave's words
    const int64_t words_ld = w_words ? p.ld_ws : p.ld_as;
    // the stage fetched next: block f_kt of tile f_tile; past the last block (tile) empty
    // resources, whose loads write zeros without memory traffic
    int f_tile = tile, f_kt = kg;
    __amdgpu_buffer_rsrc_t wres, ares;
    const uint32_t* words;
    uint32_t words_bytes;
    auto fetch_from = [&](int t) __attribute__((always_inline)) {
        int m0 = 0, n0 = 0, wrows = 0, arows = 0;
        if (t < end) {
            place<BN, BM>(p, t, m0, n0);
            wrows = min(BN, p.N - n0);
            arows = min(BM, p.M - m0);
        }
        wres = uniform_rsrc(p.W + (int64_t)n0 * p.K, (uint32_t)wrows * p.K);
        ares = uniform_rsrc(p.A + (int64_t)m0 * p.K, (uint32_t)arows * p.K);
        words = w_words ? p.ws + (n0 >> 7) : p.as + m0;
        words_bytes = 4u * (w_words ? (wrows + 127) >> 7 : arows);
    };
    auto fetch_next = [&]() __attribute__((always_inline)) {
        f_kt += KG;
        if (f_kt >= nk) {
            f_kt = 0;
            f_tile = WALK ? f_tile + stride : end;
            fetch_from(f_tile);
        }
    };
    auto load_piece = [&](int slot, int x) __attribute__((always_inline)) {
        uint8_t* st = ring + slot * STAGE;
        if (x == NP - 1) {
            const __amdgpu_buffer_rsrc_t sres = uniform_rsrc(words + (int64_t)(f_kt >> 2) * words_ld, words_bytes);
            uint8_t* dst = st + SCALES + 4 * (w_words ? W_WORDS : words0);
            if constexpr (WORD_B == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (lptr_t)dst, 16, 16 * lane, 0, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (lptr_t)dst, 4, 4 * (words0 + lane), 0, 0, 0);
            return;
        }
        const bool is_a = x >= 2 * NI;
        const int i = is_a ? x - 2 * NI : x;
        uint8_t* dst = st + (is_a ? BN * ROW + (wave * PA + i) * 1024 : (wave * 2 * NI + i) * 1024);
        const int ofs = is_a ? aoff[i < PA ? i : 0] : woff[i];
        if (is_a) __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lptr_t)dst, 16, ofs, f_kt * ROW, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (lptr_t)dst, 16, ofs, f_kt * ROW, 0, 0);
    };

    f32x16 acc[NI][MJ];
    // fragment rows: blocks of 32 rows are 4 KiB apart and have the same swizzle
    const int wrow = (wn * 32 * NI + c) * ROW, arow = BN * ROW + (wm * 32 * MJ + c) * ROW, sx = (c >> 1) & 7;
    // EXACT widens a fragment before the next half's is read into its registers
    constexpr int BUFS = EXACT ? 1 : 2;
    i32x8 wf[BUFS][NI], af[BUFS][MJ];
    int sw, sa[MJ], sw_next = 0, sa_next[MJ];
    // piece x of the fragments of half s of a stage (into buffer buf): two chunks of a row each
    auto read_piece = [&](int slot, int s, int buf, int x) __attribute__((always_inline)) {
        const int f = x >> 1, h = x & 1, at = ((4 * s + 2 * g + h) ^ sx) << 4;
        const uint8_t* from = ring + slot * STAGE + at + (f < NI ? wrow + 32 * ROW * f : arow + 32 * ROW * (f - NI));
        const i32x4 v = *reinterpret_cast<const i32x4*>(from);
        i32x8& d = f < NI ? wf[buf][f < NI ? f : 0] : af[buf][f < NI ? 0 : f - NI];
#pragma unroll
        for (int e = 0; e < 4; e++) d[4 * h + e] = v[e];
    };
    constexpr int NR = 2 * (NI + MJ);
    auto read_scales = [&](int slot) __attribute__((always_inline)) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(ring + slot * STAGE + SCALES);
#pragma unroll
        for (int j = 0; j < MJ; j++) sa_next[j] = (int)w[wm * 32 * MJ + 32 * j + c];
        sw_next = (int)w[W_WORDS + ((wn * 32 * NI) >> 7)];
    };
    auto take_scales = [&](int st) __attribute__((always_inline)) {  // the group's stage st: byte kt % 4 of the words
        const int sh = 8 * ((st * KG + kg) & 3);
        sw = __builtin_amdgcn_readfirstlane(sw_next) >> sh;
#pragma unroll
        for (int j = 0; j < MJ; j++) sa[j] = sa_next[j] >> sh;
    };
    // One half block (of: 0 or 1 of its stage); between its instructions, when `read`, the
    // reads of the next half (slot rslot, half rs) and pieces d0 .. d1 - 1 of the next
    // stage's DMA into slot dma_slot, spread evenly: an instruction of 64 cycles hides one
    // read and one piece, not two (5498 x 13824 x 2560 188 us with them in the first eight
    // of sixteen, 175 so).
    auto half = [&](int of, int rslot, int rs, bool read, int d0, int d1, int dma_slot, bool zc) __attribute__((always_inline)) {
        const int buf = of % BUFS, rbuf = (of + 1) % BUFS;
        // EXACT: fragments widen while the instructions before their first use run (all of
        // them ahead of the half: 5498 x 13824 x 2560 375 us, so 358)
        bf16x8 wb[2][4], ab[MJ][4];
        auto widen_w = [&](int i) __attribute__((always_inline)) {
            const float f = scale_of(sw & 0xff);
#pragma unroll
            for (int e = 0; e < 4; e++) wb[i & 1][e] = widen(wf[buf][i][2 * e], wf[buf][i][2 * e + 1], f);
        };
        auto widen_a = [&](int j) __attribute__((always_inline)) {
            const float f = scale_of(sa[j] & 0xff);
#pragma unroll
            for (int e = 0; e < 4; e++) ab[j][e] = widen(af[buf][j][2 * e], af[buf][j][2 * e + 1], f);
        };
        if constexpr (EXACT) {
            widen_w(0);
            widen_a(0);
        }
        constexpr int T = NI * MJ;
#pragma unroll
        for (int x = 0; x < T; x++) {
            const int i = x / MJ, j = x % MJ;
            f32x16 z;
#pragma unroll
            for (int e = 0; e < 16; e++) z[e] = 0.f;
            if constexpr (EXACT) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i & 1][0], ab[j][0], zc ? z : acc[i][j], 0, 0, 0);
#pragma unroll
                for (int e = 1; e < 4; e++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i & 1][e], ab[j][e], acc[i][j], 0, 0, 0);
                if (i == 0 && j + 1 < MJ) widen_a(j + 1);
                if (j + 1 == MJ && i + 1 < NI) widen_w(i + 1);
            } else {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[buf][i], af[buf][j], zc ? z : acc[i][j], 0, 0, 0,
                                                                           sw, 0, sa[j]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < NR; e++) {
                // EXACT: W's first fragment, A's, W's others, as they fall free
                const int k = e >> 1, f = !EXACT ? k : k == 0 ? 0 : k <= MJ ? NI + k - 1 : k - MJ;
                if (read && e * T / NR == x) read_piece(rslot, rs, rbuf, 2 * f + (e & 1));
            }
#pragma unroll
            for (int e = d0; e < d1; e++)
                if ((e - d0) * T / (d1 - d0) == x) load_piece(dma_slot, e);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // A stream of stages, tile after tile: while one is computed from slot `slot`, the
    // NS - 1 after it land in the others.  Half 0 reads half 1's fragments from the same
    // slot; then every wave waits for its own DMA of the next stage and for its LDS
    // reads, and the barrier makes that stage visible and this slot free: half 1 reads
    // the next stage's first fragments and refills this slot with the stage NS on.
    int slot = 0;
    auto next = [](int t) __attribute__((always_inline)) { return t + 1 == NS ? 0 : t + 1; };
    // With three stages or more the refill goes on through half 0 of the next stage (`more`:
    // there is one to go on with), an even stream in place of a burst that the pieces of four
    // waves queue up in (679 x 2560 x 6912 in 128 x 128 tiles 27.1 -> 23.5 us).
    constexpr int NP1 = NS > 2 ? NP / 2 : NP;
    // The sums stay where they are formed: the compiler would move the instructions whose
    // results no one reads yet past the branch of fetch_next, behind all the loads between.
    auto pin = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < NI * MJ; x++) asm volatile("" : "+a"(acc[x / MJ][x % MJ]));
    };
    auto stage = [&](int st, bool zc, bool more) __attribute__((always_inline)) {
        const int before = slot == 0 ? NS - 1 : slot - 1;
        half(0, slot, 1, true, more ? NP1 : NP, NP, before, zc);
        if (more && NP1 < NP) {
            pin();
            fetch_next();
        }
        wait_vmem_lds<(NS - 2) * NP>();
        __builtin_amdgcn_s_barrier();
        read_scales(next(slot));
        half(1, next(slot), 0, true, 0, NP1, slot, false);
        pin();
        if (NP1 == NP) fetch_next();
        take_scales(st + 1 == ns_wrap ? 0 : st + 1);
        slot = next(slot);
    };
    fetch_from(kg < nk ? tile : end);
#pragma unroll
    for (int i = 0; i < NS; i++) {
#pragma unroll
        for (int x = 0; x < NP; x++) load_piece(i, x);
        fetch_next();
    }
    wait_vmem_lds<(NS - 1) * NP>();
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int x = 0; x < NR; x++) read_piece(0, 0, 0, x);
    read_scales(0);
    take_scales(0);
    while (true) {
        int m0, n0;
        if constexpr (WALK) {
            stage(0, true, false);
            for (int st = 1; st < ns; st++) stage(st, false, false);
        } else {
            // no stage follows the last one, which only reads its own second half
            if (ns > 1) {
                stage(0, true, false);
                for (int st = 1; st + 1 < ns; st++) stage(st, false, NS > 2);
                half(0, slot, 1, true, NP, NP, 0, false);
            } else {
                half(0, slot, 1, true, NP, NP, 0, true);
            }
            half(1, slot, 0, false, NP, NP, 0, false);
        }
        place<BN, BM>(p, tile, m0, n0);
        if constexpr (!WALK) {  // the slots are free once every DMA (of nothing, by now) and read is done
            wait_vmem_lds<0>();
            __builtin_amdgcn_s_barrier();
        }
        if constexpr (KG > 1) {
            // the other groups' sums to group 0, past its staging area
            f32x4* sums = reinterpret_cast<f32x4*>(lds + 4 * STG) + tid % GT;
            auto at = [&](int from, int x, int q) __attribute__((always_inline)) {
                return sums + GT * ((from * NI * MJ + x) * 4 + q);
            };
            if (kg) {
#pragma unroll
                for (int x = 0; x < NI * MJ; x++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f32x16& v = acc[x / MJ][x % MJ];
                        *at(kg - 1, x, q) = (f32x4){v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                    }
            }
            __syncthreads();
            if (kg) return;
#pragma unroll
            for (int o = 0; o < KG - 1; o++)
#pragma unroll
                for (int x = 0; x < NI * MJ; x++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const f32x4 v = *at(o, x, q);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[x / MJ][x % MJ][4 * q + e] += v[e];
                    }
        }
        uint8_t* stg = lds + (WALK ? NS * STAGE : 0) + wave * STG;
        // the lane anew, so that the epilogue's addresses are formed here: hoisted, they
        // would cost the stages registers
        int l = 0;
        asm volatile("" : "+v"(l));
        l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, l));
        if (p.bias) epilogue<F32, true, NI, MJ>(p, acc, n0 + wn * 32 * NI, m0 + wm * 32 * MJ, l, stg);
        else epilogue<F32, false, NI, MJ>(p, acc, n0 + wn * 32 * NI, m0 + wm * 32 * MJ, l, stg);
        tile += stride;
        if (!WALK || tile >= end) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives its LDS
}

// The same for accumulators of 16 x 16: lane (c = lane % 16, q = lane / 16) of (i, j) holds row
// 16 j + c (of the other 64 rows, where kind is 1), features 16 i + 4 q + e.
template <bool BIAS>
__device__ inline void wide_epilogue(const Fp8Gemm& p, const f32x4 (&acc)[8][8], int n_base, int m_base, int kind, int lane,
                                     uint8_t* stg) {
    constexpr int SZ = 2, EPC = 8, RPI = 8, STEPS = 4;
    auto at = [&](int r, int k) __attribute__((always_inline)) { return stg + r * 128 + ((k ^ ((r >> 1) & 7)) << 4); };
    const int c = lane & 15, q = lane >> 4, k = lane & 7, r0 = lane >> 3;
    const bool vec = p.c_vec && p.N % EPC == 0;
    const int rows = min(max(p.M - m_base, 0), 128);
    const uint32_t row_bytes = (uint32_t)p.ldc * SZ;
    uint8_t* crow = reinterpret_cast<uint8_t*>(p.C) + (int64_t)m_base * p.ldc * SZ;
    const __amdgpu_buffer_rsrc_t cres = uniform_rsrc(crow, (uint32_t)rows * row_bytes);
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += 4) {
        f32x4 b[4];
        if constexpr (BIAS) {
            const __amdgpu_buffer_rsrc_t bres = uniform_rsrc(p.bias, p.N * 4);
#pragma unroll
            for (int i = 0; i < 4; i++)
                b[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bres, 4u * (n_base + 16 * (i0 + i) + 4 * q), 0, 0));
        }
        const int n = n_base + 16 * i0 + k * EPC;
        const uint32_t ofs0 = n < p.N ? r0 * row_bytes + n * SZ : 0x80000000u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int rj = 32 * (j ^ 2 * kind);
#pragma unroll
            for (int jj = 0; jj < 2; jj++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    f32x4 v = acc[i0 + i][2 * j + jj];
                    asm volatile("" : "+a"(v));
                    if constexpr (BIAS) v += b[i];
                    *reinterpret_cast<uint2*>(at(16 * jj + c, 2 * i + (q >> 1)) + 8 * (q & 1)) =
                        make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
                }
            u32x4 v[STEPS];
#pragma unroll
            for (int u = 0; u < STEPS; u++) v[u] = *reinterpret_cast<const u32x4*>(at(RPI * u + r0, k));
            if (vec) {
#pragma unroll
                for (int u = 0; u < STEPS; u++)
                    __builtin_amdgcn_raw_buffer_store_b128(v[u], cres, ofs0 + (rj + RPI * u) * row_bytes, 0, 0);
            } else {
                typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
                uint8_t* to = crow + ((rj + r0) * p.ldc + n) * SZ;
                const bool whole = n + EPC <= p.N;
#pragma unroll
                for (int u = 0; u < STEPS; u++, to += RPI * p.ldc * SZ)
                    if (whole && rj + RPI * u + r0 < rows) *reinterpret_cast<u32x4_u*>(to) = v[u];
                if (!whole && n < p.N) {
                    to = crow + ((rj + r0) * p.ldc + n) * SZ;
#pragma unroll 1
                    for (int e = 0; e < p.N - n; e++) {
                        uint16_t h[STEPS];
#pragma unroll
                        for (int u = 0; u < STEPS; u++) h[u] = reinterpret_cast<const uint16_t*>(at(RPI * u + r0, k))[e];
#pragma unroll
                        for (int u = 0; u < STEPS; u++)
                            if (rj + RPI * u + r0 < rows) reinterpret_cast<uint16_t*>(to + RPI * u * p.ldc * SZ)[e] = h[u];
                    }
                }
            }
        }
    }
}

// ---- the largest tiles --------------------------------------------------------
//
// 256 x 256 for bf16 C, a wave 128 x 128 in accumulators of 16 x 16 (one
// v_mfma_scale_f32_16x16x128_f8f6f4 a block of K), which draw a little less power than
// those of 32 x 32.  A stage is four quarters of its 64 instructions: with W's blocks in
// two halves w0, w1 and A's in f (first) and s,
//   w0 f   reads s            of this stage      DMA of w0, f of the stage after next
//   w0 s   reads w1           of this stage
//   w1 s   reads w0           of the next stage  DMA of s, w1 of the stage after next
//   w1 f   reads the next f   of the next stage
// Each fragment is read into registers whose last use is over (the next stage's f is
// this one's s: they change places from stage to stage), and each half of a slot is
// refilled as soon as every wave has read it: two barriers a stage, fragment reads and
// DMA even over all of it, and a whole stage for a refill to land, with two stages of
// LDS.  5498 x 13824 x 2560 takes 151 to 161 us (2.4 to 2.6 PFLOP/s; tiles as above 5 more), 8192^3
// 350 to 366 (3.0 to 3.1; 374), the matrix cores busy for 60 % of the cycles.  Bound by power: the
// first stages of a tile without a wait for the stores of the tile before, and LDS reads
// without bank conflicts, changed neither.
__global__ __launch_bounds__(256, 1) void gemm_fp8_wide_kernel(Fp8Gemm p) {
    constexpr int BN = 256, BM = 256;
    constexpr int SCALES = (BN + BM) * ROW, W_WORDS = 256, STAGE = SCALES + 2048;  // words of A's rows, then W's
    __shared__ __align__(16) uint8_t lds[2 * STAGE + 4 * STG];
    const int total = p.n_tiles * p.m_tiles;
    // tiles lid, lid + stride, .. of the XCD's contiguous range up to `end`
    const int per = (total + 7) >> 3, stride = gridDim.x >> 3;
    const int end = min(((int)blockIdx.x & 7) * per + per, total);
    int tile = ((int)blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (tile >= end) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave >> 1, wm = wave & 1;
    const int nk = p.K >> 7;
    int nk_wrap = nk;
    asm("" : "+s"(nk_wrap));

    // DMA as in the other tiles.  A half of an operand is rows 0 .. 63 and 128 .. 191 of the
    // tile, or 64 more: a wave's four pieces of a half are 32 neighbouring rows.
    const int row0 = (wave >> 1) * 128 + (wave & 1) * 32, lrow = lane >> 3;
    int off[2], k16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int row = row0 + 8 * i + lrow;
        off[i] = row * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
    const bool w_words = wave & 1;  // waves 0 and 2 fetch A's words, 1 and 3 W's
    const int64_t words_ld = w_words ? p.ld_ws : p.ld_as;
    int f_tile = tile, f_kt = 0;
    __amdgpu_buffer_rsrc_t wres, ares;
    const uint32_t* words;
    uint32_t words_bytes;
    auto fetch_from = [&](int t) __attribute__((always_inline)) {
        int m0 = 0, n0 = 0, wrows = 0, arows = 0;
        if (t < end) {
            place<BN, BM>(p, t, m0, n0);
            wrows = min(BN, p.N - n0);
            arows = min(BM, p.M - m0);
        }
        wres = uniform_rsrc(p.W + (int64_t)n0 * p.K, (uint32_t)wrows * p.K);
        ares = uniform_rsrc(p.A + (int64_t)m0 * p.K, (uint32_t)arows * p.K);
        words = w_words ? p.ws + (n0 >> 7) : p.as + m0;
        words_bytes = 4u * (w_words ? (wrows + 127) >> 7 : arows);
    };
    auto fetch_next = [&]() __attribute__((always_inline)) {
        if (++f_kt == nk) {
            f_kt = 0;
            f_tile += stride;
            fetch_from(f_tile);
        }
    };
    // A tile's first stage begins with A's rows of half `kind`: it goes on from the tile before.
    int kind = 0;
    // piece x (of four) of a half of W or A (A's half of this kind), or (x = 4) the words
    auto load_piece = [&](int slot, bool is_a, int half, int x) __attribute__((always_inline)) {
        uint8_t* st = lds + slot * STAGE;
        if (x == 4) {
            const __amdgpu_buffer_rsrc_t sres = uniform_rsrc(words + (int64_t)(f_kt >> 2) * words_ld, words_bytes);
            uint8_t* dst = st + SCALES + 4 * (w_words ? W_WORDS : 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (lptr_t)dst, 16, 16 * lane, 0, 0, 0);
            return;
        }
        const int h = is_a ? half ^ kind : half;
        uint8_t* dst = st + ((is_a ? BN : 0) + row0 + 64 * h + 8 * x) * ROW;
        const int ofs = off[x & 1] + (4 * h + (x >> 1)) * k16;
        if (is_a) __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lptr_t)dst, 16, ofs, f_kt * ROW, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (lptr_t)dst, 16, ofs, f_kt * ROW, 0, 0);
    };
    constexpr int G1 = 9, G2 = 8;  // DMA instructions with the first two quarters and the others

    f32x4 acc[8][8];
    const int c = lane & 15, q = lane >> 4;
    // Fragment rows: blocks of 16 rows are 2 KiB apart and have the same swizzle.  A lane takes
    // chunks q and q + 4, which keeps the lanes of one LDS pass on different banks.
    const int wrow = (wn * 128 + c) * ROW, arow = BN * ROW + (wm * 128 + c) * ROW, sx = (c >> 1) & 7;
    const int at0 = (q ^ sx) << 4, at1 = ((q + 4) ^ sx) << 4, arow_words = 4 * (wm * 128 + c);
    i32x8 wf[8], af[8];
    int sw, sa[8], sw_next = 0, sa_next[8];
    // piece x (of eight) of the four fragments of a half
    auto read_piece = [&](int slot, bool is_a, int half, int x) __attribute__((always_inline)) {
        const int f = 4 * half + (x >> 1), h = x & 1;
        const uint8_t* from = lds + slot * STAGE + (is_a ? 64 * ROW * (half ^ kind) : 64 * ROW * half);
        const i32x4 v = *reinterpret_cast<const i32x4*>(from + (h ? at1 : at0) + (is_a ? arow : wrow) + 16 * ROW * (x >> 1));
        i32x8& d = is_a ? af[f] : wf[f];
#pragma unroll
        for (int e = 0; e < 4; e++) d[4 * h + e] = v[e];
    };
    auto read_scales = [&](int slot, int kind) __attribute__((always_inline)) {
        const uint8_t* w = lds + slot * STAGE + SCALES;
#pragma unroll
        for (int j = 0; j < 8; j++)
            sa_next[j] = *reinterpret_cast<const int*>(w + arow_words + 256 * ((j >> 2) ^ kind) + 64 * (j & 3));
        sw_next = *reinterpret_cast<const int*>(w + 4 * (W_WORDS + wn));
    };
    auto take_scales = [&](int kt) __attribute__((always_inline)) {  // byte kt % 4 of the words
        const int sh = 8 * (kt & 3);
        sw = __builtin_amdgcn_readfirstlane(sw_next) >> sh;
#pragma unroll
        for (int j = 0; j < 8; j++) sa[j] = sa_next[j] >> sh;
    };
    // W's half wi with A's half aj; a read of (rslot, W or A, half rh) after every other
    // instruction, and after the odd ones, evenly, the DMA of up to two operands' halves
    auto quarter = [&](int wi, int aj, int rslot, bool rd_a, int rh, int slot, bool dma_a, int dh, int nd, bool zc)
        __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < 16; x++) {
            const int i = 4 * wi + (x >> 2), j = 4 * aj + (x & 3);
            const f32x4 z = {0.f, 0.f, 0.f, 0.f};
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[i], af[j], zc ? z : acc[i][j], 0, 0, 0, sw, 0, sa[j]);
            __builtin_amdgcn_sched_barrier(0);
            if (!(x & 1)) read_piece(rslot, rd_a, rh, x >> 1);
#pragma unroll
            for (int e = 0; e < nd; e++)
                if (e * 16 / nd + 1 == x) load_piece(slot, dma_a, dh, e);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int slot = 0;
    auto stage = [&](int kt, bool odd, bool zc) __attribute__((always_inline)) {
        const int f = odd ? 1 : 0, s = 1 - f;
        k16 = 16 * p.K;
        asm volatile("" : "+s"(k16));  // the pieces' offsets are formed at the pieces: hoisted, they would take 16 registers
        // Every wave's DMA of this stage's s and w1 has landed, and its w0, f and words are read.
        wait_vmem_lds<G1 + G2>();
        __builtin_amdgcn_s_barrier();
        quarter(0, f, slot, true, s, slot, false, 0, 5, zc);
        quarter(0, s, slot, false, 1, slot, true, f, 4, zc);
        // The next stage's w0, f and words have landed, and this one's s and w1 are read.
        wait_vmem_lds<G1 + G2>();
        __builtin_amdgcn_s_barrier();
        read_scales(slot ^ 1, kt + 1 == nk_wrap ? kind ^ (nk_wrap & 1) : kind);
        quarter(1, s, slot ^ 1, false, 0, slot, true, s, 4, zc);
        quarter(1, f, slot ^ 1, true, s, slot, false, 1, 4, zc);
        // (the sums stay where they are formed, as in the other tiles)
#pragma unroll
        for (int x = 0; x < 64; x++) asm volatile("" : "+a"(acc[x >> 3][x & 7]));
        fetch_next();
        take_scales(kt + 1 == nk_wrap ? 0 : kt + 1);
        slot ^= 1;
    };
    fetch_from(tile);
    k16 = 16 * p.K;
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int x = 0; x < 5; x++) load_piece(i, false, 0, x);
#pragma unroll
        for (int x = 0; x < 4; x++) load_piece(i, true, i, x);  // the first half of A of its kind of stage
#pragma unroll
        for (int x = 0; x < 4; x++) load_piece(i, true, 1 - i, x);
#pragma unroll
        for (int x = 0; x < 4; x++) load_piece(i, false, 1, x);
        fetch_next();
    }
    wait_vmem_lds<G2 + G1 + G2>();
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int x = 0; x < 8; x++) read_piece(0, false, 0, x);
#pragma unroll
    for (int x = 0; x < 8; x++) read_piece(0, true, 0, x);
    read_scales(0, 0);
    take_scales(0);
    while (true) {
        stage(0, false, true);
        int kt = 1;
        for (; kt + 1 < nk; kt += 2) {
            stage(kt, true, false);
            stage(kt + 1, false, false);
        }
        if (kt < nk) {
            stage(kt, true, false);
        } else {  // the next tile's first fragments of A are in s's registers
#pragma unroll
            for (int i = 0; i < 4; i++) af[i] = af[4 + i];
        }
        int m0, n0;
        place<BN, BM>(p, tile, m0, n0);
        int l = 0;  // the lane anew: see the other tiles
        asm volatile("" : "+v"(l));
        l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, l));
        uint8_t* stg = lds + 2 * STAGE + wave * STG;
        if (p.bias) wide_epilogue<true>(p, acc, n0 + wn * 128, m0 + wm * 128, kind, l, stg);
        else wide_epilogue<false>(p, acc, n0 + wn * 128, m0 + wm * 128, kind, l, stg);
        kind ^= nk & 1;
        tile += stride;
        if (tile >= end) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives its LDS
}

// The tile forms.  The large ones have the fewest operand bytes per product, the small
// ones the most workgroups, and those with groups of waves over K the most of a
// workgroup's blocks in flight: what bounds few tiles is how many bytes are on their way
// (58 x 2560 x 6912 in 64 x 64 tiles, 40 workgroups, 11.7 us; in 32 x 64, 80 of them, 9.4;
// fp32 C 17.3 and 11.6).
struct Tile {
    int ni, mj, ns, kg, nw;
    // measured, us: a block of K with one tile at work and with every CU busy, and a tile's ends
    float alone, full, ends;
};
constexpr Tile FAST[] = {{4, 4, 2, 1, 2, 1.05f, 1.30f, 6.0f}, {4, 3, 2, 1, 2, 0.95f, 0.97f, 5.5f},
                         {2, 3, 3, 1, 2, 0.42f, 0.66f, 4.3f}, {2, 2, 4, 1, 2, 0.30f, 0.42f, 4.2f},
                         {2, 1, 3, 2, 2, 0.19f, 0.29f, 4.0f}, {1, 1, 4, 2, 2, 0.13f, 0.20f, 3.9f},
                         {1, 1, 3, 4, 1, 0.105f, 0.125f, 3.7f}};
constexpr Tile FULL[] = {{4, 4, 2, 1, 2, 2.16f, 2.50f, 9.0f}, {4, 3, 2, 1, 2, 1.69f, 1.92f, 6.5f},
                         {4, 2, 2, 1, 2, 1.26f, 1.47f, 6.0f}, {2, 2, 2, 2, 2, 0.62f, 0.76f, 6.3f},
                         {2, 1, 3, 2, 2, 0.39f, 0.48f, 5.7f}, {1, 1, 2, 4, 2, 0.23f, 0.30f, 5.0f},
                         {1, 1, 3, 4, 1, 0.13f, 0.165f, 4.3f}};

// Estimated time with tiles t: rounds of one tile per CU, the last one at 0.7 of a full
// round plus 0.3 of its share (as for the bf16 GEMM).  All seven forms were timed on 38
// products of 17 to 5498 rows with either C, and with bf16 C of whole products: it takes the
// fastest of each but one, there a form 2 % behind it (512 x 512 x 512, bf16 C: 4.3 us, 4.2).
float tile_cost(const Fp8Gemm& p, const Tile& t, int cus) {
    const long tiles = ((long)p.N + 32 * t.nw * t.ni - 1) / (32 * t.nw * t.ni) * (((long)p.M + 64 * t.mj - 1) / (64 * t.mj));
    const float r = (float)tiles / cus, share = r < 1.f ? r : 1.f;
    const float rounds = r <= 1.f ? 1.f : 0.7f * (float)(long)(r + 0.9999f) + 0.3f * r;
    return rounds * ((t.alone + (t.full - t.alone) * share) * (float)(p.K / 128) + t.ends);
}

template <int NI, int WAVES>
void few_launch(const Fp8Gemm& p, hipStream_t s) {
    hipLaunchKernelGGL((gemm_fp8_few_kernel<NI, WAVES>), dim3((p.N + 16 * NI - 1) / (16 * NI)), dim3(64 * WAVES), 0, s, p);
}

}  // namespace

hipError_t launch_gemm_fp8(Fp8Gemm& p, hipStream_t s) {
    const int cus = device_cus();
    if (p.M <= 16) {
        // 16, 32 or 64 features a workgroup, by what the busiest CU fetches: its features, and for
        // each of its workgroups A, as much as 4 + 3/4 M features (1 row: 4096 x 11008 10.0 us with
        // 16, 14.4 with 32; 8000 x 5120 9.2 with 32 and 16; 24000 x 2560 12.5, 11.8 and 14.0; 16
        // rows of 13824 x 2560 12.4, 10.3 and 9.3; of nine products it takes the fastest, or one 2 %
        // behind it, but 14.7 us for 12.7 at 4 x 16000 x 4096)
        auto fetched = [&](int ni) { return ((p.N + 16 * ni - 1) / (16 * ni) + cus - 1) / cus * (64 * ni + 16 + 3 * p.M); };
        const int f1 = fetched(1), f2 = fetched(2), f4 = fetched(4);
        if (f4 < f1 && f4 < f2) few_launch<4, 4>(p, s);
        else if (f2 < f1) few_launch<2, 4>(p, s);
        else few_launch<1, 8>(p, s);
        return hipGetLastError();
    }
    const bool exact = p.c_f32 || p.whole;
    const Tile* t = exact ? FULL : FAST;
    const Tile* end = exact ? FULL + sizeof(FULL) / sizeof(Tile) : FAST + sizeof(FAST) / sizeof(Tile);
    for (const Tile* x = t + 1; x < end; x++)
        if (tile_cost(p, *x, cus) < tile_cost(p, *t, cus)) t = x;
    p.n_tiles = (p.N + 32 * t->nw * t->ni - 1) / (32 * t->nw * t->ni);
    p.m_tiles = (p.M + 64 * t->mj - 1) / (64 * t->mj);
    // two-stage forms: a workgroup per CU walks its tiles
    const long tiles = (long)p.n_tiles * p.m_tiles;
    const dim3 grid(xcd_grid(t->ns == 2 && t->kg == 1 && tiles > cus ? cus : tiles)), block(128 * t->nw * t->kg);
#define TILE(E, F, NI, MJ, NS, KG, NW)                                                               \
    if (exact == E && p.c_f32 == F && t->ni == NI && t->mj == MJ && t->ns == NS && t->kg == KG && t->nw == NW) { \
        hipLaunchKernelGGL((gemm_fp8_kernel<E, F, NI, MJ, NS, KG, NW>), grid, block, 0, s, p);         \
        return hipGetLastError();                                                                    \
    }
#define FULL_TILE(NI, MJ, NS, KG, NW) TILE(1, 1, NI, MJ, NS, KG, NW) TILE(1, 0, NI, MJ, NS, KG, NW)
    if (!exact && t->ni == 4 && t->mj == 4) {
        hipLaunchKernelGGL(gemm_fp8_wide_kernel, grid, block, 0, s, p);
        return hipGetLastError();
    }
    TILE(0, 0, 4, 3, 2, 1, 2)
    TILE(0, 0, 2, 3, 3, 1, 2)
    TILE(0, 0, 2, 2, 4, 1, 2)
    TILE(0, 0, 2, 1, 3, 2, 2)
    TILE(0, 0, 1, 1, 4, 2, 2)
    TILE(0, 0, 1, 1, 3, 4, 1)
    FULL_TILE(4, 4, 2, 1, 2)
    FULL_TILE(4, 3, 2, 1, 2)
    FULL_TILE(4, 2, 2, 1, 2)
    FULL_TILE(2, 2, 2, 2, 2)
    FULL_TILE(2, 1, 3, 2, 2)
    FULL_TILE(1, 1, 2, 4, 2)
    FULL_TILE(1, 1, 3, 4, 1)
#undef FULL_TILE
#undef TILE
    return hipErrorInvalidValue;
}

}  // namespace awa
