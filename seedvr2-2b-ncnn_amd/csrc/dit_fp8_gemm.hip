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
// 16 features x 16 MJ rows per workgroup, the blocks of K in turn over its waves,
// whose sums meet in LDS (in the waves' order).  Bound by W, which is read once,
// straight into registers; nothing is shared that LDS could hold for others.
template <int MJ, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void gemm_fp8_few_kernel(Fp8Gemm p) {
    __shared__ f32x4 part[WAVES][MJ][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = (blockIdx.x % p.n_tiles) * 16, m0 = (blockIdx.x / p.n_tiles) * (16 * MJ);
    // rows past the end repeat the last
    const uint8_t* wp = p.W + (int64_t)min(n0 + r, p.N - 1) * p.K + 16 * q;
    const uint8_t* wsp = reinterpret_cast<const uint8_t*>(p.ws + (n0 >> 7));
    const uint8_t* ap[MJ];
    const uint8_t* asp[MJ];
#pragma unroll
    for (int j = 0; j < MJ; j++) {
        const int row = min(m0 + 16 * j + r, p.M - 1);
        ap[j] = p.A + (int64_t)row * p.K + 16 * q;
        asp[j] = reinterpret_cast<const uint8_t*>(p.as + row);
    }
    const int nk = p.K >> 7;
    struct Block {
        i32x4 w[2], a[MJ][2];
        int sw, sa[MJ];
    };
    auto load = [&](Block& b, int kb) __attribute__((always_inline)) {
        const int64_t g = kb >> 2;
#pragma unroll
        for (int h = 0; h < 2; h++) b.w[h] = *reinterpret_cast<const i32x4*>(wp + kb * 128 + 64 * h);
        b.sw = wsp[4 * g * p.ld_ws + (kb & 3)];
#pragma unroll
        for (int j = 0; j < MJ; j++) {
#pragma unroll
            for (int h = 0; h < 2; h++) b.a[j][h] = *reinterpret_cast<const i32x4*>(ap[j] + kb * 128 + 64 * h);
            b.sa[j] = asp[j][4 * g * p.ld_as + (kb & 3)];
        }
    };
    f32x4 acc[MJ];
#pragma unroll
    for (int j = 0; j < MJ; j++) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto sum = [&](const Block& b) __attribute__((always_inline)) {
        const float sw = scale_of(b.sw);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bf16x8 w0 = widen(b.w[h][0], b.w[h][1], sw), w1 = widen(b.w[h][2], b.w[h][3], sw);
#pragma unroll
            for (int j = 0; j < MJ; j++) {
                const float sa = scale_of(b.sa[j]);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, widen(b.a[j][h][0], b.a[j][h][1], sa), acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, widen(b.a[j][h][2], b.a[j][h][3], sa), acc[j], 0, 0, 0);
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
    for (int j = 0; j < MJ; j++) part[wave][j][lane] = acc[j];
    __syncthreads();
    // wave j finishes row block j
    for (int j = wave; j < MJ; j += WAVES) {
        f32x4 c = part[0][j][lane];
#pragma unroll
        for (int w = 1; w < WAVES; w++) c += part[w][j][lane];
        const int m = m0 + 16 * j + r, n = n0 + 4 * q;
        if (m >= p.M) continue;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n + i < p.N) {
                const float v = c[i] + (p.bias ? p.bias[n + i] : 0.f);
                if (p.c_f32) reinterpret_cast<float*>(p.C)[m * p.ldc + n + i] = v;
                else reinterpret_cast<uint16_t*>(p.C)[m * p.ldc + n + i] = (uint16_t)bf16x2_rne(v, v);
            }
    }
}

// ---- tiles ------------------------------------------------------------------
//
// Workgroup tile 64 NI (n) x 64 MJ (m), a block of K per stage, four wave64 in a
// 2 x 2 grid, NI x MJ accumulators of 32 x 32 per wave.  As in the bf16 GEMM the
// operands' 128-byte rows reach LDS by direct DMA into NS stages, 16-byte chunks at
// chunk ^ ((row >> 1) & 7), and each half block (64 columns, one instruction per
// accumulator) runs with the next half's fragment reads and, in the half that
// refills the freed stage, the DMA pieces between its instructions.  A row's scale
// word travels with its stage (256 bytes per 64 rows beside 8 KiB of them); W's is
// the same for a whole wave and comes by scalar loads.
//
// EXACT (fp32 C): the fragments are widened to bf16 with their scales and take four
// 32x32x16 bf16 instructions in place of one 8-bit one.
constexpr int ROW = 128;  // bytes of a block's row
__device__ inline int swz(int row, int chunk) { return row * ROW + ((chunk ^ ((row >> 1) & 7)) << 4); }

// A buffer resource with wave-uniform fields (as in dit_gemm.hip): loads past
// `bytes` read zeros and stores past it are dropped.
__device__ inline __amdgpu_buffer_rsrc_t uniform_rsrc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
// Waits until at most N vector memory operations and no LDS operation are outstanding.
template <int N>
__device__ inline void wait_vmem_lds() {
    asm volatile("s_waitcnt vmcnt(%c0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// A word that no kernel writes while this one runs, at a wave-uniform address.
__device__ inline uint32_t uniform_word(const uint32_t* p) {
    return *(const __attribute__((address_space(4))) uint32_t*)reinterpret_cast<uint64_t>(p);
}

// Lane (c = lane % 32, g = lane / 32) of accumulator (i, j): row 32 j + c, features
// 32 i + 8 t + 4 g + e in register 4 t + e.  Through LDS, so that global memory sees
// whole rows: chunk k of staged row r at k ^ (r's low bits).
template <bool F32, int NI, int MJ>
__device__ inline void epilogue(const Fp8Gemm& p, f32x16 (&acc)[NI][MJ], int n_base, int m_base, int lane, uint8_t* stg) {
    constexpr int SZ = F32 ? 4 : 2, NC = 2 * NI * SZ, RPI = 64 / NC;  // 16-byte chunks per row, rows per read
    constexpr int EPC = 16 / SZ;                                     // elements per chunk
    auto swc = [](int r, int k) __attribute__((always_inline)) {
        return k ^ (NC >= 16 ? r & (NC - 1) : NC == 8 ? (r >> 1) & 7 : (r >> 2) & 3);
    };
    const int c = lane & 31, g = lane >> 5;
    const __amdgpu_buffer_rsrc_t bres = uniform_rsrc(p.bias, p.bias ? p.N * 4 : 0);
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const u32x4 b = __builtin_amdgcn_raw_buffer_load_b128(bres, 4u * (n_base + 32 * i + 8 * t + 4 * g), 0, 0);
#pragma unroll
            for (int j = 0; j < MJ; j++) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[i][j][4 * t + e] + __uint_as_float(b[e]);
                const int r = 32 * j + c;
                if constexpr (F32) {
                    *reinterpret_cast<float4*>(stg + r * (16 * NC) + (swc(r, 8 * i + 2 * t + g) << 4)) =
                        make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    *reinterpret_cast<uint2*>(stg + r * (16 * NC) + (swc(r, 4 * i + t) << 4) + 8 * g) =
                        make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
                }
            }
        }
    const int k = lane % NC, r0 = lane / NC, n = n_base + k * EPC;
    const int rows = min(max(p.M - m_base, 0), 32 * MJ);
    uint8_t* crow = reinterpret_cast<uint8_t*>(p.C) + (int64_t)m_base * p.ldc * SZ;
    constexpr int STEPS = 32 * MJ / RPI, AT = STEPS < 8 ? STEPS : 8;  // rows per lane, rows in flight
    if (p.c_vec && p.N % EPC == 0) {
        // a resource that ends at row M, and an offset past it for chunks past N
        const __amdgpu_buffer_rsrc_t cres = uniform_rsrc(crow, (uint32_t)rows * (uint32_t)p.ldc * SZ);
        const uint32_t step = (uint32_t)(RPI * p.ldc * SZ);
        const uint32_t ofs0 = n < p.N ? (uint32_t)((r0 * p.ldc + n) * SZ) : 0x80000000u;
#pragma unroll
        for (int s = 0; s < STEPS; s += AT) {
            u32x4 v[AT];
#pragma unroll
            for (int u = 0; u < AT; u++) {
                const int r = RPI * (s + u) + r0;
                v[u] = *reinterpret_cast<const u32x4*>(stg + r * (16 * NC) + (swc(r, k) << 4));
            }
#pragma unroll
            for (int u = 0; u < AT; u++) __builtin_amdgcn_raw_buffer_store_b128(v[u], cres, ofs0 + (s + u) * step, 0, 0);
        }
    } else {
        typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
        for (int s = 0; s < STEPS; s++) {
            const int r = RPI * s + r0;
            if (r >= rows || n >= p.N) continue;
            const uint8_t* at = stg + r * (16 * NC) + (swc(r, k) << 4);
            uint8_t* to = crow + (r * p.ldc + n) * SZ;
            if (n + EPC <= p.N) {
                *reinterpret_cast<u32x4_u*>(to) = *reinterpret_cast<const u32x4*>(at);
            } else {
                for (int e = 0; e < p.N - n; e++) {
                    if constexpr (F32) reinterpret_cast<uint32_t*>(to)[e] = reinterpret_cast<const uint32_t*>(at)[e];
                    else reinterpret_cast<uint16_t*>(to)[e] = reinterpret_cast<const uint16_t*>(at)[e];
                }
            }
        }
    }
}

template <bool EXACT, int NI, int MJ, int NS>
__global__ __launch_bounds__(256, 1) void gemm_fp8_kernel(Fp8Gemm p) {
    constexpr int BN = 64 * NI, BM = 64 * MJ;
    constexpr int SCALES = (BN + BM) * ROW, STAGE = SCALES + BM * 4;
    constexpr int STG = 32 * MJ * 32 * NI * (EXACT ? 4 : 2);  // the epilogue's staging area, per wave
    constexpr int LDS = NS * STAGE > 4 * STG ? NS * STAGE : 4 * STG;
    __shared__ __align__(16) uint8_t lds[LDS];
    const int total = p.n_tiles * p.m_tiles;
    const int lid = xcd_remap(total);
    if (lid >= total) return;
    // four m-tiles per group, n advancing across the group
    constexpr int GM = 4;
    const int group = lid / (GM * p.n_tiles), first_m = group * GM, gm = min(p.m_tiles - first_m, GM);
    const int in_group = lid % (GM * p.n_tiles);
    const int m0 = (first_m + in_group % gm) * BM, n0 = in_group / gm * BN;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int wn = wave >> 1, wm = wave & 1;
    const int c = lane & 31, g = lane >> 5;

    // DMA: one instruction of a wave fills 8 rows; lane l lands in row l / 8, chunk
    // l % 8, so it fetches the chunk that the swizzle maps there.  Rows past N or M
    // lie past their resource and read zeros.
    const int lrow = lane >> 3;
    const int wrows = min(BN, p.N - n0), arows = min(BM, p.M - m0);
    const __amdgpu_buffer_rsrc_t wres = uniform_rsrc(p.W + (int64_t)n0 * p.K, (uint32_t)wrows * p.K);
    const __amdgpu_buffer_rsrc_t ares = uniform_rsrc(p.A + (int64_t)m0 * p.K, (uint32_t)arows * p.K);
    int woff[2 * NI], aoff[2 * MJ];
#pragma unroll
    for (int i = 0; i < 2 * NI; i++) {
        const int row = (wave * 2 * NI + i) * 8 + lrow;
        woff[i] = row * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < 2 * MJ; i++) {
        const int row = (wave * 2 * MJ + i) * 8 + lrow;
        aoff[i] = row * p.K + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
    constexpr int NP = 2 * NI + 2 * MJ + 1;  // DMA instructions of a wave per stage
    const int srow = (wave % MJ) * 64;       // the wave's 64 scale words (waves past MJ repeat the first ones')
    auto load_piece = [&](int kt, int slot, int x) __attribute__((always_inline)) {
        uint8_t* st = lds + slot * STAGE;
        if (x == NP - 1) {
            const uint32_t* words = p.as + (int64_t)(kt >> 2) * p.ld_as + m0;
            const __amdgpu_buffer_rsrc_t sres = uniform_rsrc(words, (uint32_t)arows * 4);
            uint8_t* dst = st + SCALES + srow * 4;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sres, (lptr_t)dst, 4, (srow + lane) * 4, 0, 0, 0);
            return;
        }
        const bool is_a = x >= 2 * NI;
        const int i = is_a ? x - 2 * NI : x;
        uint8_t* dst = st + (is_a ? BN * ROW + (wave * 2 * MJ + i) * 1024 : (wave * 2 * NI + i) * 1024);
        const int ofs = is_a ? aoff[i < 2 * MJ ? i : 0] : woff[i];
        if (is_a) __builtin_amdgcn_raw_ptr_buffer_load_lds(ares, (lptr_t)dst, 16, ofs, kt * ROW, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(wres, (lptr_t)dst, 16, ofs, kt * ROW, 0, 0);
    };

    f32x16 acc[NI][MJ];
    const int nk = p.K >> 7, last = nk - 1;
    int wrow[NI], arow[MJ];
#pragma unroll
    for (int i = 0; i < NI; i++) wrow[i] = wn * 32 * NI + 32 * i + c;
#pragma unroll
    for (int j = 0; j < MJ; j++) arow[j] = wm * 32 * MJ + 32 * j + c;
    i32x8 wf[2][NI], af[2][MJ];
    int sw, sa[MJ], sw_next = 0, sa_next[MJ];
    const int nb = min(n0 + wn * 32 * NI, p.N - 1) >> 7;
    // piece x of the fragments of half s of a stage (into buffer buf): two chunks of a row each
    auto read_piece = [&](int slot, int s, int buf, int x) __attribute__((always_inline)) {
        const uint8_t* ws = lds + slot * STAGE;
        const uint8_t* as = ws + BN * ROW;
        const int f = x >> 1, h = x & 1, ch = 4 * s + 2 * g + h;
        const i32x4 v = *reinterpret_cast<const i32x4*>(f < NI ? ws + swz(wrow[f < NI ? f : 0], ch)
                                                              : as + swz(arow[f < NI ? 0 : f - NI], ch));
        i32x8& d = f < NI ? wf[buf][f < NI ? f : 0] : af[buf][f < NI ? 0 : f - NI];
#pragma unroll
        for (int e = 0; e < 4; e++) d[4 * h + e] = v[e];
    };
    constexpr int NR = 2 * (NI + MJ);
    auto read_scales = [&](int kt, int slot) __attribute__((always_inline)) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(lds + slot * STAGE + SCALES);
#pragma unroll
        for (int j = 0; j < MJ; j++) sa_next[j] = (int)words[arow[j]];
        sw_next = (int)uniform_word(p.ws + (int64_t)(kt >> 2) * p.ld_ws + nb);
    };
    auto take_scales = [&](int kt) __attribute__((always_inline)) {  // byte kt % 4 of the words
        const int sh = 8 * (kt & 3);
        sw = sw_next >> sh;
#pragma unroll
        for (int j = 0; j < MJ; j++) sa[j] = sa_next[j] >> sh;
    };
    // One half block on fragment buffer `buf`; between its instructions the reads of
    // the next half (slot rslot, half rs, into buffer buf ^ 1) and, when `dma`, the DMA
    // pieces of stage dma_kt, all in the first half of them.
    auto half = [&](int buf, int rslot, int rs, bool do_read, bool dma, int dma_kt, int dma_slot, bool zc)
        __attribute__((always_inline)) {
        bf16x8 wb[EXACT ? NI : 1][4], ab[EXACT ? MJ : 1][4];
        if constexpr (EXACT) {
            const float fw = scale_of(sw & 0xff);
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) wb[i][e] = widen(wf[buf][i][2 * e], wf[buf][i][2 * e + 1], fw);
#pragma unroll
            for (int j = 0; j < MJ; j++) {
                const float fa = scale_of(sa[j] & 0xff);
#pragma unroll
                for (int e = 0; e < 4; e++) ab[j][e] = widen(af[buf][j][2 * e], af[buf][j][2 * e + 1], fa);
            }
        }
        constexpr int T = NI * MJ, RS = (2 * NR + T - 1) / T, DS = (2 * NP + T - 1) / T;
#pragma unroll
        for (int x = 0; x < T; x++) {
            const int i = x / MJ, j = x % MJ;
            f32x16 z;
#pragma unroll
            for (int e = 0; e < 16; e++) z[e] = 0.f;
            if constexpr (EXACT) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i][0], ab[j][0], zc ? z : acc[i][j], 0, 0, 0);
#pragma unroll
                for (int e = 1; e < 4; e++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[i][e], ab[j][e], acc[i][j], 0, 0, 0);
            } else {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[buf][i], af[buf][j], zc ? z : acc[i][j], 0, 0, 0,
                                                                           sw, 0, sa[j]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < RS; e++)
                if (do_read && x * RS + e < NR) read_piece(rslot, rs, buf ^ 1, x * RS + e);
#pragma unroll
            for (int e = 0; e < DS; e++)
                if (dma && x * DS + e < NP) load_piece(dma_kt, dma_slot, x * DS + e);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // While stage kt is computed from slot kt % NS, stages kt + 1 .. kt + NS - 1 land
    // in the others.  Half 0 of stage kt reads half 1's fragments from the same slot;
    // then every wave waits for its own DMA of stage kt + 1 and for its LDS reads, and
    // the barrier makes stage kt + 1 visible and slot kt % NS free: half 1 reads stage
    // kt + 1's first fragments and refills slot kt % NS with stage kt + NS (past the
    // last stage it repeats the last one, so that the count waited for stays fixed).
#pragma unroll
    for (int i = 0; i < NS; i++)
#pragma unroll
        for (int x = 0; x < NP; x++) load_piece(min(i, last), i, x);
    wait_vmem_lds<(NS - 1) * NP>();
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int x = 0; x < NR; x++) read_piece(0, 0, 0, x);
    read_scales(0, 0);
    take_scales(0);
    int slot = 0;
    auto next = [](int t) __attribute__((always_inline)) { return t + 1 == NS ? 0 : t + 1; };
    if (last == 0) {
        half(0, 0, 1, true, false, 0, 0, true);
        half(1, 0, 0, false, false, 0, 0, false);
    } else {
        half(0, 0, 1, true, false, 0, 0, true);
        wait_vmem_lds<(NS - 2) * NP>();
        __builtin_amdgcn_s_barrier();
        read_scales(1, 1);
        half(1, 1, 0, true, true, min(NS, last), 0, false);
        take_scales(1);
        slot = 1;
        for (int kt = 1; kt < last; kt++) {
            half(0, slot, 1, true, false, 0, 0, false);
            wait_vmem_lds<(NS - 2) * NP>();
            __builtin_amdgcn_s_barrier();
            read_scales(kt + 1, next(slot));
            half(1, next(slot), 0, true, true, min(kt + NS, last), slot, false);
            take_scales(kt + 1);
            slot = next(slot);
        }
        half(0, slot, 1, true, false, 0, 0, false);
        half(1, slot, 0, false, false, 0, 0, false);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last refills, which nobody reads
    __syncthreads();  // every wave is done with the operands: LDS becomes the staging area
    epilogue<EXACT, NI, MJ>(p, acc, n0 + wn * 32 * NI, m0 + wm * 32 * MJ, lane, lds + wave * STG);
}

struct Tile {
    int ni, mj, ns;
    float step, ends;  // measured, us: a block of K with every CU busy, and a tile's ends
};
constexpr Tile FAST[] = {{4, 4, 2, 1.0f, 6.f}, {4, 3, 2, 0.8f, 6.f}, {4, 2, 3, 0.55f, 5.f}, {2, 3, 3, 0.45f, 5.f},
                         {2, 2, 4, 0.32f, 4.f}, {2, 1, 4, 0.22f, 4.f}, {1, 1, 4, 0.15f, 3.f}};
constexpr Tile FULL[] = {{4, 2, 3, 1.0f, 6.f}, {2, 2, 4, 0.5f, 5.f}, {2, 1, 4, 0.3f, 4.f}, {1, 1, 4, 0.2f, 3.f}};

long tiles_of(const Fp8Gemm& p, const Tile& t) {
    return ((long)p.N + 64 * t.ni - 1) / (64 * t.ni) * (((long)p.M + 64 * t.mj - 1) / (64 * t.mj));
}
// rounds of one tile per CU, the last at 0.7 of a full round plus 0.3 of its share (as for the bf16 GEMM)
float tile_cost(const Fp8Gemm& p, const Tile& t, int cus) {
    const float r = (float)tiles_of(p, t) / cus;
    const float rounds = r <= 1.f ? 1.f : 0.7f * (float)(long)(r + 0.9999f) + 0.3f * r;
    return rounds * (t.step * (float)(p.K / 128) + t.ends);
}

template <int MJ>
void few_launch(Fp8Gemm& p, hipStream_t s) {
    constexpr int WAVES = 8;
    p.n_tiles = (p.N + 15) / 16;
    p.m_tiles = (p.M + 16 * MJ - 1) / (16 * MJ);
    hipLaunchKernelGGL((gemm_fp8_few_kernel<MJ, WAVES>), dim3(p.n_tiles * p.m_tiles), dim3(64 * WAVES), 0, s, p);
}

}  // namespace

hipError_t launch_gemm_fp8(Fp8Gemm& p, hipStream_t s) {
    if (p.M <= 64) {
        if (p.M <= 16) few_launch<1>(p, s);
        else if (p.M <= 32) few_launch<2>(p, s);
        else few_launch<4>(p, s);
        return hipGetLastError();
    }
    const int cus = device_cus();
    const Tile* t = p.c_f32 ? FULL : FAST;
    const Tile* end = p.c_f32 ? FULL + sizeof(FULL) / sizeof(Tile) : FAST + sizeof(FAST) / sizeof(Tile);
    for (const Tile* x = t + 1; x < end; x++)
        if (tile_cost(p, *x, cus) < tile_cost(p, *t, cus)) t = x;
    p.n_tiles = (p.N + 64 * t->ni - 1) / (64 * t->ni);
    p.m_tiles = (p.M + 64 * t->mj - 1) / (64 * t->mj);
    const dim3 grid(xcd_grid((long)p.n_tiles * p.m_tiles)), block(256);
#define TILE(E, NI, MJ, NS)                                                     \
    if (p.c_f32 == E && t->ni == NI && t->mj == MJ) {                           \
        hipLaunchKernelGGL((gemm_fp8_kernel<E, NI, MJ, NS>), grid, block, 0, s, p); \
        return hipGetLastError();                                               \
    }
    TILE(0, 4, 4, 2)
    TILE(0, 4, 3, 2)
    TILE(0, 4, 2, 3)
    TILE(0, 2, 3, 3)
    TILE(0, 2, 2, 4)
    TILE(0, 2, 1, 4)
    TILE(0, 1, 1, 4)
    TILE(1, 4, 2, 3)
    TILE(1, 2, 2, 4)
    TILE(1, 2, 1, 4)
    TILE(1, 1, 1, 4)
#undef TILE
    return hipErrorInvalidValue;
}

}  // namespace awa
