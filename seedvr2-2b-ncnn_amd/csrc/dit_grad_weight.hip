// dit_grad_weight.hip — a weight's gradient from 8-bit rows: dW[n][k] = sum over m of dy[m][n] x[m][k].
//
// The sum runs over rows, so a row's scale cannot wait for the accumulator: x is widened to bf16 with
// its scale on the way into LDS (bf16 holds every e4m3 value, times any power of two).  Both operands
// lie in LDS as rows m of columns, and the matrix instructions' operands, eight m of one column a lane,
// come from transposed reads; x's columns are the instruction's rows and dy's its columns, so that a
// lane ends with four consecutive k of one n.  fp32 dy is taken apart into three bf16 values, which hold
// its 24 bits, and takes three instructions.  db is a product with ones, in the workgroups of the first
// columns of x.
//
// Where dW has few tiles the rows are divided over workgroups, whose sums a second kernel adds in order.
//
// Bound by LDS: of the 1,930 cycles of a stage of a 256 x 256 tile its 192 transposed reads (6 cycles for 512 bytes, in any
// layout) and the 32 KB that are written take 1,400, its matrix instructions 1,024; in tiles of 128 x 128 the share is larger.
// bf16 dy and dW: 5498 x 13824 x 2560 327 to 346 us (1.16 PFLOP/s), 5498 x 7680 x 2560 196 to 210 (1.1), 5498 x 2560 x 2560 87 to 94,
// 679 x 7680 x 2560 41 to 46, 58 x 7680 x 2560 15 to 16.  fp32 dy: 5498 x 13824 x 2560 1010 to 1040 (three instructions a product:
// 1.1 PFLOP/s of them), 1237 x 1999 x 2693 57.
#include <algorithm>

#include "dit_device.hpp"
#include "dit_train_internal.hpp"

namespace awa {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __attribute__((address_space(3))) bf16x4 lbf16x4_t;

constexpr int MS = 32;  // rows of a stage: one instruction's

__device__ inline float scale_of(uint32_t b) { return __uint_as_float(b ? b << 23 : 0x400000u); }  // 2^(b - 127)
__device__ inline uint32_t pk(bf16x2 v) { return __builtin_bit_cast(uint32_t, v); }
// upper halves of a and b as one word
__device__ inline uint32_t upper(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ inline float truncated(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }

// Eight columns of a row of dy, and the bf16 parts that they are the sum of
template <int PARTS> struct DyPiece;
template <> struct DyPiece<1> {
    using T = uint16_t;
    u32x4 v;
    __device__ void load(const T* p) { v = *reinterpret_cast<const u32x4_2*>(p); }
    __device__ void load_some(const T* p, int n) {
        v = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
    __device__ void zero() { v = (u32x4){0, 0, 0, 0}; }
    __device__ void parts(u32x4 (&out)[1]) const { out[0] = v; }
};
template <> struct DyPiece<3> {
    using T = float;
    f32x4 v[2];
    __device__ void load(const T* p) {
        v[0] = *reinterpret_cast<const f32x4_4*>(p);
        v[1] = *reinterpret_cast<const f32x4_4*>(p + 4);
    }
    __device__ void load_some(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i >> 2][i & 3] = i < n ? p[i] : 0.f;
    }
    __device__ void zero() { v[0] = v[1] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
    // each part the upper 16 bits of what the parts before it leave: 8 + 8 + 8 bits
    __device__ void parts(u32x4 (&out)[3]) const {
        float r[8], top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            r[i] = v[i >> 2][i & 3];
            top = fmaxf(top, fabsf(r[i]));
        }
        const bool infinite = __builtin_amdgcn_ballot_w64(top == INFINITY) != 0;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            out[k] = (u32x4){upper(r[0], r[1]), upper(r[2], r[3]), upper(r[4], r[5]), upper(r[6], r[7])};
#pragma unroll
            for (int i = 0; i < 8 && k < 2; i++) r[i] -= truncated(r[i]);
            if (k == 0 && infinite) {  // an infinity is all in the first part
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (fabsf(v[i >> 2][i & 3]) == INFINITY) r[i] = 0.f;
            }
        }
    }
};

// Chunk c (16 bytes) of row m lies at chunk c ^ sw(m): the eight rows of which 32 lanes of a transposed read
// take two neighbouring chunks, and the every other chunk of two rows that 16 lanes write, are in different banks.
__device__ inline int sw(int m) { return ((m & 7) << 1) | (m & 1); }

// Four columns of a row of dW, of which `left` are there
__device__ inline void put(const GradWeight& p, int row, int col, int left, f32x4 v) {
    if (p.w_f32) {
        float* to = reinterpret_cast<float*>(p.dw) + row * p.ldw + col;
        if (left >= 4) {
            if (p.add) v += *reinterpret_cast<const f32x4_4*>(to);
            *reinterpret_cast<f32x4_4*>(to) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < left) to[e] = p.add ? to[e] + v[e] : v[e];
        }
    } else {
        typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
        uint16_t* to = reinterpret_cast<uint16_t*>(p.dw) + row * p.ldw + col;
        const u32x2_2 w = {bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3])};
        if (left >= 4) {
            *reinterpret_cast<u32x2_2*>(to) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < left) to[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}

// Tile t: four n tiles side by side, k advancing
template <int BN, int BK>
__device__ inline void place(const GradWeight& p, int t, int& n0, int& k0) {
    constexpr int GN = 4;
    const int group = t / (GN * p.k_tiles), first = group * GN, gn = min(p.n_tiles - first, GN);
    const int in = t - group * (GN * p.k_tiles);
    n0 = (first + in % gn) * BN;
    k0 = in / gn * BK;
}

// TN x TK accumulators of 16 x 16 a wave, WN x WK waves; at least two waves a SIMD.
template <int PARTS, int TN, int TK, int WN, int WK, int DEPTH>
__global__ __launch_bounds__(64 * WN * WK, 2) void grad_weight_kernel(GradWeight p) {
    constexpr int BN = 16 * TN * WN, BK = 16 * TK * WK, THREADS = 64 * WN * WK;
    constexpr int CN = BN / 8, CK = BK / 8;  // chunks of a row
    // a thread's pieces: 8 columns of dy, 16 of x (8 where there are more threads)
    constexpr int XC = MS * CK / 2 >= THREADS ? 2 : 1, XR = CK / XC;
    constexpr int NR = MS * CN / THREADS, KR = MS * XR / THREADS;
    static_assert(NR >= 1 && KR >= 1 && MS * CN % THREADS == 0 && MS * XR % THREADS == 0, "pieces");
    typedef uint32_t xpiece __attribute__((ext_vector_type(2 * XC)));
    constexpr int PART = MS * BN * 2, STAGE = PARTS * PART + MS * BK * 2;
    __shared__ __align__(16) uint8_t lds[2 * STAGE];
    // whole tiles, then those whose rows are divided
    int tile, split = -1;
    if ((int)blockIdx.x < p.whole) {
        // the XCD's contiguous range; the few past a multiple of 8 are the last ones
        const int per = p.whole >> 3, b = (int)blockIdx.x;
        tile = b < 8 * per ? (b & 7) * per + (b >> 3) : b;
    } else {
        const int b = (int)blockIdx.x - p.whole, rest = p.n_tiles * p.k_tiles - p.whole, per = (rest * p.splits + 7) >> 3;
        const int i = (b & 7) * per + (b >> 3);
        if (i >= rest * p.splits) return;
        split = i / rest;
        tile = p.whole + i - split * rest;
    }
    int n0, k0;
    place<BN, BK>(p, tile, n0, k0);
    const int m_first = max(split, 0) * p.rows_per, m_end = split < 0 ? p.M : min(m_first + p.rows_per, p.M);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / WK, wk = wave % WK;

    // pieces: the same columns in every stage
    const int nc = tid % CN, nr = tid / CN, kc = tid % XR, kr = tid / XR;
    using TD = typename DyPiece<PARTS>::T;
    const int n = n0 + 8 * nc, k = k0 + 8 * XC * kc, block = k >> 7;
    struct Pieces {
        DyPiece<PARTS> d[NR];
        xpiece x[KR];
        uint32_t xs[KR];
    };
    // A lane's offsets inside a stage are the same for all (32 bits: rows are at most 2^20 elements), its rows' address is
    // the wave's.  Columns past N or K only reach results past them, so only rows past the end have to be zeros: pieces past
    // the last column are read from the tile's first, and one across it goes on into the next row, where there is one.
    // Stages for which that holds are loaded without a branch, so that the loads of several are on their way at once.
    const uint32_t dy_of = (uint32_t)nr * (uint32_t)p.lddy + (n < p.N ? 8 * nc : 0);
    const uint32_t q_of = (uint32_t)kr * (uint32_t)p.kp + (k < p.kp ? 8 * XC * kc : 0);
    const TD* const dy0 = reinterpret_cast<const TD*>(p.dy) + n0;
    const uint8_t* const q0 = p.q + k0;
    const uint32_t* const s0 = p.s + (int64_t)(k0 >> 9) * p.ld_s;  // a tile's columns have one word a row
    const int plain = p.N < 8 ? 0 : (n0 + BN <= p.N || m_end < p.M ? m_end - m_first : m_end - m_first - 1) / MS;
    auto load = [&](Pieces& r, int st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NR; j++) r.d[j].load(dy0 + (m_first + st * MS + j * (THREADS / CN)) * p.lddy + dy_of);
#pragma unroll
        for (int j = 0; j < KR; j++) {
            const int m = m_first + st * MS + j * (THREADS / XR);
            r.x[j] = *reinterpret_cast<const xpiece*>(q0 + (int64_t)m * p.kp + q_of);
            r.xs[j] = (s0 + m)[kr];
        }
    };
    // any stage
    auto load_any = [&](Pieces& r, int st) __attribute__((always_inline)) {
        if (st < plain) {
            load(r, st);
            return;
        }
#pragma unroll
        for (int j = 0; j < NR; j++) {
            const int m = m_first + st * MS + j * (THREADS / CN);
            r.d[j].zero();
            if (m + nr < m_end && n + 8 <= p.N) r.d[j].load(dy0 + m * p.lddy + dy_of);
            else if (m + nr < m_end && n < p.N) r.d[j].load_some(dy0 + m * p.lddy + dy_of, p.N - n);
        }
#pragma unroll
        for (int j = 0; j < KR; j++) {
            const int m = m_first + st * MS + j * (THREADS / XR);
            r.x[j] = (xpiece)0u;
            r.xs[j] = 0;
            if (m + kr < m_end) {
                r.x[j] = *reinterpret_cast<const xpiece*>(q0 + (int64_t)m * p.kp + q_of);
                r.xs[j] = (s0 + m)[kr];
            }
        }
    };
    auto store = [&](const Pieces& r, uint8_t* st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NR; j++) {
            const int m = nr + j * (THREADS / CN);
            u32x4 part[PARTS];
            r.d[j].parts(part);
#pragma unroll
            for (int i = 0; i < PARTS; i++)
                *reinterpret_cast<u32x4*>(st + i * PART + m * (2 * BN) + ((nc ^ sw(m)) << 4)) = part[i];
        }
#pragma unroll
        for (int j = 0; j < KR; j++) {
            const int m = kr + j * (THREADS / XR);
            const float sc = scale_of(r.xs[j] >> (8 * (block & 3)) & 0xff);
            uint8_t* row = st + PARTS * PART + m * (2 * BK);
#pragma unroll
            for (int h = 0; h < XC; h++) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    w[2 * i] = pk(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[j][2 * h + i], sc, false));
                    w[2 * i + 1] = pk(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[j][2 * h + i], sc, true));
                }
                *reinterpret_cast<u32x4*>(row + (((XC * kc + h) ^ sw(m)) << 4)) = w;
            }
        }
    };

    f32x4 acc[TK][TN], sum[TN];
#pragma unroll
    for (int i = 0; i < TK; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < TN; j++) sum[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const bool sums = p.db && k0 == 0 && wk == 0;
    const __bf16 one = (__bf16)1.f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};
    // lane 16 g + 4 i + a of a transposed read addresses row 4 g + i, columns 4 a .. 4 a + 3 of the block,
    // and receives its own column's rows 4 g .. 4 g + 3
    const int tr_row = 4 * (lane >> 4) + ((lane >> 2) & 3), tr_a = lane & 3;
    auto frag = [&](const uint8_t* rows, int width, int col16) __attribute__((always_inline)) {
        const uint8_t* at = rows + tr_row * width + (((2 * col16 + (tr_a >> 1)) ^ sw(tr_row)) << 4) + ((tr_a & 1) << 3);
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lbf16x4_t*)at);
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lbf16x4_t*)(at + 16 * width));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // a stage's loads have DEPTH stages to arrive
    const int stages = (m_end - m_first + MS - 1) / MS;
    Pieces r0, r1;
    // A stage's products, and `aside`, the next stage's way into LDS.  For bf16 dy fragments are asked for a block of x ahead
    // of their use, with `aside` behind the first ones, and fences keep that order: without them each block's reads come right
    // before its products, which wait for them (5498 x 13824 x 2560 327 to 346 us for 360 to 390).  With three parts the products hide the
    // reads and the order costs (1237 x 1999 x 2693 61 us for 57).
    auto products = [&](const uint8_t* now, auto aside) __attribute__((always_inline)) {
        constexpr bool AHEAD = PARTS == 1;
        if constexpr (!AHEAD) aside();
        const uint8_t* const x = now + PARTS * PART;
        bf16x8 b[PARTS][TN], a[2];
        a[0] = frag(x, 2 * BK, wk * TK);
#pragma unroll
        for (int h = 0; h < PARTS; h++)
#pragma unroll
            for (int j = 0; j < TN; j++) b[h][j] = frag(now + h * PART, 2 * BN, wn * TN + j);
        if constexpr (AHEAD) {
            __builtin_amdgcn_sched_barrier(0);
            aside();
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < TK; i++) {
            if (i + 1 < TK) a[(i + 1) & 1] = frag(x, 2 * BK, wk * TK + i + 1);
            if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = PARTS - 1; h >= 0; h--)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i & 1], b[h][j], acc[i][j], 0, 0, 0);
            if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
        if (sums) {
#pragma unroll
            for (int h = PARTS - 1; h >= 0; h--)
#pragma unroll
                for (int j = 0; j < TN; j++) sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, b[h][j], sum[j], 0, 0, 0);
        }
    };
    // stage st, while the next one goes to LDS and the DEPTH-th after that is fetched
    auto step = [&](int st, Pieces& r) __attribute__((always_inline)) {
        __syncthreads();
        products(lds + (st & 1) * STAGE, [&]() __attribute__((always_inline)) {
            store(r, lds + ((st + 1) & 1) * STAGE);
            load(r, st + 1 + DEPTH);
        });
    };
    auto step_any = [&](int st, Pieces& r) __attribute__((always_inline)) {
        __syncthreads();
        products(lds + (st & 1) * STAGE, [&]() __attribute__((always_inline)) {
            if (st + 1 >= stages) return;
            store(r, lds + ((st + 1) & 1) * STAGE);
            load_any(r, st + 1 + DEPTH);
        });
    };
    int st = 0;
    if (stages > 0) {
        load_any(r0, 0);
        if constexpr (DEPTH == 2) load_any(r1, 1);
        store(r0, lds);
        load_any(r0, DEPTH);
    }
    Pieces& odd = DEPTH == 2 ? r1 : r0;  // of stage 1
    for (; st + 2 + DEPTH < plain; st += 2) {
        step(st, odd);
        step(st + 1, r0);
    }
#pragma unroll 1
    for (; st < stages; st += 2) {
        step_any(st, odd);
        if (st + 1 < stages) step_any(st + 1, r0);
    }

    const bool whole = split < 0;
    // a part of a divided tile: [BN][BK], then db's [BN]
    float* part = whole ? nullptr : p.part + ((int64_t)(tile - p.whole) * p.splits + split) * ((int64_t)BN * BK + BN);
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int row = n0 + (wn * TN + j) * 16 + (lane & 15);
        const bool there = row < p.N;
        if (sums && there && lane < 16) {
            if (!whole) part[BN * BK + row - n0] = sum[j][0];
            else p.db[row] = p.add ? p.db[row] + sum[j][0] : sum[j][0];
        }
        const int g = lane >> 4, col0 = k0 + wk * TK * 16;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < TK; i++) {
                const int col = col0 + 16 * i + 4 * g;
                if (there && col < p.K) *reinterpret_cast<f32x4*>(part + (row - n0) * BK + (col - k0)) = acc[i][j];
            }
        } else if (p.w_f32) {
#pragma unroll
            for (int i = 0; i < TK; i++) {
                const int col = col0 + 16 * i + 4 * g;
                if (there && col < p.K) put(p, row, col, p.K - col, acc[i][j]);
            }
        } else {
            // neighbouring lane groups exchange halves of two blocks, so that each stores 16 bytes
#pragma unroll
            for (int i = 0; i < TK; i += 2) {
                const f32x4 a = acc[i][j], b = acc[i + 1][j];
                const auto x = __builtin_amdgcn_permlane16_swap(bf16x2_rne(a[0], a[1]), bf16x2_rne(b[0], b[1]), false, false);
                const auto y = __builtin_amdgcn_permlane16_swap(bf16x2_rne(a[2], a[3]), bf16x2_rne(b[2], b[3]), false, false);
                const u32x4_2 w = {x[0], y[0], x[1], y[1]};
                const int col = col0 + 16 * (i + (g & 1)) + 8 * (g >> 1), left = there ? p.K - col : 0;
                uint16_t* to = reinterpret_cast<uint16_t*>(p.dw) + row * p.ldw + col;
                if (left >= 8) {
                    *reinterpret_cast<u32x4_2*>(to) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (e < left) to[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
}

// The divided tiles' parts, in their order: four columns a thread, a tile's rows over the grid's second dimension
template <int BN, int BK>
__global__ __launch_bounds__(256) void grad_weight_join_kernel(GradWeight p) {
    constexpr int ROWS = 1024 / BK;  // of a workgroup
    constexpr int64_t SIZE = (int64_t)BN * BK + BN;
    int n0, k0;
    place<BN, BK>(p, p.whole + blockIdx.x, n0, k0);
    const float* part = p.part + (int64_t)blockIdx.x * p.splits * SIZE;
    const int r = blockIdx.y * ROWS + threadIdx.x / (BK / 4), c = threadIdx.x % (BK / 4) * 4;
    const int row = n0 + r, col = k0 + c, left = p.K - col;
    if (row >= p.N) return;
    if (p.db && k0 == 0 && c == 0) {
        float s = 0.f;
        for (int i = 0; i < p.splits; i++) s += part[i * SIZE + BN * BK + r];
        p.db[row] = p.add ? p.db[row] + s : s;
    }
    if (left <= 0) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < p.splits; i++) v += *reinterpret_cast<const f32x4*>(part + i * SIZE + r * BK + c);
    put(p, row, col, left, v);
}

template <int PARTS, int TN, int TK, int WN, int WK, int DEPTH>
hipError_t run(const GradWeight& a, hipStream_t s) {
    constexpr int BN = 16 * TN * WN, BK = 16 * TK * WK;
    const int rest = a.n_tiles * a.k_tiles - a.whole;
    hipLaunchKernelGGL((grad_weight_kernel<PARTS, TN, TK, WN, WK, DEPTH>), dim3((unsigned)a.whole + xcd_grid((long)rest * a.splits)),
                       dim3(64 * WN * WK), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || rest == 0) return e;
    hipLaunchKernelGGL((grad_weight_join_kernel<BN, BK>), dim3((unsigned)rest, BN * BK / 1024), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

// Tiles of 256 x 256 (a workgroup per CU; not for fp32 dy) or 128 x 128 (two).  Tiles fill the chip in whole rounds; the
// rows of those that are left over (all, of a small dW) may be divided so that they fill one more.  Tile and parts are
// those with the least estimated time: a stage of 32 rows takes 0.82 us and a tile's ends 9 for 256 x 256, 0.58 and 5 for two
// of 128 x 128 (fp32 dy 1.1 and 6), the parts' sums 5 and their bytes, written and read, at 8 TB/s (from the caches).
GradWeightPlan grad_weight_plan(int dtype_dy, int M, int N, int K) {
    GradWeightPlan best{};
    double least = 0;
    for (int tile : {128, 256}) {
        if (tile == 256 && dtype_dy == AWA_F32) continue;
        const int64_t all = (int64_t)((N + tile - 1) / tile) * ((K + tile - 1) / tile), slots = tile == 256 ? 256 : 512;
        const int64_t rest = all % slots, stages = (M + MS - 1) / MS;
        const double ts = tile == 256 ? 0.82 : dtype_dy == AWA_F32 ? 1.1 : 0.58, t0 = tile == 256 ? 9 : dtype_dy == AWA_F32 ? 6 : 5;
        const int64_t most = rest ? std::max<int64_t>(std::min<int64_t>({slots / rest, stages / 4, 64}), 1) : 1;
        for (int64_t s = 1; s <= most; s++) {
            const int64_t per = (stages + s - 1) / s;
            const double bytes = (double)(rest * s) * tile * tile * 8;
            const double alone = slots == 512 && rest * s <= 256 ? 0.6 : 1.0;  // one workgroup a CU
            const double t = (double)(all / slots) * ((double)stages * ts + t0) + (rest ? (double)per * ts * alone + t0 : 0.0) +
                             (s > 1 ? 5.0 + bytes / 8e6 : 0.0);
            if (best.tile && t >= least) continue;
            least = t;
            best.tile = tile;
            best.splits = (int)s;
            best.whole = (int)(s > 1 ? all - rest : all);
            best.rows_per = s > 1 ? (int)per * MS : M;
            best.work = s > 1 ? rest * s * ((int64_t)tile * tile + tile) * 4 : 0;
        }
    }
    return best;
}

hipError_t launch_grad_weight(int dtype_dy, GradWeight& a, hipStream_t s) {
    const GradWeightPlan p = grad_weight_plan(dtype_dy, a.M, a.N, a.K);
    a.n_tiles = (a.N + p.tile - 1) / p.tile;
    a.k_tiles = (a.K + p.tile - 1) / p.tile;
    a.whole = p.whole;
    a.splits = p.splits;
    a.rows_per = p.rows_per;
    if (dtype_dy == AWA_F32) return run<3, 4, 4, 2, 2, 2>(a, s);
    return p.tile == 256 ? run<1, 8, 4, 2, 4, 1>(a, s) : run<1, 4, 4, 2, 2, 2>(a, s);
}

}  // namespace awa
