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
__device__ inline uint32_t upper(float a, float b) { return (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u); }
__device__ inline float truncated(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }

// Eight columns of a row of dy as PARTS words of bf16 pairs
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
    __device__ u32x4 part(int) const { return v; }
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
    // part x: the bits that the parts before it leave; an infinity is all in the first
    __device__ u32x4 part(int x) const {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            r[i] = v[i >> 2][i & 3];
            for (int k = 0; k < x; k++) {
                const float h = truncated(r[i]);
                r[i] = h == r[i] ? 0.f : r[i] - h;
            }
        }
        return (u32x4){upper(r[0], r[1]), upper(r[2], r[3]), upper(r[4], r[5]), upper(r[6], r[7])};
    }
};

// Chunk c (16 bytes) of row m lies at chunk c ^ sw(m): the four rows that 16 lanes of a transposed read
// touch begin at different banks.
__device__ inline int sw(int m) { return (m & 3) << 1; }

// TN x TK accumulators of 16 x 16 a wave, WN x WK waves.
template <int PARTS, int TN, int TK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) void grad_weight_kernel(GradWeight p) {
    constexpr int BN = 16 * TN * WN, BK = 16 * TK * WK, THREADS = 64 * WN * WK;
    constexpr int CN = BN / 8, CK = BK / 8;  // chunks of a row
    constexpr int NR = MS * CN / THREADS, KR = MS * CK / 2 / THREADS;  // a thread's pieces: 8 columns of dy, 16 of x
    static_assert(NR >= 1 && KR >= 1 && MS * CN % THREADS == 0 && MS * CK / 2 % THREADS == 0, "pieces");
    constexpr int PART = MS * BN * 2, STAGE = PARTS * PART + MS * BK * 2;
    __shared__ __align__(16) uint8_t lds[2 * STAGE];
    const int total = p.n_tiles * p.k_tiles * p.splits;
    const int wg = xcd_remap(total);
    if (wg >= total) return;
    const int per_split = p.n_tiles * p.k_tiles, split = wg / per_split;
    int n0, k0;
    {  // four n tiles side by side, k advancing
        constexpr int GN = 4;
        const int t = wg - split * per_split, group = t / (GN * p.k_tiles), first = group * GN, gn = min(p.n_tiles - first, GN);
        const int in = t - group * (GN * p.k_tiles);
        n0 = (first + in % gn) * BN;
        k0 = in / gn * BK;
    }
    const int m_first = split * p.rows_per, m_end = min(m_first + p.rows_per, p.M);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave / WK, wk = wave % WK;

    // pieces: the same columns in every stage
    const int nc = tid % CN, nr = tid / CN, kc = tid % (CK / 2), kr = tid / (CK / 2);
    using TD = typename DyPiece<PARTS>::T;
    const int n = n0 + 8 * nc, k = k0 + 16 * kc, block = k >> 7;
    const TD* dy = reinterpret_cast<const TD*>(p.dy) + n;
    const uint8_t* q = p.q + k;
    const uint32_t* words = p.s + (int64_t)(block >> 2) * p.ld_s;
    DyPiece<PARTS> d[NR];
    u32x4 x[KR];
    uint32_t xs[KR];
    auto load = [&](int m0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NR; j++) {
            const int m = m0 + nr + j * (THREADS / CN);
            if (m < m_end && n + 8 <= p.N) d[j].load(dy + (int64_t)m * p.lddy);
            else if (m < m_end && n < p.N) d[j].load_some(dy + (int64_t)m * p.lddy, p.N - n);
            else d[j].zero();
        }
#pragma unroll
        for (int j = 0; j < KR; j++) {
            const int m = m0 + kr + j * (THREADS / (CK / 2));
            x[j] = (u32x4){0, 0, 0, 0};
            xs[j] = 0;
            if (m < m_end && k < p.kp) {
                x[j] = *reinterpret_cast<const u32x4*>(q + (int64_t)m * p.kp);
                xs[j] = words[m];
            }
        }
    };
    auto store = [&](uint8_t* st) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NR; j++) {
            const int m = nr + j * (THREADS / CN);
#pragma unroll
            for (int i = 0; i < PARTS; i++)
                *reinterpret_cast<u32x4*>(st + i * PART + m * (2 * BN) + ((nc ^ sw(m)) << 4)) = d[j].part(i);
        }
#pragma unroll
        for (int j = 0; j < KR; j++) {
            const int m = kr + j * (THREADS / (CK / 2));
            const float sc = scale_of(xs[j] >> (8 * (block & 3)) & 0xff);
            uint8_t* row = st + PARTS * PART + m * (2 * BK);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    w[2 * i] = pk(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[j][2 * h + i], sc, false));
                    w[2 * i + 1] = pk(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[j][2 * h + i], sc, true));
                }
                *reinterpret_cast<u32x4*>(row + (((2 * kc + h) ^ sw(m)) << 4)) = w;
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

    const int stages = (m_end - m_first + MS - 1) / MS;
    if (stages > 0) {
        load(m_first);
        store(lds);
        load(m_first + MS);
    }
    for (int st = 0; st < stages; st++) {
        __syncthreads();
        const uint8_t* now = lds + (st & 1) * STAGE;
        if (st + 1 < stages) {
            store(lds + ((st + 1) & 1) * STAGE);
            load(m_first + (st + 2) * MS);
        }
        bf16x8 b[PARTS][TN];
#pragma unroll
        for (int i = 0; i < PARTS; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) b[i][j] = frag(now + i * PART, 2 * BN, wn * TN + j);
#pragma unroll
        for (int i = 0; i < TK; i++) {
            const bf16x8 a = frag(now + PARTS * PART, 2 * BK, wk * TK + i);
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int h = PARTS - 1; h >= 0; h--)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[h][j], acc[i][j], 0, 0, 0);
        }
        if (sums) {
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int h = PARTS - 1; h >= 0; h--)
                    sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, b[h][j], sum[j], 0, 0, 0);
        }
    }

    const bool whole = p.splits == 1;
    float* part = whole ? nullptr : p.part + (int64_t)split * ((int64_t)p.N * p.K + p.N);
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int row = n0 + (wn * TN + j) * 16 + (lane & 15);
        if (row >= p.N) continue;
        if (sums && lane < 16) {
            if (!whole) part[(int64_t)p.N * p.K + row] = sum[j][0];
            else p.db[row] = p.add ? p.db[row] + sum[j][0] : sum[j][0];
        }
#pragma unroll
        for (int i = 0; i < TK; i++) {
            const int col = k0 + (wk * TK + i) * 16 + 4 * (lane >> 4), left = p.K - col;
            if (left <= 0) continue;
            f32x4 v = acc[i][j];
            if (!whole || p.w_f32) {
                float* to = whole ? reinterpret_cast<float*>(p.dw) + row * p.ldw + col : part + (int64_t)row * p.K + col;
                if (whole && p.add) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e < left) v[e] += to[e];
                }
                if (left >= 4) {
                    *reinterpret_cast<f32x4_4*>(to) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e < left) to[e] = v[e];
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
    }
}

// The splits' sums, in their order: four columns a thread, rows over the grid's second dimension
__global__ __launch_bounds__(256) void grad_weight_join_kernel(GradWeight p) {
    const int64_t stride = (int64_t)p.N * p.K + p.N;
    for (int64_t row = blockIdx.y; row < p.N; row += gridDim.y) {
        if (p.db && blockIdx.x == 0 && threadIdx.x == 0) {
            float s = p.add ? p.db[row] : 0.f, t = 0.f;
            for (int i = 0; i < p.splits; i++) t += p.part[i * stride + (int64_t)p.N * p.K + row];
            p.db[row] = s + t;
        }
        const int col = (blockIdx.x * 256 + threadIdx.x) * 4, left = p.K - col;
        if (left <= 0) continue;
        const float* from = p.part + row * p.K + col;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (left >= 4) {
            for (int i = 0; i < p.splits; i++) v += *reinterpret_cast<const f32x4_4*>(from + i * stride);
        } else {
            for (int i = 0; i < p.splits; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (e < left) v[e] += from[i * stride + e];
        }
        const int count = min(left, 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (e >= count) continue;
            if (p.w_f32) {
                float* to = reinterpret_cast<float*>(p.dw) + row * p.ldw + col + e;
                *to = p.add ? *to + v[e] : v[e];
            } else {
                reinterpret_cast<uint16_t*>(p.dw)[row * p.ldw + col + e] = (uint16_t)bf16x2_rne(v[e], v[e]);
            }
        }
    }
}

template <int PARTS, int TN, int TK, int WN, int WK>
void run(GradWeight& a, hipStream_t s) {
    a.n_tiles = (a.N + 16 * TN * WN - 1) / (16 * TN * WN);
    a.k_tiles = (a.K + 16 * TK * WK - 1) / (16 * TK * WK);
    hipLaunchKernelGGL((grad_weight_kernel<PARTS, TN, TK, WN, WK>), dim3(xcd_grid((long)a.n_tiles * a.k_tiles * a.splits)),
                       dim3(64 * WN * WK), 0, s, a);
}

}  // namespace

int grad_weight_splits(int dtype_dy, int dtype_w, int M, int N, int K) {
    const int64_t tiles = (int64_t)((N + 127) / 128) * ((K + 127) / 128);
    const int64_t fill = 512 / std::max<int64_t>(tiles, 1);
    return (int)std::max<int64_t>(1, std::min<int64_t>({fill, M / 256, 16}));
}

hipError_t launch_grad_weight(int dtype_dy, GradWeight& a, hipStream_t s) {
    a.rows_per = ((a.M + a.splits - 1) / a.splits + MS - 1) / MS * MS;
    if (dtype_dy == AWA_F32) run<3, 4, 4, 2, 2>(a, s);
    else run<1, 4, 4, 2, 2>(a, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(grad_weight_join_kernel, dim3((unsigned)((a.K + 1023) / 1024), (unsigned)std::min(a.N, 65535)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace awa
