// dit_norm.hip — layer norm of rows and its gradient.
//
// Forward.  A row stays in registers: its sum gives a first mean, a second pass over the
// registers the mean of what is left and the squares of it, so that neither a large common
// value nor the first sum's rounding reaches the variance:
//   d = x - m0,  r = sum d / K,  mean = m0 + r,  var = sum d^2 / K - r^2.
// Backward.  With h = (x - mean) rstd and a = dy w a row needs sum a and sum a h, and every
// column sum dy h and sum dy over the rows: lanes keep their columns' sums in registers over
// all rows of their wave, waves add theirs in LDS in a fixed order, workgroups leave a row of
// partial sums each, which a second kernel adds in their order.
//
// Both are bound by HBM: each value is read once and written once.  Calls back to back on two inputs in turn; one input alone
// stays partly in the memory-side cache (times in brackets).  Forward, 27258 x 2560: fp32 to bf16 81 us (70; 5.2 TB/s), bf16 56 to 60
// (48; 4.7 TB/s); 12370 x 2693 bf16 32.5; 5498 x 2560 bf16 14.7 (12.7).  Gradient, bf16 dy and dx: 27258 x 2560 with bf16 x
// 82 us (76; 5.1 TB/s), 8-bit x 89 (79), fp32 x 104; 5498 x 2560 bf16 23, fp32 x and dx 29; 12370 x 2693 with 8-bit x 47, where rows
// that begin anywhere cost 8 % (2688 columns 44; 82 MB are written for 67); of these 4 us are the partial sums' kernel.
#include <algorithm>

#include "dit_train_internal.hpp"

namespace awa {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
// rows are only known to be aligned to their elements
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

struct Fp8 {
    uint8_t v;
};

// A lane's piece: four consecutive columns, 256 between the pieces of a lane.
constexpr int V = 4, STEP = 64 * V;

template <typename T> struct Raw;
template <> struct Raw<float> {
    f32x4 v;
    __device__ void load(const float* p) { v = *reinterpret_cast<const f32x4_4*>(p); }
    __device__ void load_some(const float* p, int n) {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = i < n ? p[i] : 0.f;
    }
    __device__ float get(int i) const { return v[i]; }
};
template <> struct Raw<uint16_t> {
    u32x2 v;
    __device__ void load(const uint16_t* p) { v = *reinterpret_cast<const u32x2_2*>(p); }
    __device__ void load_some(const uint16_t* p, int n) {
        v = (u32x2){0, 0};
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    }
    __device__ float get(int i) const { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
};

template <typename T>
__device__ inline void load_piece(Raw<T>& r, const T* row, int col, int K) {
    if (col + V <= K) r.load(row + col);
    else r.load_some(row + col, max(K - col, 0));
}

__device__ inline void store_piece(float* p, const f32x4& v, int n) {
    if (n >= V) {
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4_4*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = v[i];
    }
}
__device__ inline void store_piece(uint16_t* p, const f32x4& v, int n) {
    const u32x2 w = {bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3])};
    if (n >= V) {
        __builtin_nontemporal_store(w, reinterpret_cast<u32x2_2*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

template <int CTRL>
__device__ inline float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false));
}
// over the 64 lanes, the same bits in each
__device__ inline float wave_sum(float v) {
    v = dpp_add<0xB1>(v);   // lane ^ 1
    v = dpp_add<0x4E>(v);   // lane ^ 2
    v = dpp_add<0x141>(v);  // mirrored in 8: the other four
    v = dpp_add<0x140>(v);  // mirrored in 16
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// two sums over the WPR waves of a row, in the waves' order; `at`: LDS that no other call of the row's
// uses (a wave may run ahead by one call)
template <int WPR>
__device__ inline void row_sums(float& a, float& b, float2* at, int wave) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) at[wave] = make_float2(a, b);
        __syncthreads();
        a = 0.f;
        b = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; i++) {
            a += at[i].x;
            b += at[i].y;
        }
    }
}

// R pieces a lane; WPR waves a row, 4 waves a workgroup.
template <typename TX, typename TY, int R, int WPR>
__global__ __launch_bounds__(256) void layer_norm_kernel(NormFwd a) {
    constexpr int WAVES = 4, ROWS = WAVES / WPR;
    __shared__ float2 part[2][WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + wave / WPR;
    if (row >= a.M) return;  // whole workgroups where waves share a row
    const int col0 = (wave % WPR) * (R * STEP) + lane * V;
    const TX* x = reinterpret_cast<const TX*>(a.x) + row * a.ldx;
    Raw<TX> v[R];
#pragma unroll
    for (int i = 0; i < R; i++) load_piece(v[i], x, col0 + i * STEP, a.K);
    const float inv = 1.f / (float)a.K;
    float s = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < R; i++) s += (v[i].get(0) + v[i].get(1)) + (v[i].get(2) + v[i].get(3));
    row_sums<WPR>(s, none, part[0], wave);
    const float m0 = s * inv;
    float sd = 0.f, ss = 0.f;
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = col0 + i * STEP + j < a.K ? v[i].get(j) - m0 : 0.f;
            sd += d;
            ss += d * d;
        }
    row_sums<WPR>(sd, ss, part[1], wave);
    const float r = sd * inv, var = fmaxf(ss * inv - r * r, 0.f);
    // fmaxf takes a NaN's other operand
    const float rstd = 1.f / sqrtf((ss == ss ? var : ss) + a.eps);
    if (a.stats && lane == 0 && wave % WPR == 0) a.stats[row] = make_float2(m0 + r, rstd);
    TY* y = reinterpret_cast<TY*>(a.y) + row * a.ldy;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int col = col0 + i * STEP;
        if (col >= a.K) continue;
        f32x4 w = {1.f, 1.f, 1.f, 1.f}, b = {0.f, 0.f, 0.f, 0.f};
        if (a.w) {
            Raw<float> t;
            load_piece(t, a.w, col, a.K);
            w = t.v;
        }
        if (a.b) {
            Raw<float> t;
            load_piece(t, a.b, col, a.K);
            b = t.v;
        }
        f32x4 o;
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = ((v[i].get(j) - m0) - r) * rstd * w[j] + b[j];
        store_piece(y + col, o, a.K - col);
    }
}

// A lane's piece of a row for the gradient: W consecutive columns (4; 1 for rows of fewer than four), read without a branch
// so that the next row's pieces are on their way while this row's are worked on.
template <typename T, int W> struct Bits;
template <> struct Bits<float, 4> {
    f32x4 v;
    __device__ void load(const float* p) { v = *reinterpret_cast<const f32x4_4*>(p); }
    __device__ float get(int i) const { return v[i]; }
};
template <> struct Bits<uint16_t, 4> {
    u32x2 v;
    __device__ void load(const uint16_t* p) { v = *reinterpret_cast<const u32x2_2*>(p); }
    __device__ float get(int i) const { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
};
template <> struct Bits<Fp8, 4> {
    uint32_t v;
    __device__ void load(const Fp8* p) {
        typedef uint32_t u32_1 __attribute__((aligned(1)));
        v = *reinterpret_cast<const u32_1*>(p);
    }
    __device__ float get(int i) const {
        const f32x2 f = i & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false);
        return f[i & 1];
    }
};
template <> struct Bits<float, 1> {
    float v;
    __device__ void load(const float* p) { v = *p; }
    __device__ float get(int) const { return v; }
};
template <> struct Bits<uint16_t, 1> {
    uint32_t v;
    __device__ void load(const uint16_t* p) { v = *p; }
    __device__ float get(int) const { return __uint_as_float(v << 16); }
};
template <> struct Bits<Fp8, 1> {
    uint32_t v;
    __device__ void load(const Fp8* p) { v = p->v; }
    __device__ float get(int) const { return __builtin_amdgcn_cvt_f32_fp8((int)v, 0); }
};

// Rows in turn over the workgroups, WPR of the eight waves a row, R pieces a lane; the next row's loads are in flight over
// each row.  w stays in LDS: with two rows and the columns' sums in registers it would be the part that does not fit.
// A piece past the last column is read at the last whole one's place; its elements before `skip` belong to another lane.
template <typename TD, typename TX, int R, int WPR, int W>
__global__ __launch_bounds__(512, 2) void layer_norm_grad_kernel(NormGrad a) {
    constexpr int WAVES = 8, ROWS = WAVES / WPR, PIECES = 64 * W, COLS = WPR * R * PIECES;
    constexpr int BUFS = ROWS > 1 ? ROWS / 2 : 1;  // half of the rows' sums of columns at a time
    __shared__ float2 part[2][WAVES];
    __shared__ __align__(16) float ws[COLS];
    __shared__ __align__(16) float cols[ROWS > 1 ? BUFS * 2 * COLS : 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = wave / WPR, first = (wave % WPR) * (R * PIECES), col0 = first + lane * W;
    const float inv = 1.f / (float)a.K;
    for (int c = tid; c < COLS; c += 512) ws[c] = c >= a.K ? 0.f : a.w ? a.w[c] : 1.f;
    __syncthreads();
    struct Row {
        Bits<TD, W> d[R];
        Bits<TX, W> v[R];
        uint32_t word[R];
        float2 st;
    };
    auto place = [&](int i) __attribute__((always_inline)) { return min(col0 + i * PIECES, a.K - W); };
    auto load = [&](Row& r, int64_t row) __attribute__((always_inline)) {
        row = min(row, (int64_t)a.M - 1);
        const TD* dy = reinterpret_cast<const TD*>(a.dy) + row * a.lddy;
        const TX* x = reinterpret_cast<const TX*>(a.x) + row * a.ldx;
#pragma unroll
        for (int i = 0; i < R; i++) {
            r.d[i].load(dy + place(i));
            r.v[i].load(x + place(i));
            if constexpr (sizeof(TX) == 1) {  // a wave's piece lies in one word's 512 columns
                typedef const __attribute__((address_space(4))) uint32_t* constant_t;
                const int group = min(first + i * PIECES, a.K - 1) >> 9;
                r.word[i] = *((constant_t)a.xs + group * a.ld_xs + row);
            }
        }
        r.st = a.stats[row];
    };
    f32x4 dw[R], db[R];
#pragma unroll
    for (int i = 0; i < R; i++) dw[i] = db[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int turn = 0;
    auto work = [&](const Row& r, int64_t row) __attribute__((always_inline)) {
        float2* at = part[turn & 1] + sub * WPR;
        turn++;
        if (ROWS > 1 && row >= a.M) {
            float z0 = 0.f, z1 = 0.f;
            if constexpr (WPR > 1) row_sums<WPR>(z0, z1, at, wave % WPR);  // meets the barrier of the other rows' waves
            return;
        }
        float h[R][W], g[R][W];
        float sa = 0.f, sah = 0.f;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int col = col0 + i * PIECES, skip = col - place(i);
            float sc = 1.f;
            if constexpr (sizeof(TX) == 1) {
                const uint32_t b = r.word[i] >> (8 * ((min(col, a.K - 1) >> 7) & 3)) & 0xff;
                sc = __uint_as_float(b ? b << 23 : 0x400000u);  // 2^(b - 127)
            }
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float xv = sizeof(TX) == 1 ? r.v[i].get(j) * sc : r.v[i].get(j);
                h[i][j] = (xv - r.st.x) * r.st.y;
                g[i][j] = r.d[i].get(j);
                if (first + (i + 1) * PIECES > a.K && j < skip) h[i][j] = g[i][j] = 0.f;
                dw[i][j] += g[i][j] * h[i][j];
                db[i][j] += g[i][j];
                g[i][j] *= ws[place(i) + j];
                sa += g[i][j];
                sah += g[i][j] * h[i][j];
            }
        }
        row_sums<WPR>(sa, sah, at, wave % WPR);
        if (!a.dx) return;
        const float ma = sa * inv, mah = sah * inv;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int col = col0 + i * PIECES, at = place(i);
            f32x4 o;
#pragma unroll
            for (int j = 0; j < W; j++) o[j] = r.st.y * (g[i][j] - ma - h[i][j] * mah);
            if (W == 4 && col + W <= a.K) {
                if (a.dx_f32) store_piece(reinterpret_cast<float*>(a.dx) + row * a.lddx + col, o, 4);
                else store_piece(reinterpret_cast<uint16_t*>(a.dx) + row * a.lddx + col, o, 4);
            } else {
#pragma unroll
                for (int j = 0; j < W; j++) {
                    if (col >= a.K || at + j < col) continue;
                    if (a.dx_f32) reinterpret_cast<float*>(a.dx)[row * a.lddx + at + j] = o[j];
                    else reinterpret_cast<uint16_t*>(a.dx)[row * a.lddx + at + j] = (uint16_t)bf16x2_rne(o[j], o[j]);
                }
            }
        }
    };
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    if constexpr (R > 4) {  // the widest rows: one is all that registers hold
        for (int64_t row = row0; row < a.M; row += step) {
            Row r;
            load(r, row + sub);
            work(r, row + sub);
        }
    } else {
        Row r0, r1;
        load(r0, row0 + sub);
        for (int64_t row = row0; row < a.M; row += 2 * step) {
            load(r1, row + step + sub);
            work(r0, row + sub);
            if (row + step >= a.M) break;
            load(r0, row + 2 * step + sub);
            work(r1, row + step + sub);
        }
    }
    if (!a.part) return;
    // the rows' column sums: the upper half's to the lower half, and again
#pragma unroll
    for (int n = ROWS; n > 1; n >>= 1) {
        __syncthreads();
        float* at = cols + (sub % (n / 2)) * (2 * COLS) + (wave % WPR) * (R * PIECES);
        if (sub >= n / 2 && sub < n) {
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    at[i * PIECES + j * 64 + lane] = dw[i][j];
                    at[COLS + i * PIECES + j * 64 + lane] = db[i][j];
                }
        }
        __syncthreads();
        if (sub < n / 2) {
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < W; j++) {
                    dw[i][j] += at[i * PIECES + j * 64 + lane];
                    db[i][j] += at[COLS + i * PIECES + j * 64 + lane];
                }
        }
    }
    if (sub) return;
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.K;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int col = col0 + i * PIECES;
#pragma unroll
        for (int j = 0; j < W; j++)
            if (col < a.K && place(i) + j >= col) {
                out[place(i) + j] = dw[i][j];
                out[a.K + place(i) + j] = db[i][j];
            }
    }
}

// dw and db from the workgroups' partial sums: 64 of the 2 K columns a workgroup, a part of the rows each of its 16 waves.
__global__ __launch_bounds__(1024) void norm_params_kernel(const float* part, int groups, int K, float* dw, float* db) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (c < 2 * K) {
        const int per = (groups + 15) / 16, end = min((wave + 1) * per, groups);
#pragma unroll 8
        for (int g = wave * per; g < end; g++) s += part[(int64_t)g * 2 * K + c];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || c >= 2 * K) return;
#pragma unroll
    for (int w = 1; w < 16; w++) s += sums[w][lane];
    if (c < K) {
        if (dw) dw[c] = s;
    } else if (db) {
        db[c - K] = s;
    }
}

__global__ __launch_bounds__(256) void norm_zero_kernel(int K, float* dw, float* db) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= K) return;
    if (dw) dw[c] = 0.f;
    if (db) db[c] = 0.f;
}

template <typename TX, typename TY, int R, int WPR>
void fwd(const NormFwd& a, hipStream_t s) {
    // a dimension of a launch has fewer than 2^32 threads, which the most rows of four waves do not leave
    const unsigned n = (unsigned)((a.M + 4 / WPR - 1) / (4 / WPR)), y = (n + 65535) / 65536;
    hipLaunchKernelGGL((layer_norm_kernel<TX, TY, R, WPR>), dim3((n + y - 1) / y, y), dim3(256), 0, s, a);
}
// A wave a row as long as its pieces fit its registers (the least that hold them), four waves beyond
template <typename TX, typename TY>
void fwd_any(const NormFwd& a, hipStream_t s) {
    const int n = (a.K + STEP - 1) / STEP;  // pieces of a row, by 64 lanes
    if (n <= 2) fwd<TX, TY, 2, 1>(a, s);
    else if (n <= 4) fwd<TX, TY, 4, 1>(a, s);
    else if (n <= 6) fwd<TX, TY, 6, 1>(a, s);
    else if (n <= 8) fwd<TX, TY, 8, 1>(a, s);
    else if (n <= 10) fwd<TX, TY, 10, 1>(a, s);
    else if (n <= 12) fwd<TX, TY, 12, 1>(a, s);
    else if (n <= 16) fwd<TX, TY, 16, 1>(a, s);
    else if (n <= 32) fwd<TX, TY, 8, 4>(a, s);
    else fwd<TX, TY, 16, 4>(a, s);
}

template <typename TD, typename TX, int R, int WPR, int W = 4>
void grad(const NormGrad& a, hipStream_t s) {
    hipLaunchKernelGGL((layer_norm_grad_kernel<TD, TX, R, WPR, W>), dim3((unsigned)a.groups), dim3(512), 0, s, a);
}
// As many waves a row as leave each at most four pieces (12 columns' sums and two rows of them in registers): 2560 columns
// with two waves of five, one row at a time, took 33 us at 5498 rows, with four waves of three and the next row ahead 24.
template <typename TD, typename TX>
void grad_any(const NormGrad& a, hipStream_t s) {
    const int n = (a.K + STEP - 1) / STEP;
    if (a.K < 4) grad<TD, TX, 1, 1, 1>(a, s);
    else if (n <= 2) grad<TD, TX, 2, 1>(a, s);
    else if (n <= 4) grad<TD, TX, 4, 1>(a, s);
    else if (n <= 6) grad<TD, TX, 3, 2>(a, s);
    else if (n <= 8) grad<TD, TX, 4, 2>(a, s);
    else if (n <= 12) grad<TD, TX, 3, 4>(a, s);
    else if (n <= 16) grad<TD, TX, 4, 4>(a, s);
    else if (n <= 24) grad<TD, TX, 3, 8>(a, s);
    else if (n <= 32) grad<TD, TX, 4, 8>(a, s);
    else if (n <= 48) grad<TD, TX, 6, 8>(a, s);
    else grad<TD, TX, 8, 8>(a, s);
}
template <typename TD>
void grad_in(int dtype_x, const NormGrad& a, hipStream_t s) {
    if (dtype_x == AWA_F32) grad_any<TD, float>(a, s);
    else if (dtype_x == AWA_BF16) grad_any<TD, uint16_t>(a, s);
    else grad_any<TD, Fp8>(a, s);
}

// rows that a workgroup of the gradient takes at once
int rows_at_once(int K) {
    const int n = (K + STEP - 1) / STEP;
    return n <= 4 ? 8 : n <= 8 ? 4 : n <= 16 ? 2 : 1;
}

}  // namespace

int norm_grad_groups(int M, int K) {
    const int rows = rows_at_once(K);
    return std::min((M + rows - 1) / rows, 256);
}

hipError_t launch_layer_norm(int dtype_x, int dtype_y, const NormFwd& a, hipStream_t s) {
    if (dtype_x == AWA_F32) {
        if (dtype_y == AWA_F32) fwd_any<float, float>(a, s);
        else fwd_any<float, uint16_t>(a, s);
    } else {
        if (dtype_y == AWA_F32) fwd_any<uint16_t, float>(a, s);
        else fwd_any<uint16_t, uint16_t>(a, s);
    }
    return hipGetLastError();
}

hipError_t launch_layer_norm_grad(int dtype_dy, int dtype_x, const NormGrad& a, hipStream_t s) {
    if (a.M == 0) {
        hipLaunchKernelGGL(norm_zero_kernel, dim3((unsigned)((a.K + 255) / 256)), dim3(256), 0, s, a.K, a.dw, a.db);
        return hipGetLastError();
    }
    if (dtype_dy == AWA_F32) grad_in<float>(dtype_x, a, s);
    else grad_in<uint16_t>(dtype_x, a, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.part) return e;
    hipLaunchKernelGGL(norm_params_kernel, dim3((unsigned)((2 * a.K + 63) / 64)), dim3(1024), 0, s, a.part, a.groups, a.K, a.dw, a.db);
    return hipGetLastError();
}

}  // namespace awa
