// dit_rope.hip — rotary positions on rows of heads.
//
// A thread owns a piece of the head (V pairs, 16 bytes a load where the sizes allow)
// of one token: it forms the V sines and cosines once and turns that piece of
// every head of its part.  HBM-bound: each channel is read and written once: 5440 x 40 x
// 128 bf16 inside rows of 7680 19.2 us (5.8 TB/s), 20000 x 12 x 96 fp32 30 (6.2; 35 with other
// tensors each time), 4096 x 40 x 128 fp32 26.1 (6.4); one token of 40 heads 3.3 us.
//
// Angles: position times quarter turns per position in fp64, less the nearest whole
// number of quarters (exact): far positions lose only what fp64 loses on the angle
// (2^-21 at a position of 2^31 and one radian a step).  Sine and cosine of the rest by
// their Taylor series, cut where the next term is below 2^-28.  For fp32 channels its first
// two terms and the factor are fp64, so that what a channel is multiplied with is rounded
// once (all in fp32, the roundings of the rest, of pi / 2 and of the factor made results of
// 20000 x 12 x 96 4.4e-8 of their size off, so 3.6e-8; 60000 x 64 in one head 7.1 us for
// 6.7).  For bf16 channels, whose step is 2^16 times theirs, they are fp32 (60000 x 128 in
// two heads 10.6 us, with fp64 12.0).
#include "dit_ops_internal.hpp"

namespace awa {

namespace {

struct CosSin {
    float c, s;
};
// cosine and sine of that many quarter turns, times the factors
template <typename T>
__device__ inline CosSin cos_sin(double quarters, double cos_scale, double sin_scale) {
    // 1.5 2^52 more leaves the nearest integer in the low bits (|quarters| < 2^51)
    constexpr double BIG = 6755399441055744.0;
    const double n = quarters + BIG;
    const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, n);
    // quarter 0: (c, s)  1: (-s, c)  2: (-c, -s)  3: (s, -c)
    const bool odd = k & 1;
    float c, s;
    if constexpr (sizeof(T) == 4) {
        const double x = (quarters - (n - BIG)) * (0.5 * M_PI), z = x * x;  // at most pi / 4
        const float xf = (float)x, zf = xf * xf, zz = zf * zf;
        const float st = xf * zz * (1.f / 120 + zf * (-1.f / 5040 + zf * (1.f / 362880)));
        const float ct = zz * (1.f / 24 + zf * (-1.f / 720 + zf * (1.f / 40320 + zf * (-1.f / 3628800))));
        const double sd = x * (1.0 - z * (1.0 / 6)) + (double)st, cd = (1.0 - 0.5 * z) + (double)ct;
        c = (float)(cos_scale * (odd ? sd : cd));
        s = (float)(sin_scale * (odd ? cd : sd));
    } else {
        const float x = (float)(quarters - (n - BIG)) * 1.57079632679489662f;
        const float z = x * x;
        const float sf = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
        const float cf = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
        c = (odd ? sf : cf) * (float)cos_scale;
        s = (odd ? cf : sf) * (float)sin_scale;
    }
    return {__uint_as_float(__float_as_uint(c) ^ ((k + 1) & 2) << 30), __uint_as_float(__float_as_uint(s) ^ (k & 2) << 30)};
}

template <typename T> struct Chan;
template <> struct Chan<uint16_t> {
    static __device__ inline float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ inline void put(uint16_t* to, float a, float b) {
        const uint32_t u = bf16x2_rne(a, b);
        to[0] = (uint16_t)u;
        to[1] = (uint16_t)(u >> 16);
    }
};
template <> struct Chan<float> {
    static __device__ inline float get(float v) { return v; }
    static __device__ inline void put(float* to, float a, float b) {
        to[0] = a;
        to[1] = b;
    }
};

// N channels that are only known to be aligned to one.  Stores of 16 bytes go past the
// caches (5440 x 40 x 128 bf16 25.9 -> 18.9 us).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    T v[N];
    __device__ inline void store(T* to) const {
        if constexpr (N * sizeof(T) == 16) {
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            typedef uint32_t u32x4_t __attribute__((ext_vector_type(4), aligned(2)));
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, *this), reinterpret_cast<u32x4_t*>(to));
        } else {
            *reinterpret_cast<Piece*>(to) = *this;
        }
    }
};

// V pairs per thread: interleaved 2 V neighbouring channels, half V and V.  Channels
// that only pass go in pieces of as many.  Neighbouring threads take the pieces of a
// head, then of the next heads of the token; grid.y is the tensor.
template <typename T, int LAYOUT, int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    constexpr bool HALF = LAYOUT == DIT_ROPE_HALF;
    constexpr int W = HALF ? V : 2 * V;  // channels per load
    using P = Piece<T, W>;
    const int t = blockIdx.y, heads = a.heads[t], step = a.lanes[t];
    const uint32_t item = blockIdx.x * 256u + threadIdx.x, part = item / (uint32_t)a.units;
    const int u = (int)(item - part * (uint32_t)a.units);
    const uint32_t tok = part / (uint32_t)step;
    if (tok >= (uint32_t)a.tokens) return;
    const int h0 = (int)(part - tok * (uint32_t)step);
    const bool turns = u < a.rot_units;
    const int ch = turns ? u * W : (HALF ? 2 * a.pairs : W * a.rot_units) + (u - a.rot_units) * W;
    const T* x = reinterpret_cast<const T*>(a.x[t]) + tok * a.x_token[t] + h0 * a.x_head[t] + ch;
    T* o = reinterpret_cast<T*>(a.out[t]) + tok * a.out_token[t] + h0 * a.out_head[t] + ch;
    const int64_t xs = step * a.x_head[t], os = step * a.out_head[t];
    if (!turns) {
        for (int h = h0; h < heads; h += step, x += xs, o += os) {
            if (V > 1 || ch + W <= a.head_d) reinterpret_cast<const P*>(x)->store(o);
            else *o = *x;  // the last of an odd number
        }
        return;
    }
    const int second = HALF ? a.pairs : 0;  // from a pair's first piece to its second
    // heads in flight: 64 bytes a thread (half, 5440 x 40 x 128 bf16: two 21.1 us, four 21.6)
    constexpr int R = HALF && V == 8 ? 2 : 4;
    P f[R], g[R];
    auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; r++, x += xs)
            if (h + r * step < heads) {
                f[r] = *reinterpret_cast<const P*>(x);
                if (HALF) g[r] = *reinterpret_cast<const P*>(x + second);
            }
    };
    load(h0);  // on their way while the angles are formed
    float c[V], s[V];
    const int32_t* pos = a.pos + (int64_t)tok * a.axes;
    const int32_t pos0 = pos[0];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int p = u * V + j;
        c[j] = 1.f;
        s[j] = 0.f;
        if (p < a.pairs) {
            int32_t at = pos0;
            if (a.axes > 1) {
                int axis = 0;
#pragma unroll
                for (int k = 0; k + 1 < DIT_ROPE_MAX_AXES; k++) axis += p >= a.axis_end[k];
                at = pos[axis];
            }
            const CosSin v = cos_sin<T>((double)at * a.quarters[p], a.cos_scale, a.sin_scale);
            c[j] = v.c;
            s[j] = v.s;
        }
    }
    for (int h = h0; h < heads; h += R * step) {
#pragma unroll
        for (int r = 0; r < R; r++, o += os) {
            if (h + r * step >= heads) continue;
            if constexpr (HALF) {
                P p, q;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float m = Chan<T>::get(f[r].v[j]), n = Chan<T>::get(g[r].v[j]);
                    T y[2];
                    Chan<T>::put(y, m * c[j] - n * s[j], m * s[j] + n * c[j]);
                    p.v[j] = y[0];
                    q.v[j] = y[1];
                }
                p.store(o);
                q.store(o + second);
            } else {
                P p;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float m = Chan<T>::get(f[r].v[2 * j]), n = Chan<T>::get(f[r].v[2 * j + 1]);
                    Chan<T>::put(p.v + 2 * j, m * c[j] - n * s[j], m * s[j] + n * c[j]);
                    if (V > 1 && u * V + j >= a.pairs) {  // channels that only pass, as they are (also infinities)
                        p.v[2 * j] = f[r].v[2 * j];
                        p.v[2 * j + 1] = f[r].v[2 * j + 1];
                    }
                }
                p.store(o);
            }
        }
        if (h + R * step < heads) load(h + R * step);
    }
}

template <typename T, int LAYOUT, int V>
void launch(RopeArgs& a, hipStream_t s) {
    constexpr bool HALF = LAYOUT == DIT_ROPE_HALF;
    constexpr int W = HALF ? V : 2 * V;
    a.rot_units = (a.pairs + V - 1) / V;
    const int pass0 = HALF ? 2 * a.pairs : W * a.rot_units;
    a.units = a.rot_units + (a.copy && a.head_d > pass0 ? (a.head_d - pass0 + W - 1) / W : 0);
    if (a.units == 0) return;
    // sines and cosines serve as many heads as leave 2048 workgroups (8 per CU) and fewer
    // than 2^32 threads
    const int64_t one = (int64_t)a.tokens * a.units;  // threads if each took every head
    int64_t threads = 0;
    for (int t = 0; t < 2; t++) {
        const int64_t lanes = (2048 * 256 + one - 1) / one;
        a.lanes[t] = (int)(lanes < a.heads[t] ? lanes : a.heads[t] > 1 ? a.heads[t] : 1);
        const int64_t n = one * a.lanes[t];
        threads = n > threads ? n : threads;
    }
    hipLaunchKernelGGL((rope_kernel<T, LAYOUT, V>), dim3((unsigned)((threads + 255) / 256), a.heads[1] ? 2 : 1),
                       dim3(256), 0, s, a);
}

// the widest piece (up to 16 bytes) that the pairs and the head are whole numbers of
template <typename T, int LAYOUT, int V>
void pick(RopeArgs& a, hipStream_t s) {
    if constexpr (V > 1) {
        const bool fits = LAYOUT == DIT_ROPE_HALF ? a.pairs % V == 0 && a.head_d % V == 0 : a.head_d % (2 * V) == 0;
        if (!fits) return pick<T, LAYOUT, V / 2>(a, s);
    }
    launch<T, LAYOUT, V>(a, s);
}

}  // namespace

hipError_t launch_rope(int dtype, int layout, RopeArgs& a, hipStream_t s) {
    if (dtype == AWA_F32) {
        if (layout == DIT_ROPE_HALF) pick<float, DIT_ROPE_HALF, 4>(a, s);
        else pick<float, DIT_ROPE_INTERLEAVED, 2>(a, s);
    } else {
        if (layout == DIT_ROPE_HALF) pick<uint16_t, DIT_ROPE_HALF, 8>(a, s);
        else pick<uint16_t, DIT_ROPE_INTERLEAVED, 4>(a, s);
    }
    return hipGetLastError();
}

}  // namespace awa
