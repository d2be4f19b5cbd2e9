// dit_rope.hip — rotary positions on rows of heads.
//
// A thread owns a piece of the head (V pairs, 16 bytes a load where the sizes allow)
// of one token: it forms the V sines and cosines once and turns that piece of
// every head of its part.  HBM-bound: each channel is read and written once.
//
// Angles: position times turns per position in fp64, less the nearest whole
// turn (exact), then less the nearest quarter (exact): what is left, at most an
// eighth of a turn, is rounded to fp32 once, so far positions lose only what
// fp64 loses on the angle (2^-21 at a position of 2^31 and one radian a step).
// Sine and cosine of the rest by their Taylor series, cut where the next term is
// below 2^-28.
#include "dit_ops_internal.hpp"

namespace awa {

namespace {

struct CosSin {
    float c, s;
};
__device__ inline CosSin cos_sin(double turns) {
    turns -= __builtin_rint(turns);
    const double q4 = 4.0 * turns, n = __builtin_rint(q4);
    const int quarter = (int)n;                          // -2 .. 2
    const float x = (float)(q4 - n) * 1.57079632679489662f;  // at most pi / 4
    const float z = x * x;
    const float s = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
    const bool odd = quarter & 1;
    const float cc = odd ? s : c, ss = odd ? c : s;      // up to signs
    // quarter 0: (c, s)  1: (-s, c)  2, -2: (-c, -s)  -1: (s, -c)
    return {quarter == 1 || (quarter & 3) == 2 ? -cc : cc, quarter < 0 || quarter == 2 ? -ss : ss};
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

// N channels that are only known to be aligned to one
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    T v[N];
};

// V pairs per thread: interleaved 2 V neighbouring channels, half V and V.  Channels
// that only pass go in pieces of as many.
template <typename T, int LAYOUT, int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    constexpr bool HALF = LAYOUT == DIT_ROPE_HALF;
    constexpr int W = HALF ? V : 2 * V;  // channels per load
    using P = Piece<T, W>;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    const uint32_t tok = item / (uint32_t)a.units;
    if (tok >= (uint32_t)a.tokens) return;
    const int u = (int)(item - tok * (uint32_t)a.units);
    const int h0 = blockIdx.y * a.heads_per_block, h1 = min(h0 + a.heads_per_block, a.heads);
    const bool turns = u < a.rot_units;
    const int ch = turns ? u * W : (HALF ? 2 * a.pairs : W * a.rot_units) + (u - a.rot_units) * W;
    auto from = [&](int h) __attribute__((always_inline)) {
        const int t = h >= a.heads0, hh = h - (t ? a.heads0 : 0);
        return reinterpret_cast<const T*>(a.x[t]) + hh * a.x_head[t] + tok * a.x_token[t] + ch;
    };
    auto to = [&](int h) __attribute__((always_inline)) {
        const int t = h >= a.heads0, hh = h - (t ? a.heads0 : 0);
        return reinterpret_cast<T*>(a.out[t]) + hh * a.out_head[t] + tok * a.out_token[t] + ch;
    };
    if (!turns) {
        for (int h = h0; h < h1; h++) {
            if (V > 1 || ch + W <= a.head_d) *reinterpret_cast<P*>(to(h)) = *reinterpret_cast<const P*>(from(h));
            else *to(h) = *from(h);  // the last of an odd number
        }
        return;
    }
    const int second = HALF ? a.pairs : 0;  // from a pair's first piece to its second
    constexpr int R = 4;                    // heads in flight
    P x[R], y[R];
    auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; r++)
            if (h + r < h1) {
                const T* f = from(h + r);
                x[r] = *reinterpret_cast<const P*>(f);
                if (HALF) y[r] = *reinterpret_cast<const P*>(f + second);
            }
    };
    load(h0);  // on their way while the angles are formed
    float c[V], s[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int p = u * V + j;
        c[j] = 1.f;
        s[j] = 0.f;
        if (p < a.pairs) {
            int axis = 0;
#pragma unroll
            for (int k = 0; k + 1 < DIT_ROPE_MAX_AXES; k++) axis += p >= a.axis_end[k];
            const CosSin v = cos_sin((double)a.pos[(int64_t)tok * a.axes + axis] * a.turns[p]);
            c[j] = v.c * a.cos_scale;
            s[j] = v.s * a.sin_scale;
        }
    }
    for (int h = h0; h < h1; h += R) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (h + r >= h1) continue;
            T* o = to(h + r);
            if constexpr (HALF) {
                P p, q;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float f = Chan<T>::get(x[r].v[j]), g = Chan<T>::get(y[r].v[j]);
                    T t[2];
                    Chan<T>::put(t, f * c[j] - g * s[j], f * s[j] + g * c[j]);
                    p.v[j] = t[0];
                    q.v[j] = t[1];
                }
                *reinterpret_cast<P*>(o) = p;
                *reinterpret_cast<P*>(o + second) = q;
            } else {
                P p;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float f = Chan<T>::get(x[r].v[2 * j]), g = Chan<T>::get(x[r].v[2 * j + 1]);
                    Chan<T>::put(p.v + 2 * j, f * c[j] - g * s[j], f * s[j] + g * c[j]);
                }
                *reinterpret_cast<P*>(o) = p;
            }
        }
        if (h + R < h1) load(h + R);
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
    const int64_t blocks = ((int64_t)a.tokens * a.units + 255) / 256;
    // sines and cosines serve as many heads as leave 2048 workgroups (8 per CU)
    const int64_t per = blocks * a.heads / 2048;
    a.heads_per_block = (int)(per < 1 ? 1 : per > a.heads ? a.heads : per);
    const unsigned parts = (a.heads + a.heads_per_block - 1) / a.heads_per_block;
    hipLaunchKernelGGL((rope_kernel<T, LAYOUT, V>), dim3((unsigned)blocks, parts), dim3(256), 0, s, a);
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
