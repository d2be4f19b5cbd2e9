// dit_rope.hip — rotary positions on rows of heads.
//
// A thread owns a piece of the head (V pairs, so that what it loads is 16 bytes)
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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
    static __device__ inline uint16_t put(float v) { return (uint16_t)bf16x2_rne(v, v); }
};
template <> struct Chan<float> {
    static __device__ inline float get(float v) { return v; }
    static __device__ inline float put(float v) { return v; }
};

template <typename T, int LAYOUT, bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    constexpr int CH = VEC ? 16 / sizeof(T) : 1;            // channels per load
    constexpr int V = LAYOUT == DIT_ROPE_HALF ? CH : VEC ? CH / 2 : 1;  // pairs per unit
    constexpr int CW = LAYOUT == DIT_ROPE_HALF ? V : 2 * V;  // channels of a unit that only passes
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    const uint32_t tok = item / (uint32_t)a.units;
    if (tok >= (uint32_t)a.tokens) return;
    const int u = (int)(item - tok * (uint32_t)a.units);
    const int h0 = blockIdx.y * a.heads_per_block, h1 = min(h0 + a.heads_per_block, a.heads);
    const bool turns = u < a.rot_units;
    float c[V], s[V];
    if (turns) {
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
    }
    const int pass0 = LAYOUT == DIT_ROPE_HALF ? 2 * a.pairs : 2 * V * a.rot_units;
    const int ch0 = turns ? (LAYOUT == DIT_ROPE_HALF ? u * V : 2 * u * V) : pass0 + (u - a.rot_units) * CW;
    for (int h = h0; h < h1; h++) {
        const int t = h >= a.heads0, hh = h - (t ? a.heads0 : 0);
        const T* x = reinterpret_cast<const T*>(a.x[t]) + tok * a.x_token[t] + hh * a.x_head[t] + ch0;
        T* o = reinterpret_cast<T*>(a.out[t]) + tok * a.out_token[t] + hh * a.out_head[t] + ch0;
        if (!turns) {
#pragma unroll
            for (int i = 0; i < CW; i++)
                if (ch0 + i < a.head_d) o[i] = x[i];
        } else {
            constexpr int STEP = LAYOUT == DIT_ROPE_HALF ? 1 : 2;
            const int second = LAYOUT == DIT_ROPE_HALF ? a.pairs : 1;
            T lo[V], hi[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                lo[j] = x[STEP * j];
                hi[j] = x[STEP * j + second];
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float p = Chan<T>::get(lo[j]), r = Chan<T>::get(hi[j]);
                o[STEP * j] = Chan<T>::put(p * c[j] - r * s[j]);
                o[STEP * j + second] = Chan<T>::put(p * s[j] + r * c[j]);
            }
        }
    }
}

template <typename T, int LAYOUT, bool VEC>
void launch(RopeArgs& a, hipStream_t s) {
    constexpr int CH = VEC ? 16 / sizeof(T) : 1;
    constexpr int V = LAYOUT == DIT_ROPE_HALF ? CH : VEC ? CH / 2 : 1;
    constexpr int CW = LAYOUT == DIT_ROPE_HALF ? V : 2 * V;
    a.rot_units = (a.pairs + V - 1) / V;
    const int pass0 = LAYOUT == DIT_ROPE_HALF ? 2 * a.pairs : 2 * V * a.rot_units;
    a.units = a.rot_units + (a.copy && a.head_d > pass0 ? (a.head_d - pass0 + CW - 1) / CW : 0);
    if (a.units == 0) return;
    const unsigned blocks = (unsigned)(((int64_t)a.tokens * a.units + 255) / 256);
    a.heads_per_block = 8;
    hipLaunchKernelGGL((rope_kernel<T, LAYOUT, VEC>), dim3(blocks, (a.heads + 7) / 8), dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_rope(int dtype, int layout, RopeArgs& a, hipStream_t s) {
    if (dtype == AWA_F32) {
        if (layout == DIT_ROPE_HALF) launch<float, DIT_ROPE_HALF, false>(a, s);
        else launch<float, DIT_ROPE_INTERLEAVED, false>(a, s);
    } else {
        if (layout == DIT_ROPE_HALF) launch<uint16_t, DIT_ROPE_HALF, false>(a, s);
        else launch<uint16_t, DIT_ROPE_INTERLEAVED, false>(a, s);
    }
    return hipGetLastError();
}

}  // namespace awa
