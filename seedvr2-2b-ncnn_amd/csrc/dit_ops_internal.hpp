// dit_ops_internal.hpp — shared definitions of the operators of dit_ops.h.
#pragma once

#include "dit_internal.hpp"
#include "dit_ops.h"

namespace awa {

struct QuantArgs {
    const void* x;       // [M][K], ldx elements apart
    int64_t ldx;
    int M, K, kp;        // kp: K rounded up to whole blocks
    uint8_t* q;          // [M][kp]
    uint32_t* scale;     // [groups][ld_scale] words
    int64_t ld_scale;
};
hipError_t launch_quant_rows(int dtype, const QuantArgs& a, hipStream_t s);
hipError_t launch_quant_blocks(int dtype, const QuantArgs& a, hipStream_t s);

struct Fp8Gemm {
    const uint8_t* A;    // [M][K] e4m3
    const uint32_t* as;  // [groups][ld_as] words
    int64_t ld_as;
    const uint8_t* W;    // [N][K]
    const uint32_t* ws;  // [groups][ld_ws], a word per 128 rows
    int64_t ld_ws;
    const float* bias;   // [N] or null
    void* C;
    int64_t ldc;
    int M, N, K;
    int c_f32;           // C fp32, else bf16
    int whole;           // bf16 C: every product enters the sums whole
    int c_vec;           // C's rows allow 16-byte stores
    int n_tiles, m_tiles;
};
hipError_t launch_gemm_fp8(Fp8Gemm& p, hipStream_t s);

struct RopeArgs {
    const void* x[2];
    void* out[2];
    int64_t x_token[2], x_head[2], out_token[2], out_head[2];
    int heads[2];
    int tokens, head_d;
    int pairs;               // rotated pairs, all axes
    int axes, axis_end[DIT_ROPE_MAX_AXES];  // pairs up to each axis's end
    int copy;                // channels past the pairs go from x to out (not in place)
    int rot_units, units;    // pieces of a head that turn, and all; filled by launch_rope
    int lanes[2];            // threads per token and piece, each with every lanes-th head; likewise
    const int32_t* pos;
    double cos_scale, sin_scale;
    double quarters[DIT_ROPE_MAX_PAIRS];  // quarter turns per position
};
hipError_t launch_rope(int dtype, int layout, RopeArgs& a, hipStream_t s);

}  // namespace awa
