// dit_cross.hip — attention to states of another length: the forward pass and the gradient of the queries.
//
// A workgroup takes a block of columns (queries of one head, or of the heads that share a key head: see
// CrossItem) over a run of keys.  Scores are formed transposed, S^T = K Q^T, so that a lane owns one column: its
// softmax needs two lane exchanges a tile, and the probabilities leave the accumulator as the operand of
// O^T += V^T P^T (dit_cross_device.hpp).  Keys and values reach LDS by DMA, the next tile's during this one's
// products; masked keys and rows past the end are fetched from past the buffer and so become zeros, whatever memory
// holds there, and their scores -infinity.  The gradient of the queries is the same walk with P from the kept
// lse: dP^T = V dO^T, dS = P (dP - D), dQ^T += K^T dS^T.
//
// Two shapes: blocks of 128 columns, four waves of 32 that share the tiles; and for few columns (tokens being
// generated) blocks of 16 or 32, waves that take tiles of their own in turn and add their results in LDS.
// Runs of keys of one block that go to different workgroups leave fp32 partial results, which a second kernel joins.
//
// In blocks of 128 a wave's 32 columns make as many cycles of LDS reads as of products, and half as many of the softmax's VALU
// instructions (51 % issue), which bounds them, two waves a SIMD filling each other's waits: 27200 queries x 1024 keys x 20 heads of 128
// 311 us (0.92 PFLOP/s; 48 columns a wave, which spills, 320; 16 425), 16384 x 384 83 (0.78).  With up to 64 keys one tile is all:
// half the LDS, no second maximum, four workgroups a CU (5440 x 58 16.6 -> 14.9 us, 16384 x 64 32.5).  Few columns are bound by
// the keys' bytes: 32 tokens x 1500 keys, 20 heads on 4, 23 us (4.3 TB/s; in blocks of 128 91), 64 x 2048, 32 on 8, 97 (5.5).  fp32
// by its matrix rate: 5440 x 512 x 20 heads 311 us (92 TFLOP/s).
#include "dit_cross_device.hpp"

namespace awa {

using namespace cross;

namespace {

template <typename T, int DP, int NQ, int WQ, int WK, int KT, bool GRAD, bool ONE>
__global__ __launch_bounds__(64 * WQ * WK, (T::SIZE == 2 && WK == 1 ? (ONE && !(GRAD && T::WHOLE) ? 3 : 2) : 1)) void cross_queries_kernel(CrossArgs p) {
    using Frag = typename T::Frag;
    using L = Tile<T, DP>;
    constexpr int KS = DP / 32, DB = DP / 16, KB = KT / 16, WAVES = WQ * WK;
    constexpr int TILE_B = KT * L::ROW, STAGE = 2 * TILE_B;  // K, then V
    constexpr int JOIN = WK > 1 ? WAVES * NQ * 16 * (DP + 2) * 4 : 0;
    constexpr int RING = WK * (ONE ? 1 : 2) * STAGE, LDS = RING > JOIN ? RING : JOIN;
    static_assert(LDS <= 160 * 1024 && (WQ == 1 || WK == 1), "LDS");
    __shared__ __align__(16) char lds[LDS];
    const int groups = p.heads / p.qs.pack;
    CrossItem it;
    int hb;
    if (p.qs.n_listed) {
        it = table_entry(p.qs.items, (int)blockIdx.x);
        if (it.cols == 0) return;
        hb = it.group;
    } else {
        const int total = p.qs.n_items * groups, wg = xcd_remap(total);
        if (wg >= total) return;
        hb = wg / p.qs.n_items;
        it = table_entry(p.qs.items, wg - hb * p.qs.n_items);
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wq = wave % WQ, wk = wave / WQ, g = lane >> 4;
    const int head0 = hb * p.qs.pack, kv_head = head0 / (p.heads / p.kv_heads);
    const int width = p.head_d * T::SIZE;

    const int tiles = (it.kn + KT - 1) / KT;
    const uint8_t* mask = p.mask ? p.mask + it.k0 : nullptr;
    auto mask_byte = [&](int t) __attribute__((always_inline)) {
        const int key = t * KT + lane;
        return mask && lane < KT && key < it.kn ? (int)mask[key] : 1;
    };
    auto valid_of = [&](int t, int byte) __attribute__((always_inline)) {
        return __builtin_amdgcn_ballot_w64(lane < KT && t * KT + lane < it.kn && byte);
    };
    char* ring = lds + wk * (ONE ? 1 : 2) * STAGE;
    auto fetch = [&](int t, int slot, uint64_t valid) __attribute__((always_inline)) {
        const int64_t first = it.k0 + (int64_t)t * KT;
        const __amdgpu_buffer_rsrc_t kr = uniform_rsrc(p.k + kv_head * p.k_head + first * p.k_row, 0x7fffffffu);
        const __amdgpu_buffer_rsrc_t vr = uniform_rsrc(p.v + kv_head * p.v_head + first * p.v_row, 0x7fffffffu);
        char* st = ring + slot * STAGE;
        constexpr int N = TILE_B / 1024;
#pragma unroll
        for (int i = 0; i < N / WQ; i++) {
            L::dma(st, wq * (N / WQ) + i, kr, p.k_row, valid, width, lane);
            L::dma(st + TILE_B, wq * (N / WQ) + i, vr, p.v_row, valid, width, lane);
        }
    };
    // the first tile is on its way before the queries are asked for
    uint64_t valid = 0;
    int byte = 1;
    if (wk < tiles) {
        valid = valid_of(wk, mask_byte(wk));
        byte = mask_byte(wk + WK);
        fetch(wk, 0, valid);
    }
    // the wave's columns
    int row[NQ], head[NQ];
    bool there[NQ];
    Frag q[NQ][KS], dout[GRAD ? NQ : 1][KS];
    float lse2[NQ], dsum[NQ];  // GRAD: lse in powers of two, rowsum(dout out)
#pragma unroll
    for (int j = 0; j < NQ; j++) {
        const int c = (wq * NQ + j) * 16 + (lane & 15);
        there[j] = c < it.cols;
        row[j] = it.q0 + c;
        head[j] = head0;
        if constexpr (WQ == 1) {  // heads that share their keys
            row[j] = it.q0 + c / p.qs.pack;
            head[j] = head0 + c % p.qs.pack;
        }
        lse2[j] = dsum[j] = 0.f;
        // One head's rows: columns and channels that are not there lie past resources, without branches (16384 queries x 64
        // keys: gradients 112 us with them, 109 so; the forward pass, which loads a third, gains nothing).
        if constexpr (WQ > 1 && GRAD) {
            const __amdgpu_buffer_rsrc_t qr = uniform_rsrc(p.q + it.q0 * p.q_row + head0 * p.q_head, 0x7fffffffu);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d = 32 * ks + 8 * g;
                const bool in = there[j] && d < p.head_d;
                q[j][ks] = buffer_frag<T>(qr, in ? (uint32_t)c * (uint32_t)p.q_row + d * T::SIZE : 0x80000000u);
            }
            const __amdgpu_buffer_rsrc_t dr = uniform_rsrc(p.dout + it.q0 * p.dout_row + head0 * p.dout_head, 0x7fffffffu);
            const __amdgpu_buffer_rsrc_t orr = uniform_rsrc(p.out + it.q0 * p.out_row + head0 * p.out_head, 0x7fffffffu);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d = 32 * ks + 8 * g;
                const bool in = there[j] && d < p.head_d;
                dout[j][ks] = buffer_frag<T>(dr, in ? (uint32_t)c * (uint32_t)p.dout_row + d * T::SIZE : 0x80000000u);
                dsum[j] += T::dot(dout[j][ks], buffer_frag<T>(orr, in ? (uint32_t)c * (uint32_t)p.out_row + d * T::SIZE : 0x80000000u));
            }
        } else {
            const char* at = p.q + row[j] * p.q_row + head[j] * p.q_head;
            const char* dat = p.dout + row[j] * p.dout_row + head[j] * p.dout_head;
            const char* oat = p.out + row[j] * p.out_row + head[j] * p.out_head;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int d = 32 * ks + 8 * g;
                const bool in = there[j] && d < p.head_d;
                q[j][ks] = T::zero();
                if (in) q[j][ks] = T::load(at + d * T::SIZE);
                if constexpr (GRAD) {
                    dout[j][ks] = T::zero();
                    if (in) {
                        dout[j][ks] = T::load(dat + d * T::SIZE);
                        dsum[j] += T::dot(dout[j][ks], T::load(oat + d * T::SIZE));
                    }
                }
            }
        }
        if constexpr (GRAD) {
            dsum[j] = sum4(dsum[j]);
            if (there[j]) {
                const float l = p.lse[head[j] * p.ld_lse + row[j]];
                lse2[j] = l * LOG2E;
                if (l == -INFINITY) {  // a row without scores: P = 0, and nothing that comes back counts
                    lse2[j] = INFINITY;
                    dsum[j] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) dout[j][ks] = T::zero();
                }
                if (it.first && wk == 0 && g == 0) {
                    p.dsum[head[j] * p.ld_dsum + row[j]] = dsum[j];
                    p.lse2[head[j] * p.ld_dsum + row[j]] = lse2[j];
                }
            }
        }
    }

    f32x4 acc[DB][NQ];
    float top[NQ], sum[NQ];
#pragma unroll
    for (int j = 0; j < NQ; j++) {
        top[j] = -INFINITY;
        sum[j] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; db++) acc[db][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    int slot = 0;
    for (int t = wk; t < tiles; t += WK, slot ^= 1) {
        wait_vmem_lds<0>();  // this tile has landed (and what was read of the other slot has arrived)
        if constexpr (WQ > 1) __syncthreads();
        const uint64_t next = valid_of(t + WK, byte);
        byte = mask_byte(t + 2 * WK);
        if (!ONE && t + WK < tiles) fetch(t + WK, slot ^ 1, next);
        const char* kt = ring + slot * STAGE;
        const char* vt = kt + TILE_B;

        f32x4 s[KB][NQ], dp[GRAD ? KB : 1][NQ];
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const Frag kf = L::row_frag(kt, 16 * b + (lane & 15), ks, g);
#pragma unroll
                for (int j = 0; j < NQ; j++) s[b][j] = T::mma(kf, q[j][ks], ks ? s[b][j] : (f32x4){0.f, 0.f, 0.f, 0.f});
                if constexpr (GRAD) {
                    const Frag vf = L::row_frag(vt, 16 * b + (lane & 15), ks, g);
#pragma unroll
                    for (int j = 0; j < NQ; j++)
                        dp[b][j] = T::mma(vf, dout[j][ks], ks ? dp[b][j] : (f32x4){0.f, 0.f, 0.f, 0.f});
                }
            }
        constexpr uint64_t ALL = KT == 64 ? ~(uint64_t)0 : ((uint64_t)1 << (KT & 63)) - 1;
        if (valid != ALL) {
            const uint64_t mine = valid >> (4 * g);
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (!((mine >> (16 * b + r)) & 1))
#pragma unroll
                        for (int j = 0; j < NQ; j++) s[b][j][r] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            if constexpr (GRAD) {
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float e = exp2_of(__builtin_fmaf(s[b][j][r], p.c, -lse2[j]));
                        s[b][j][r] = e * (dp[b][j][r] - dsum[j]);
                    }
            } else {
                float m = s[0][j][0];
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++) m = fmaxf(m, s[b][j][r]);
                m = max4(m);
                // the maximum that exponents refer to stays until one exceeds it 2^8 times: sums and results
                // are as exact for it, and are scaled anew in few tiles
                if (__builtin_amdgcn_ballot_w64((m - top[j]) * p.c > 8.f)) {
                    m = fmaxf(m, top[j]);
                    const float fade = exp2_of(top[j] * p.c - (m == -INFINITY ? 0.f : m * p.c));
                    top[j] = m;
                    sum[j] *= fade;
                    if constexpr (!ONE) {
#pragma unroll
                        for (int db = 0; db < DB; db++) acc[db][j] *= fade;
                    }
                }
                const float ref = top[j] == -INFINITY ? 0.f : top[j] * p.c;
                float add = 0.f;
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        s[b][j][r] = exp2_of(__builtin_fmaf(s[b][j][r], p.c, -ref));
                        add += s[b][j][r];
                    }
                sum[j] += add;
            }
        }
#pragma unroll
        for (int h = 0; h < KB / 2; h++) {
            typename T::Packed pf[NQ];
#pragma unroll
            for (int j = 0; j < NQ; j++) pf[j] = T::pack(s[2 * h][j], s[2 * h + 1][j]);
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const Frag f = L::column_frag(GRAD ? kt : vt, 32 * h, db, lane);
#pragma unroll
                for (int j = 0; j < NQ; j++) acc[db][j] = T::mma_packed(f, pf[j], acc[db][j]);
            }
        }
        valid = next;
        if constexpr (ONE) break;
    }

    const int d = p.head_d;
    char* const to = GRAD ? p.dq : p.o;
    const int64_t to_row = GRAD ? p.dq_row : p.o_row, to_head = GRAD ? p.dq_head : p.o_head;
    float* const part = it.part < 0 ? nullptr : p.qpart + ((int64_t)it.part * groups + hb) * cross_query_part(p.qs.block, d);
#pragma unroll
    for (int j = 0; j < NQ; j++) sum[j] = sum4(sum[j]);
    // a row without scores gets zeros: its probabilities are, but what they met may have been infinite
#pragma unroll
    for (int j = 0; j < NQ; j++) {
        const bool none = GRAD ? lse2[j] == INFINITY : WK == 1 && !part && no_score(top[j], sum[j]);
        if (__builtin_amdgcn_ballot_w64(none)) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[db][j][r] = none ? 0.f : acc[db][j][r];
        }
    }
    if constexpr (WK == 1) {
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            const int c = (wq * NQ + j) * 16 + (lane & 15);
            if (part) {
                if (!there[j]) continue;
#pragma unroll
                for (int db = 0; db < DB; db++)
                    if (16 * db + 4 * g < d) *reinterpret_cast<f32x4*>(part + (int64_t)c * d + 16 * db + 4 * g) = acc[db][j];
            } else {
                const float f = GRAD ? p.scale : inverse_of(top[j], sum[j]);
                // lanes exchange channels before the ones of no column drop out
#pragma unroll
                for (int db = 0; db < DB; db += 2)
                    T::store_blocks(to + row[j] * to_row + head[j] * to_head, db, g, there[j] ? d : 0, acc[db][j] * f, acc[db + 1][j] * f);
                if (!there[j]) continue;
            }
            if (!GRAD && g == 0) {
                if (part) *reinterpret_cast<f32x2*>(part + (int64_t)p.qs.block * d + 2 * c) = (f32x2){top[j], sum[j]};
                else if (p.lse) p.lse[head[j] * p.ld_lse + row[j]] = lse_of(top[j], sum[j], p.scale);
            }
        }
    } else {
        // the waves' results, in their order
        constexpr int COLS = 16 * NQ;
        float* all = reinterpret_cast<float*>(lds);
        float* ml = all + WAVES * COLS * DP;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NQ; j++) {
            const int c = 16 * j + (lane & 15);
#pragma unroll
            for (int db = 0; db < DB; db++)
                *reinterpret_cast<f32x4*>(all + (wave * COLS + c) * DP + 16 * db + 4 * g) = acc[db][j];
            if (g == 0) *reinterpret_cast<f32x2*>(ml + 2 * (wave * COLS + c)) = (f32x2){top[j], sum[j]};
        }
        __syncthreads();
        for (int e = threadIdx.x; e < COLS * (DP / 4); e += 64 * WAVES) {
            const int c = e / (DP / 4), ch = e % (DP / 4) * 4;
            if (c >= it.cols || ch >= d) continue;
            float m = -INFINITY, l = 0.f;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if constexpr (!GRAD) {
#pragma unroll
                for (int w = 0; w < WAVES; w++) m = fmaxf(m, ml[2 * (w * COLS + c)]);
            }
            const float ref = m == -INFINITY ? 0.f : m * p.c;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float f = GRAD ? 1.f : exp2_of(ml[2 * (w * COLS + c)] * p.c - ref);
                v += *reinterpret_cast<const f32x4*>(all + (w * COLS + c) * DP + ch) * f;
                if constexpr (!GRAD) l += ml[2 * (w * COLS + c) + 1] * f;
            }
            const int r = it.q0 + c / p.qs.pack, h = head0 + c % p.qs.pack;
            const float f = part ? 1.f : GRAD ? p.scale : inverse_of(m, l);
            if (part) *reinterpret_cast<f32x4*>(part + (int64_t)c * d + ch) = v;
            else T::store4(to + r * to_row + h * to_head + ch * T::SIZE, !GRAD && no_score(m, l) ? (f32x4){0.f, 0.f, 0.f, 0.f} : v * f);
            if (!GRAD && ch == 0) {
                if (part) *reinterpret_cast<f32x2*>(part + (int64_t)p.qs.block * d + 2 * c) = (f32x2){m, l};
                else if (p.lse) p.lse[h * p.ld_lse + r] = lse_of(m, l, p.scale);
            }
        }
    }
}

// Blocks whose keys went to several workgroups: the parts in their order, a piece of four channels a thread.
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs p) {
    const int groups = p.heads / p.qs.pack, hb = blockIdx.x / p.qs.n_joins;
    const CrossJoin it = table_entry(p.qs.joins, blockIdx.x - hb * p.qs.n_joins);
    const int d = p.head_d, pieces = d / 4;
    const int64_t stride = (int64_t)groups * cross_query_part(p.qs.block, d);
    const float* first = p.qpart + ((int64_t)it.part0 * groups + hb) * cross_query_part(p.qs.block, d);
    const int e = blockIdx.y * 256 + threadIdx.x;
    if (e < it.cols * pieces) {
        const int c = e / pieces, ch = e % pieces * 4;
        const float* o = first + (int64_t)c * d + ch;
        const float* ml = first + (int64_t)p.qs.block * d + 2 * c;
        float m = -INFINITY, l = 0.f;
        if constexpr (!GRAD)
            for (int i = 0; i < it.parts; i++) m = fmaxf(m, ml[i * stride]);
        const float ref = m == -INFINITY ? 0.f : m * p.c;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < it.parts; i++) {
            const float f = GRAD ? 1.f : exp2_of(ml[i * stride] * p.c - ref);
            v += *reinterpret_cast<const f32x4*>(o + i * stride) * f;
            if constexpr (!GRAD) l += ml[i * stride + 1] * f;
        }
        const int r = it.q0 + c / p.qs.pack, h = hb * p.qs.pack + c % p.qs.pack;
        const float f = GRAD ? p.scale : inverse_of(m, l);
        char* to = GRAD ? p.dq + r * p.dq_row + h * p.dq_head : p.o + r * p.o_row + h * p.o_head;
        T::store4(to + ch * T::SIZE, !GRAD && no_score(m, l) ? (f32x4){0.f, 0.f, 0.f, 0.f} : v * f);
        if (!GRAD && ch == 0 && p.lse) p.lse[h * p.ld_lse + r] = lse_of(m, l, p.scale);
    }
}

template <typename T, int DP, int NQ, int WQ, int WK, int KT, bool GRAD, bool ONE = false>
void run(const CrossArgs& a, hipStream_t s) {
    const unsigned grid = a.qs.n_listed ? (unsigned)a.qs.n_listed : xcd_grid((long)a.qs.n_items * (a.heads / a.qs.pack));
    hipLaunchKernelGGL((cross_queries_kernel<T, DP, NQ, WQ, WK, KT, GRAD, ONE>), dim3(grid), dim3(64 * WQ * WK), 0, s, a);
}
template <typename T, int DP, bool GRAD>
void run_block(const CrossArgs& a, hipStream_t s) {
    constexpr int WK = T::SIZE == 2 ? 4 : 2;
    if constexpr (T::SIZE == 2)
        if (a.qs.block == 128 && a.qs.most_keys <= 64) return run<T, DP, 2, 4, 1, 64, GRAD, true>(a, s);
    // tiles of 32 keys where 64 would spill (gradients with 16 bits a probability, 16384 x 384: 381 us with spills, 370 so)
    constexpr int KT = T::SIZE == 4 || (GRAD && T::WHOLE && DP == 128) ? 32 : 64;
    if (a.qs.block == 128) run<T, DP, 2, 4, 1, KT, GRAD>(a, s);
    else if (a.qs.block == 32) run<T, DP, 2, 1, WK, 32, GRAD>(a, s);
    else run<T, DP, 1, 1, WK, 32, GRAD>(a, s);
}
template <typename T, bool GRAD>
hipError_t run_all(const CrossArgs& a, hipStream_t s) {
    if (a.qs.n_items == 0) return hipSuccess;
    if (a.head_d <= 64) run_block<T, 64, GRAD>(a, s);
    else if (a.head_d <= 96) run_block<T, 96, GRAD>(a, s);
    else run_block<T, 128, GRAD>(a, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.qs.n_joins == 0) return e;
    hipLaunchKernelGGL((cross_join_kernel<Rows<T>, GRAD>), dim3((unsigned)(a.qs.n_joins * (a.heads / a.qs.pack)), (unsigned)((a.qs.block * (a.head_d / 4) + 255) / 256)),
                       dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cross_forward(int dtype, const CrossArgs& a, hipStream_t s) {
    return dtype == AWA_F32 ? run_all<F32, false>(a, s) : a.whole ? run_all<Bf16Whole, false>(a, s) : run_all<Bf16, false>(a, s);
}
hipError_t launch_cross_grad_queries(int dtype, const CrossArgs& a, hipStream_t s) {
    return dtype == AWA_F32 ? run_all<F32, true>(a, s) : a.whole ? run_all<Bf16Whole, true>(a, s) : run_all<Bf16, true>(a, s);
}

}  // namespace awa
