// dit_cross_keys.hip — attention to states of another length: the gradient of keys and values.
//
// A workgroup takes a block of keys of one key head over a run of units, up to 64 query rows of one head each, of
// all sequences that attend to these keys and all heads that share the key head.  Here keys are the columns: with K
// and V as operands in registers, S = Q K^T and dP = dO V^T come out with a key per lane, P and dS leave the
// accumulators as operands of dV^T += dO^T P and dK^T += Q^T dS (dit_cross_device.hpp), and the sums stay in registers
// over the run.  Q and dO reach LDS by DMA, the next unit's during this one's products.
//
// Keys are few where queries are many, so the units are divided over workgroups, whose fp32 partial sums a second
// kernel adds in their order.
//
// Bound by LDS: a wave reads 64 KB of a unit, twice the cycles of its 64 matrix instructions.  Both gradients (this kernel a little
// over half from some hundred keys on, a third at 64), on two inputs in turn: 16384 queries x 384 keys x 20 heads 316 us (0.71
// PFLOP/s of seven products; 297 on one input, part of which stays in the memory-side cache), x 128 176, x 64 142 (130); 5440 x 58 56; four
// clips of up to 5440 x 512, masked, 283; 32 tokens x 750 to 1500 keys, 20 heads on 4, 117.  fp32, 10 heads of 80 on 2, 2 x up to 1237 x
// 300: 98.
#include <type_traits>

#include "dit_cross_device.hpp"

namespace awa {

using namespace cross;

namespace {

// NK blocks of 16 keys a wave, WKEY waves over the keys; where SUBS is 2 as many more take the second 32 rows of a
// unit, and the two halves' sums meet in LDS at the end.
template <typename T, int DP, int NK, int WKEY, int SUBS>
__global__ __launch_bounds__(64 * WKEY * SUBS, 2) void cross_keys_kernel(CrossArgs p) {
    using Frag = typename T::Frag;
    using L = Tile<T, DP>;
    constexpr int KS = DP / 32, DB = DP / 16, QT = CROSS_QT, WAVES = WKEY * SUBS;
    constexpr int TILE_B = QT * L::ROW, STAGE = 2 * TILE_B + 2 * QT * 4;  // Q, dO, lse, dsum
    constexpr int JOIN = SUBS > 1 ? 2 * 64 * WKEY * NK * DB * 16 : 0;
    constexpr int LDS = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
    static_assert(LDS <= 160 * 1024, "LDS");
    __shared__ __align__(16) char lds[LDS];
    CrossKeys it;
    int kv_head;
    if (p.ks.n_listed) {
        it = table_entry(p.ks.items, (int)blockIdx.x);
        if (it.kn == 0) return;
        kv_head = it.group;
    } else {
        const int total = p.ks.n_items * p.kv_heads, wg = xcd_remap(total);
        if (wg >= total) return;
        kv_head = wg / p.ks.n_items;
        it = table_entry(p.ks.items, wg - kv_head * p.ks.n_items);
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wk = wave % WKEY, sub0 = wave / WKEY, g = lane >> 4;
    const int width = p.head_d * T::SIZE;

    // the wave's keys
    Frag k[NK][KS], v[NK][KS];
    bool in[NK];  // takes part
#pragma unroll
    for (int j = 0; j < NK; j++) {
        const int c = (wk * NK + j) * 16 + (lane & 15);
        in[j] = c < it.kn && (!p.mask || p.mask[it.k0 + c]);
        const char* kp = p.k + (int64_t)(it.k0 + c) * p.k_row + kv_head * p.k_head;
        const char* vp = p.v + (int64_t)(it.k0 + c) * p.v_row + kv_head * p.v_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const int d = 32 * ks + 8 * g;
            k[j][ks] = v[j][ks] = T::zero();
            if (in[j] && d < p.head_d) {
                k[j][ks] = T::load(kp + d * T::SIZE);
                v[j][ks] = T::load(vp + d * T::SIZE);
            }
        }
    }
    f32x4 dk[DB][NK], dv[DB][NK];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int j = 0; j < NK; j++) dk[db][j] = dv[db][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // the run's units, one ahead of the tiles that are fetched
    int at = it.first % it.units, head = kv_head * (p.heads / p.kv_heads) + it.first / it.units;
    CrossUnit next = table_entry(p.ks.units, it.unit0 + at);
    auto fetch = [&](int slot) __attribute__((always_inline)) {
        const uint64_t valid = next.rows == 64 ? ~(uint64_t)0 : ((uint64_t)1 << next.rows) - 1;
        const __amdgpu_buffer_rsrc_t qr = uniform_rsrc(p.q + next.q0 * p.q_row + head * p.q_head, 0x7fffffffu);
        const __amdgpu_buffer_rsrc_t dr = uniform_rsrc(p.dout + next.q0 * p.dout_row + head * p.dout_head, 0x7fffffffu);
        char* st = lds + slot * STAGE;
        constexpr int N = TILE_B / 1024 / WAVES;
#pragma unroll
        for (int i = 0; i < N; i++) {
            L::dma(st, wave * N + i, qr, p.q_row, valid, width, lane);
            L::dma(st + TILE_B, wave * N + i, dr, p.dout_row, valid, width, lane);
        }
        if (wave < 2) {
            const float* from = (wave ? p.dsum : p.lse2) + head * p.ld_dsum + next.q0;
            const __amdgpu_buffer_rsrc_t r = uniform_rsrc(from, (uint32_t)next.rows * 4);
            dma4(st + 2 * TILE_B + wave * QT * 4, r, 4 * lane);
        }
        if (++at == it.units) {
            at = 0;
            head++;
        }
    };
    if (it.count > 0) fetch(0);
    for (int n = 0; n < it.count; n++) {
        const int rows = next.rows;
        if (n + 1 < it.count) next = table_entry(p.ks.units, it.unit0 + at);
        wait_vmem_lds<0>();
        __syncthreads();
        char* qt = lds + (n & 1) * STAGE;
        char* dt = qt + TILE_B;
        const float* lse = reinterpret_cast<const float*>(qt + 2 * TILE_B);
        const float mine = lse[lane];
        if (n + 1 < it.count) fetch((n + 1) & 1);
        // rows without scores take no part, whatever they and what comes back to them hold
        const uint64_t none = __builtin_amdgcn_ballot_w64(mine == INFINITY);
        if (none) {
            for (int r = wave; r < rows; r += WAVES)
                if ((none >> r) & 1 && lane < L::CHUNKS)
                    reinterpret_cast<u32x4*>(qt + r * L::ROW)[lane] = reinterpret_cast<u32x4*>(dt + r * L::ROW)[lane] = (u32x4){0, 0, 0, 0};
            __syncthreads();
        }
        const uint64_t out = rows == 64 ? none : none | ~(uint64_t)0 << rows;
        // 32 HALVES rows from base on (64 at once where registers allow: more products that do not wait for each other)
        auto take = [&](auto halves, int base) __attribute__((always_inline)) {
            constexpr int HALVES = decltype(halves)::value, NB = 2 * HALVES;
            f32x4 s[NB][NK], dp[NB][NK];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const Frag qf = L::row_frag(qt, base + 16 * b + (lane & 15), ks, g);
                    const Frag df = L::row_frag(dt, base + 16 * b + (lane & 15), ks, g);
#pragma unroll
                    for (int j = 0; j < NK; j++) {
                        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
                        s[b][j] = T::mma(qf, k[j][ks], ks ? s[b][j] : z);
                        dp[b][j] = T::mma(df, v[j][ks], ks ? dp[b][j] : z);
                    }
                }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int r0 = base + 16 * b + 4 * g;
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse + r0), d4 = *reinterpret_cast<const f32x4*>(lse + QT + r0);
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int j = 0; j < NK; j++) {
                        const float e = exp2_of(__builtin_fmaf(s[b][j][r], p.c, -l4[r]));
                        dp[b][j][r] = e * (dp[b][j][r] - d4[r]);
                        s[b][j][r] = e;
                    }
            }
            if (HALVES == 2 ? out : (uint32_t)(out >> base)) {  // rows past the end hold zeros as well, but infinite keys times zero are not
                const uint64_t its = out >> (base + 4 * g);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if ((its >> (16 * b + r)) & 1)
#pragma unroll
                            for (int j = 0; j < NK; j++) s[b][j][r] = dp[b][j][r] = 0.f;
            }
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                if (h) __builtin_amdgcn_sched_barrier(0xf);  // arithmetic may pass: reads that move further up spill registers
                typename T::Packed pf[NK], sf[NK];
#pragma unroll
                for (int j = 0; j < NK; j++) {
                    pf[j] = T::pack(s[2 * h][j], s[2 * h + 1][j]);
                    sf[j] = T::pack(dp[2 * h][j], dp[2 * h + 1][j]);
                }
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const Frag df = L::column_frag(dt, base + 32 * h, db, lane);
#pragma unroll
                    for (int j = 0; j < NK; j++) dv[db][j] = T::mma_packed(df, pf[j], dv[db][j]);
                    const Frag qf = L::column_frag(qt, base + 32 * h, db, lane);
#pragma unroll
                    for (int j = 0; j < NK; j++) dk[db][j] = T::mma_packed(qf, sf[j], dk[db][j]);
                }
            }
        };
        typedef std::integral_constant<int, 1> One;
        typedef std::integral_constant<int, 2> Two;
        if constexpr (SUBS == 2) {
            if (32 * sub0 < rows) take(One(), 32 * sub0);
        } else {
            take(Two(), 0);
        }
    }
    if constexpr (SUBS > 1) {
        // the second halves' sums, to the first's
        __syncthreads();
        f32x4* at = reinterpret_cast<f32x4*>(lds) + (wk * 64 + lane);
        constexpr int STEP = 64 * WKEY;
        if (sub0) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int j = 0; j < NK; j++) {
                    at[(2 * (db * NK + j)) * STEP] = dk[db][j];
                    at[(2 * (db * NK + j) + 1) * STEP] = dv[db][j];
                }
        }
        __syncthreads();
        if (sub0) return;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int j = 0; j < NK; j++) {
                dk[db][j] += at[(2 * (db * NK + j)) * STEP];
                dv[db][j] += at[(2 * (db * NK + j) + 1) * STEP];
            }
    }
    const int d = p.head_d;
    float* const part = it.part < 0 ? nullptr : p.kpart + ((int64_t)it.part * p.kv_heads + kv_head) * cross_key_part(CROSS_KEYS, d);
#pragma unroll
    for (int j = 0; j < NK; j++) {
        // the lane counted anew: kept over the loop, what follows from it would cost registers there
        const int own = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
        const int c = (wk * NK + j) * 16 + (own & 15), ch0 = 4 * (own >> 4);
        const bool there = c < it.kn;
        char* kp = p.dk + (int64_t)(it.k0 + c) * p.dk_row + kv_head * p.dk_head;
        char* vp = p.dv + (int64_t)(it.k0 + c) * p.dv_row + kv_head * p.dv_head;
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int db = 0; db < DB; db++) {
            dk[db][j] = in[j] ? dk[db][j] * p.scale : z;
            dv[db][j] = in[j] ? dv[db][j] : z;
            const int ch = 16 * db + ch0;
            if (part && there && ch < d) {
                *reinterpret_cast<f32x4*>(part + (int64_t)c * d + ch) = dk[db][j];
                *reinterpret_cast<f32x4*>(part + (int64_t)(CROSS_KEYS + c) * d + ch) = dv[db][j];
            }
        }
        if (part) continue;
#pragma unroll
        for (int db = 0; db < DB; db += 2) {
            T::store_blocks(kp, db, own >> 4, there ? d : 0, dk[db][j], dk[db + 1][j]);
            T::store_blocks(vp, db, own >> 4, there ? d : 0, dv[db][j], dv[db + 1][j]);
        }
    }
}

// Blocks of keys whose units went to several workgroups: the parts in their order, four channels a thread.
template <typename T>
__global__ __launch_bounds__(256) void cross_keys_join_kernel(CrossArgs p) {
    const int kv_head = blockIdx.x / p.ks.n_joins;
    const CrossKeyJoin it = table_entry(p.ks.joins, blockIdx.x - kv_head * p.ks.n_joins);
    const int d = p.head_d, pieces = d / 4, e = blockIdx.y * 256 + threadIdx.x;
    if (e >= 2 * it.kn * pieces) return;
    const int64_t size = cross_key_part(CROSS_KEYS, d), stride = p.kv_heads * size;
    const int which = e / (it.kn * pieces), c = e / pieces % it.kn, ch = e % pieces * 4;
    const float* from = p.kpart + ((int64_t)it.part0 * p.kv_heads + kv_head) * size + (int64_t)(which * CROSS_KEYS + c) * d + ch;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < it.parts; i++) v += *reinterpret_cast<const f32x4*>(from + i * stride);
    char* to = which ? p.dv + (int64_t)(it.k0 + c) * p.dv_row + kv_head * p.dv_head
                     : p.dk + (int64_t)(it.k0 + c) * p.dk_row + kv_head * p.dk_head;
    T::store4(to + ch * T::SIZE, v);
}

template <typename T, int DP>
void run(const CrossArgs& a, hipStream_t s) {
    const dim3 grid(a.ks.n_listed ? (unsigned)a.ks.n_listed : xcd_grid((long)a.ks.n_items * a.kv_heads));
    // fp32: tiles are twice as large, so that one workgroup fills a CU's LDS; twice the waves on them
    constexpr int SUBS = T::SIZE == 2 ? 1 : 2;
    hipLaunchKernelGGL((cross_keys_kernel<T, DP, 1, CROSS_KEYS / 16, SUBS>), grid, dim3(4 * CROSS_KEYS * SUBS), 0, s, a);
}
template <typename T>
hipError_t run_all(const CrossArgs& a, hipStream_t s) {
    if (a.ks.n_items == 0) return hipSuccess;
    if (a.head_d <= 64) run<T, 64>(a, s);
    else if (a.head_d <= 96) run<T, 96>(a, s);
    else run<T, 128>(a, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.ks.n_joins == 0) return e;
    const int pieces = 2 * CROSS_KEYS * (a.head_d / 4);
    hipLaunchKernelGGL((cross_keys_join_kernel<Rows<T>>), dim3((unsigned)(a.ks.n_joins * a.kv_heads), (unsigned)((pieces + 255) / 256)),
                       dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cross_grad_keys(int dtype, const CrossArgs& a, hipStream_t s) {
    return dtype == AWA_F32 ? run_all<F32>(a, s) : a.whole ? run_all<Bf16Whole>(a, s) : run_all<Bf16>(a, s);
}

}  // namespace awa
