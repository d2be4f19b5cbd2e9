// dit_ops.cpp — C ABI of the operators of dit_ops.h: argument checks and launches.
#include <cmath>
#include <utility>

#include "dit_ops_internal.hpp"

using namespace awa;

namespace {

size_t elem(int dtype) { return dtype == AWA_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == AWA_F32 || dtype == AWA_BF16; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t groups_of(int k) { return ((int64_t)k + 511) / 512; }
// strides far enough below 2^63 for the checks' own arithmetic
constexpr int64_t STRIDE_MAX = (int64_t)1 << 36;
// bytes from the first to past the last element of rows ld elements apart
size_t span(int64_t rows, int64_t ld, int64_t cols, size_t size) {
    return rows > 0 ? (size_t)((rows - 1) * ld + cols) * size : 0;
}

// A view of a tensor for the checks below: token and head strides (a stride of
// one thing only does not matter and becomes 0).
struct View {
    uintptr_t at;
    int64_t token, head;  // bytes
    int64_t width;        // bytes of a head's channels
    int64_t tokens, heads;
    uintptr_t end() const { return at + (tokens - 1) * token + (heads - 1) * head + width; }
};
View view_of(const void* p, int64_t token, int64_t head, int tokens, int heads, int head_d, size_t size) {
    return {reinterpret_cast<uintptr_t>(p), tokens > 1 ? token * (int64_t)size : 0,
            heads > 1 ? head * (int64_t)size : 0, head_d * (int64_t)size, tokens, heads};
}
// whether the elements of a view are all different
bool separate(const View& v) {
    int64_t n[2] = {v.tokens, v.heads}, st[2] = {v.token, v.head};
    if (n[0] > 1 && n[1] > 1 && st[0] < st[1]) { std::swap(n[0], n[1]); std::swap(st[0], st[1]); }
    // st[0] the larger of the strides that count
    if (n[1] > 1 && st[1] < v.width) return false;
    const int64_t inner = (n[1] - 1) * st[1] + v.width;
    return n[0] <= 1 || st[0] >= inner;
}
// whether two views are known to share no element: apart in memory, or side by
// side inside a common period (the token stride, or the head stride of both)
bool apart(const View& a, const View& b) {
    if (a.end() <= b.at || b.end() <= a.at) return true;
    auto beside = [&](int64_t period, int64_t wa, int64_t wb) {
        if (period <= 0 || wa > period || wb > period) return false;
        // where b begins in a's period
        const int64_t off = b.at >= a.at ? (int64_t)((b.at - a.at) % (uintptr_t)period)
                                         : (period - (int64_t)((a.at - b.at) % (uintptr_t)period)) % period;
        return off >= wa && off + wb <= period;
    };
    const int64_t ia = (a.heads - 1) * a.head + a.width, ib = (b.heads - 1) * b.head + b.width;
    if (a.token == b.token && beside(a.token, ia, ib)) return true;
    // the same steps: all offsets are whole numbers of head strides apart
    if (a.head > 0 && a.head == b.head && a.token % a.head == 0 && b.token % a.head == 0)
        return beside(a.head, a.width, b.width);
    return false;
}

}  // namespace

extern "C" {

int dit_quant_fp8(awa_ctx* ctx, int dtype, const void* d_x, int64_t ldx, int M, int K, int block_rows,
                  uint8_t* d_q, uint32_t* d_scale, int64_t ld_scale, awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    if (!d_x || !d_q || !d_scale || !dtype_ok(dtype) || M < 0 || M > DIT_OPS_ROWS_MAX || K < 1 ||
        K > DIT_OPS_COLS_MAX || (block_rows != 1 && block_rows != DIT_FP8_BLOCK)) {
        set_err(ctx, "dit_quant_fp8: bad argument dtype=%d M=%d K=%d block_rows=%d (M <= %d, 1 <= K <= %d, block_rows 1 or %d)",
                dtype, M, K, block_rows, DIT_OPS_ROWS_MAX, DIT_OPS_COLS_MAX, DIT_FP8_BLOCK);
        return AWA_EARG;
    }
    const int64_t srows = block_rows == 1 ? M : (M + DIT_FP8_BLOCK - 1) / DIT_FP8_BLOCK;
    if ((M > 1 && (ldx < K || ldx > STRIDE_MAX)) || ld_scale < srows || ld_scale > STRIDE_MAX) {
        set_err(ctx, "dit_quant_fp8: ldx=%lld (at least K=%d), ld_scale=%lld (at least %lld; both at most 2^36)", (long long)ldx, K,
                (long long)ld_scale, (long long)srows);
        return AWA_EARG;
    }
    if (!aligned(d_x, elem(dtype)) || !aligned(d_q, 16) || !aligned(d_scale, 4)) {
        set_err(ctx, "dit_quant_fp8: d_q must be 16-byte, d_scale 4-byte and d_x element aligned");
        return AWA_EARG;
    }
    if (M == 0) return AWA_OK;
    QuantArgs a{};
    a.x = d_x; a.ldx = M > 1 ? ldx : K; a.M = M; a.K = K;
    a.kp = (K + DIT_FP8_BLOCK - 1) / DIT_FP8_BLOCK * DIT_FP8_BLOCK;
    a.q = d_q; a.scale = d_scale; a.ld_scale = ld_scale;
    const size_t xb = span(M, a.ldx, K, elem(dtype)), qb = (size_t)M * a.kp;
    const size_t sb = span(groups_of(K), ld_scale, srows, 4);
    if (overlaps(d_x, xb, d_q, qb) || overlaps(d_x, xb, d_scale, sb) || overlaps(d_q, qb, d_scale, sb)) {
        set_err(ctx, "dit_quant_fp8: outputs lie over the input or each other");
        return AWA_EARG;
    }
    DeviceGuard dg(ctx->device);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (block_rows == 1) HIPCK(ctx, launch_quant_rows(dtype, a, s));
    else HIPCK(ctx, launch_quant_blocks(dtype, a, s));
    return AWA_OK;
}

int dit_gemm_fp8(awa_ctx* ctx, const uint8_t* d_a, const uint32_t* d_as, int64_t ld_as, const uint8_t* d_w,
                 const uint32_t* d_ws, int64_t ld_ws, const float* d_bias, int dtype_c, void* d_c, int64_t ldc,
                 int M, int N, int K, awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    const bool whole = dtype_c == (AWA_F32 | DIT_FP8_WHOLE) || dtype_c == (AWA_BF16 | DIT_FP8_WHOLE);
    if (whole) dtype_c &= ~DIT_FP8_WHOLE;
    if (!d_a || !d_as || !d_w || !d_ws || !d_c || !dtype_ok(dtype_c) || M < 0 || M > DIT_OPS_ROWS_MAX || N < 1 ||
        N > DIT_OPS_COLS_MAX || K < DIT_FP8_BLOCK || K % DIT_FP8_BLOCK || K > DIT_OPS_COLS_MAX) {
        set_err(ctx, "dit_gemm_fp8: bad argument dtype=%d M=%d N=%d K=%d (M <= %d, N, K <= %d, K %% %d == 0)", dtype_c, M,
                N, K, DIT_OPS_ROWS_MAX, DIT_OPS_COLS_MAX, DIT_FP8_BLOCK);
        return AWA_EARG;
    }
    const int64_t nb = (N + DIT_FP8_BLOCK - 1) / DIT_FP8_BLOCK;
    if ((M > 1 && (ldc < N || ldc > DIT_OPS_COLS_MAX)) || ld_as < M || ld_as > STRIDE_MAX || ld_ws < nb ||
        ld_ws > STRIDE_MAX) {
        set_err(ctx, "dit_gemm_fp8: ldc=%lld (%d .. %d), ld_as=%lld (at least %d), ld_ws=%lld (at least %lld; both at most 2^36)",
                (long long)ldc, N, DIT_OPS_COLS_MAX, (long long)ld_as, M, (long long)ld_ws, (long long)nb);
        return AWA_EARG;
    }
    if (!aligned(d_a, 16) || !aligned(d_w, 16) || !aligned(d_as, 4) || !aligned(d_ws, 4) || !aligned(d_bias, 4) ||
        !aligned(d_c, elem(dtype_c))) {
        set_err(ctx, "dit_gemm_fp8: d_a and d_w must be 16-byte, scales and bias 4-byte, d_c element aligned");
        return AWA_EARG;
    }
    if (M == 0) return AWA_OK;
    Fp8Gemm p{};
    p.A = d_a; p.as = d_as; p.ld_as = ld_as;
    p.W = d_w; p.ws = d_ws; p.ld_ws = ld_ws;
    p.bias = d_bias;
    p.C = d_c; p.ldc = M > 1 ? ldc : N;
    p.M = M; p.N = N; p.K = K;
    p.c_f32 = dtype_c == AWA_F32;
    p.whole = whole;
    p.c_vec = aligned(d_c, 16) && p.ldc * elem(dtype_c) % 16 == 0;
    const size_t cb = span(M, p.ldc, N, elem(dtype_c));
    const int64_t g = groups_of(K);
    if (overlaps(d_c, cb, d_a, (size_t)M * K) || overlaps(d_c, cb, d_w, (size_t)N * K) ||
        overlaps(d_c, cb, d_as, span(g, ld_as, M, 4)) || overlaps(d_c, cb, d_ws, span(g, ld_ws, nb, 4)) ||
        (d_bias && overlaps(d_c, cb, d_bias, (size_t)N * 4))) {
        set_err(ctx, "dit_gemm_fp8: C lies over an input");
        return AWA_EARG;
    }
    DeviceGuard dg(ctx->device);
    HIPCK(ctx, launch_gemm_fp8(p, reinterpret_cast<hipStream_t>(stream)));
    return AWA_OK;
}

int dit_rope(awa_ctx* ctx, int dtype, const dit_rope_rows* rows, int n_rows, int n_tokens, int head_d,
             const dit_rope_plan* plan, const int32_t* d_pos, awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    if (!rows || !plan || !dtype_ok(dtype) || n_rows < 1 || n_rows > 2 || n_tokens < 0 ||
        n_tokens > DIT_OPS_ROWS_MAX || head_d < 1 || head_d > 2 * DIT_ROPE_MAX_PAIRS ||
        (plan->layout != DIT_ROPE_INTERLEAVED && plan->layout != DIT_ROPE_HALF) || plan->axes < 1 ||
        plan->axes > DIT_ROPE_MAX_AXES || !std::isfinite((float)plan->scale)) {
        set_err(ctx, "dit_rope: bad argument (dtype=%d, %d tensors, %d tokens, head_d=%d, at most %d; plan: layout, axes 1 .. %d, finite scale)",
                dtype, n_rows, n_tokens, head_d, 2 * DIT_ROPE_MAX_PAIRS, DIT_ROPE_MAX_AXES);
        return AWA_EARG;
    }
    RopeArgs a{};
    for (int i = 0; i < DIT_ROPE_MAX_AXES; i++) {
        if (i < plan->axes) {
            if (plan->pairs[i] < 0 || plan->pairs[i] > head_d / 2 - a.pairs) {
                set_err(ctx, "dit_rope: the axes' pairs must be at least 0, together at most head_d / 2 = %d", head_d / 2);
                return AWA_EARG;
            }
            a.pairs += plan->pairs[i];
        }
        a.axis_end[i] = a.pairs;
    }
    for (int i = 0; i < a.pairs; i++) {
        if (!(std::fabs(plan->freq[i]) <= DIT_ROPE_MAX_FREQ)) {
            set_err(ctx, "dit_rope: frequency %d is %g (a finite number of at most %d either way)", i, plan->freq[i],
                    DIT_ROPE_MAX_FREQ);
            return AWA_EARG;
        }
        a.quarters[i] = plan->freq[i] / (0.5 * M_PI);
    }
    a.axes = plan->axes;
    a.cos_scale = plan->scale;
    a.sin_scale = plan->inverse ? -plan->scale : plan->scale;
    a.tokens = n_tokens;
    a.head_d = head_d;
    a.pos = d_pos;
    View vx[2], vo[2];
    bool in_place = true;
    const size_t size = elem(dtype);
    for (int t = 0; t < n_rows; t++) {
        const dit_rope_rows& r = rows[t];
        if (r.heads < 0 || r.heads > 32767) {
            set_err(ctx, "dit_rope: heads=%d of tensor %d (0 .. 32767)", r.heads, t);
            return AWA_EARG;
        }
        if (r.heads == 0 || n_tokens == 0) continue;
        if (!r.x || !r.out || !d_pos || !aligned(r.x, size) || !aligned(r.out, size) || !aligned(d_pos, 4)) {
            set_err(ctx, "dit_rope: null or misaligned pointer (tensor %d)", t);
            return AWA_EARG;
        }
        for (int64_t st : {r.x_token, r.x_head, r.out_token, r.out_head}) {
            if (st < 0 || st > STRIDE_MAX) {
                set_err(ctx, "dit_rope: stride %lld of tensor %d", (long long)st, t);
                return AWA_EARG;
            }
        }
        vx[t] = view_of(r.x, r.x_token, r.x_head, n_tokens, r.heads, head_d, size);
        vo[t] = view_of(r.out, r.out_token, r.out_head, n_tokens, r.heads, head_d, size);
        const bool same = vx[t].at == vo[t].at && vx[t].token == vo[t].token && vx[t].head == vo[t].head;
        const size_t pos_bytes = (size_t)n_tokens * plan->axes * 4;
        if (!separate(vo[t]) || (!same && !apart(vx[t], vo[t])) ||
            overlaps(r.out, vo[t].end() - vo[t].at, d_pos, pos_bytes)) {
            set_err(ctx, "dit_rope: elements of tensor %d's output coincide, or lie over its input or the positions", t);
            return AWA_EARG;
        }
        if (!same) in_place = false;
    }
    if (n_rows == 2 && rows[0].heads && rows[1].heads && n_tokens &&
        (!apart(vo[0], vo[1]) || !apart(vo[0], vx[1]) || !apart(vx[0], vo[1]))) {
        set_err(ctx, "dit_rope: an output of one tensor lies over the other tensor");
        return AWA_EARG;
    }
    for (int t = 0; t < n_rows; t++) {
        if (rows[t].heads == 0) continue;
        const int i = a.heads[0] ? 1 : 0;
        a.x[i] = rows[t].x; a.out[i] = rows[t].out;
        a.x_token[i] = rows[t].x_token; a.x_head[i] = rows[t].x_head;
        a.out_token[i] = rows[t].out_token; a.out_head[i] = rows[t].out_head;
        a.heads[i] = rows[t].heads;
    }
    if (n_tokens == 0 || a.heads[0] == 0) return AWA_OK;
    a.copy = !in_place;
    DeviceGuard dg(ctx->device);
    HIPCK(ctx, launch_rope(dtype, plan->layout, a, reinterpret_cast<hipStream_t>(stream)));
    return AWA_OK;
}

int dit_rope_freqs(int kind, int n, double base, double factor, double trained, double low, double high,
                   double* h_freq) {
    if (!h_freq || n < 1 || n > DIT_ROPE_MAX_PAIRS || !(base > 0) || !std::isfinite(base) || !(factor >= 1) ||
        !std::isfinite(factor) || kind < DIT_ROPE_PLAIN || kind > DIT_ROPE_BANDS || (kind == DIT_ROPE_BASE && n < 2))
        return AWA_EARG;
    if (kind == DIT_ROPE_BANDS &&
        (!(trained > 0) || !std::isfinite(trained) || !(low < high) || !std::isfinite(low) || !std::isfinite(high)))
        return AWA_EARG;
    if (kind == DIT_ROPE_BASE) base *= std::pow(factor, (double)n / (n - 1));
    for (int i = 0; i < n; i++) {
        double f = std::pow(base, -(double)i / n);
        if (kind == DIT_ROPE_LINEAR) f /= factor;
        if (kind == DIT_ROPE_BANDS) {
            const double r = trained * f / (2.0 * M_PI);
            const double t = std::fmin(std::fmax((r - low) / (high - low), 0.0), 1.0);
            f *= t + (1.0 - t) / factor;
        }
        h_freq[i] = f;
    }
    return AWA_OK;
}

}  // extern "C"
