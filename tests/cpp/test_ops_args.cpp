// Argument checks of dit_ops.h's entry points on the CPU: csrc/dit_ops.cpp is
// compiled into this program, the launches and the shared helpers are the stubs
// below, so that an accepted call only counts.  Prints one line per failed check.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <limits>
#include <vector>

#include "dit_ops_internal.hpp"

static int launches, failures, checks;
static awa::RopeArgs last_rope;

namespace awa {
void set_err(awa_ctx* ctx, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    ctx->err = buf;
}
DeviceGuard::DeviceGuard(int) {}
DeviceGuard::~DeviceGuard() {}
hipError_t launch_quant_rows(int, const QuantArgs&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_quant_blocks(int, const QuantArgs&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_gemm_fp8(Fp8Gemm&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_rope(int, int, RopeArgs& a, hipStream_t) { launches++; last_rope = a; return hipSuccess; }
}  // namespace awa

static awa_ctx ctx;

// want: AWA_EARG with a message and no launch, or AWA_OK with `n` launches
static void check(const char* what, int rc, int want, int n = 1) {
    checks++;
    const bool ok = rc == want && launches == (want == AWA_OK ? n : 0) && (want == AWA_OK || !ctx.err.empty());
    if (!ok) {
        failures++;
        printf("FAILED %s: rc %d (want %d), %d launches, \"%s\"\n", what, rc, want, launches, ctx.err.c_str());
    }
    launches = 0;
    ctx.err.clear();
}

int main() {
    // addresses that are only compared, never read
    char* const X = (char*)0x100000000, *const Q = (char*)0x200000000, *const S = (char*)0x300000000;
    char* const W = (char*)0x400000000, *const SW = (char*)0x500000000, *const C = (char*)0x600000000;
    const int bad = AWA_EARG, ok = AWA_OK;

    auto quant = [&](int dt, const void* x, int64_t ldx, int M, int K, int br, void* q, void* s, int64_t lds) {
        return dit_quant_fp8(&ctx, dt, x, ldx, M, K, br, (uint8_t*)q, (uint32_t*)s, lds, nullptr);
    };
    check("quant", quant(AWA_BF16, X, 200, 7, 200, 1, Q, S, 7), ok);
    check("quant blocks", quant(AWA_F32, X, 201, 300, 200, 128, Q, S, 3), ok);
    check("quant no rows", quant(AWA_BF16, X, 200, 0, 200, 1, Q, S, 0), ok, 0);
    check("quant one row, any stride", quant(AWA_BF16, X, 0, 1, 200, 1, Q, S, 1), ok);
    check("quant unaligned x", quant(AWA_BF16, X + 2, 200, 7, 200, 1, Q, S, 7), ok);
    check("quant null ctx", (launches = 0, ctx.err = "-", dit_quant_fp8(nullptr, AWA_F32, X, 8, 1, 8, 1, (uint8_t*)Q, (uint32_t*)S, 1, nullptr)), bad);
    check("quant null x", quant(AWA_BF16, nullptr, 200, 7, 200, 1, Q, S, 7), bad);
    check("quant null q", quant(AWA_BF16, X, 200, 7, 200, 1, nullptr, S, 7), bad);
    check("quant null scale", quant(AWA_BF16, X, 200, 7, 200, 1, Q, nullptr, 7), bad);
    check("quant dtype", quant(2, X, 200, 7, 200, 1, Q, S, 7), bad);
    check("quant rows < 0", quant(AWA_BF16, X, 200, -1, 200, 1, Q, S, 7), bad);
    check("quant too many rows", quant(AWA_BF16, X, 200, DIT_OPS_ROWS_MAX + 1, 200, 1, Q, S, 1 << 30), bad);
    check("quant no columns", quant(AWA_BF16, X, 200, 7, 0, 1, Q, S, 7), bad);
    check("quant too many columns", quant(AWA_BF16, X, 1 << 21, 7, DIT_OPS_COLS_MAX + 1, 1, Q, S, 7), bad);
    check("quant block_rows", quant(AWA_BF16, X, 200, 7, 200, 64, Q, S, 7), bad);
    check("quant ldx", quant(AWA_BF16, X, 199, 7, 200, 1, Q, S, 7), bad);
    check("quant huge ldx", quant(AWA_BF16, X, (int64_t)1 << 60, 7, 200, 1, Q, S, 7), bad);
    check("quant huge ld_scale", quant(AWA_BF16, X, 200, 7, 2000, 1, Q, S, (int64_t)1 << 61), bad);
    check("quant ld_scale", quant(AWA_BF16, X, 200, 7, 200, 1, Q, S, 6), bad);
    check("quant ld_scale blocks", quant(AWA_BF16, X, 200, 129, 200, 128, Q, S, 1), bad);
    check("quant q alignment", quant(AWA_BF16, X, 200, 7, 200, 1, Q + 8, S, 7), bad);
    check("quant scale alignment", quant(AWA_BF16, X, 200, 7, 200, 1, Q, S + 2, 7), bad);
    check("quant x alignment", quant(AWA_F32, X + 2, 200, 7, 200, 1, Q, S, 7), bad);
    check("quant q over x", quant(AWA_BF16, X, 200, 7, 200, 1, X + 2784, S, 7), bad);
    check("quant q after x", quant(AWA_BF16, X, 200, 7, 200, 1, X + 2800, S, 7), ok);
    check("quant scale over q", quant(AWA_BF16, X, 200, 7, 200, 1, Q, Q + 1788, 7), bad);

    auto gemm = [&](const void* a, const void* as, int64_t lda, const void* w, const void* ws, int64_t ldw,
                    const void* b, int dt, void* c, int64_t ldc, int M, int N, int K) {
        return dit_gemm_fp8(&ctx, (const uint8_t*)a, (const uint32_t*)as, lda, (const uint8_t*)w, (const uint32_t*)ws,
                            ldw, (const float*)b, dt, c, ldc, M, N, K, nullptr);
    };
    check("gemm", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), ok);
    check("gemm no rows", gemm(Q, S, 0, W, SW, 2, nullptr, AWA_BF16, C, 200, 0, 200, 256), ok, 0);
    check("gemm one row, any stride", gemm(Q, S, 1, W, SW, 2, nullptr, AWA_F32, C, 0, 1, 200, 256), ok);
    check("gemm unaligned C", gemm(Q, S, 5, W, SW, 2, X, AWA_BF16, C + 2, 201, 5, 200, 256), ok);
    check("gemm whole", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16 | DIT_FP8_WHOLE, C, 200, 5, 200, 256), ok);
    check("gemm whole fp32", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_F32 | DIT_FP8_WHOLE, C, 200, 5, 200, 256), ok);
    check("gemm whole dtype", gemm(Q, S, 5, W, SW, 2, nullptr, 7 | DIT_FP8_WHOLE, C, 200, 5, 200, 256), bad);
    check("gemm other flag", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16 | 2 * DIT_FP8_WHOLE, C, 200, 5, 200, 256), bad);
    check("gemm whole and other flag", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16 | 3 * DIT_FP8_WHOLE, C, 200, 5, 200, 256), bad);
    check("gemm whole c alignment", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_F32 | DIT_FP8_WHOLE, C + 2, 200, 5, 200, 256), bad);
    check("gemm null a", gemm(nullptr, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm null as", gemm(Q, nullptr, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm null w", gemm(Q, S, 5, nullptr, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm null ws", gemm(Q, S, 5, W, nullptr, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm null c", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, nullptr, 200, 5, 200, 256), bad);
    check("gemm dtype", gemm(Q, S, 5, W, SW, 2, nullptr, 7, C, 200, 5, 200, 256), bad);
    check("gemm rows < 0", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, -5, 200, 256), bad);
    check("gemm N 0", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 0, 256), bad);
    check("gemm N large", gemm(Q, S, 5, W, SW, 1 << 20, nullptr, AWA_BF16, C, 1 << 21, 5, DIT_OPS_COLS_MAX + 1, 256), bad);
    check("gemm K 0", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 0), bad);
    check("gemm K 200", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 200), bad);
    check("gemm K large", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, DIT_OPS_COLS_MAX + 128), bad);
    check("gemm ldc", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 199, 5, 200, 256), bad);
    check("gemm ldc large", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, C, DIT_OPS_COLS_MAX + 1, 5, 200, 256), bad);
    check("gemm huge ld_as", gemm(Q, S, (int64_t)1 << 61, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 1024), bad);
    check("gemm huge ld_ws", gemm(Q, S, 5, W, SW, (int64_t)1 << 61, nullptr, AWA_BF16, C, 200, 5, 200, 1024), bad);
    check("gemm ld_as", gemm(Q, S, 4, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm ld_ws", gemm(Q, S, 5, W, SW, 1, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm a alignment", gemm(Q + 8, S, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm w alignment", gemm(Q, S, 5, W + 4, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm scale alignment", gemm(Q, S + 1, 5, W, SW, 2, nullptr, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm bias alignment", gemm(Q, S, 5, W, SW, 2, X + 2, AWA_BF16, C, 200, 5, 200, 256), bad);
    check("gemm c alignment", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_F32, C + 2, 200, 5, 200, 256), bad);
    check("gemm c over a", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, Q + 1264, 200, 5, 200, 256), bad);
    check("gemm c after a", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, Q + 1280, 200, 5, 200, 256), ok);
    check("gemm c over w", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, W + 51184, 200, 5, 200, 256), bad);
    check("gemm c over as", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, S + 16, 200, 5, 200, 256), bad);
    check("gemm c over ws", gemm(Q, S, 5, W, SW, 2, nullptr, AWA_BF16, SW + 4, 200, 5, 200, 256), bad);
    check("gemm c over bias", gemm(Q, S, 5, W, SW, 2, X, AWA_BF16, X + 784, 200, 5, 200, 256), bad);

    // rope: 10 tokens of 4 heads of 64 channels in fp32 rows of 768 (q, k and v of 4 heads each)
    dit_rope_plan plan{};
    plan.layout = DIT_ROPE_HALF; plan.axes = 2; plan.pairs[0] = 16; plan.pairs[1] = 8; plan.scale = 1.0;
    for (int i = 0; i < 24; i++) plan.freq[i] = 0.5;
    const int32_t* pos = (const int32_t*)SW;
    auto rows = [](char* x, char* o, int heads, int64_t xt, int64_t xh, int64_t ot, int64_t oh) {
        return dit_rope_rows{x, o, heads, xt, xh, ot, oh};
    };
    auto rope = [&](std::vector<dit_rope_rows> r, int tokens = 10, int d = 64, int dt = AWA_F32) {
        return dit_rope(&ctx, dt, r.data(), (int)r.size(), tokens, d, &plan, pos, nullptr);
    };
    const dit_rope_rows q = rows(X, X, 4, 768, 64, 768, 64), k = rows(X + 1024, X + 1024, 4, 768, 64, 768, 64);
    const dit_rope_rows copy = rows(X, C, 4, 768, 64, 256, 64);
    check("rope in place", rope({q}), ok);
    check("rope q and k of a row", rope({q, k}), ok);
    check("rope copy", rope({copy}), ok);
    check("rope no tokens", rope({q}, 0), ok, 0);
    check("rope no heads", rope({rows(X, X, 0, 0, 0, 0, 0)}), ok, 0);
    check("rope no heads of the first", (rope({rows(nullptr, nullptr, 0, 0, 0, 0, 0), k})), ok);
    if (last_rope.heads[0] != 4 || last_rope.heads[1] != 0 || last_rope.x[0] != k.x) { failures++; printf("FAILED second alone\n"); }
    check("rope heads outside tokens", rope({rows(X, X, 4, 64, 640, 64, 640)}), ok);
    check("rope per head q|k|v", rope({rows(X, X, 4, 768, 192, 768, 192), rows(X + 256, X + 256, 4, 768, 192, 768, 192)}), ok);
    check("rope into other columns", rope({rows(X, X + 2048, 4, 768, 64, 768, 64)}), ok);
    check("rope broadcast input", rope({rows(X, C, 4, 0, 64, 256, 64)}), ok);
    check("rope one token, any token stride", rope({rows(X, X, 4, 0, 64, 0, 64)}, 1), ok);
    check("rope same tensor twice", rope({q, q}), bad);
    check("rope overlapping tensors", rope({q, rows(X + 512, X + 512, 4, 768, 64, 768, 64)}), bad);
    check("rope output over the other input", rope({rows(X, X + 1024, 4, 768, 64, 768, 64), rows(X + 1024, C, 4, 768, 64, 256, 64)}), bad);
    check("rope shifted in place", rope({rows(X, X + 4, 4, 768, 64, 768, 64)}), bad);
    check("rope other strides in place", rope({rows(X, X, 4, 768, 64, 256, 64)}), bad);
    check("rope output heads overlap", rope({rows(X, C, 4, 768, 64, 256, 32)}), bad);
    check("rope output tokens overlap", rope({rows(X, C, 4, 768, 64, 128, 64)}), bad);
    check("rope broadcast in place", rope({rows(X, X, 4, 0, 64, 0, 64)}), bad);
    check("rope output over positions", rope({rows(X, SW - 1024, 4, 768, 64, 256, 64)}), bad);
    check("rope negative stride", rope({rows(X, C, 4, -768, 64, 256, 64)}), bad);
    check("rope huge stride", rope({rows(X, C, 4, (int64_t)1 << 40, 64, 256, 64)}), bad);
    check("rope null x", rope({rows(nullptr, C, 4, 768, 64, 256, 64)}), bad);
    check("rope null out", rope({rows(X, nullptr, 4, 768, 64, 256, 64)}), bad);
    check("rope x alignment", rope({rows(X + 2, C, 4, 768, 64, 256, 64)}), bad);
    check("rope heads < 0", rope({rows(X, C, -1, 768, 64, 256, 64)}), bad);
    check("rope dtype", rope({q}, 10, 64, 5), bad);
    check("rope tokens < 0", rope({q}, -1), bad);
    check("rope too many tokens", rope({q}, DIT_OPS_ROWS_MAX + 1), bad);
    check("rope head_d under the pairs", rope({q}, 10, 47), bad);
    check("rope head_d odd", rope({rows(X, X, 4, 768, 64, 768, 64)}, 10, 49), ok);
    check("rope head_d over 256", rope({rows(X, X, 2, 768, 300, 768, 300)}, 10, 257), bad);
    check("rope three tensors", rope({q, k, copy}), bad);
    check("rope no tensors", rope({}), bad);
    check("rope null plan", dit_rope(&ctx, AWA_F32, &q, 1, 10, 64, nullptr, pos, nullptr), bad);
    check("rope null positions", dit_rope(&ctx, AWA_F32, &q, 1, 10, 64, &plan, nullptr, nullptr), bad);
    auto with = [&](const char* what, auto&& change) {
        const dit_rope_plan was = plan;
        change(plan);
        check(what, rope({q}), bad);
        plan = was;
    };
    with("rope layout", [](dit_rope_plan& p) { p.layout = 2; });
    with("rope axes 0", [](dit_rope_plan& p) { p.axes = 0; });
    with("rope axes 5", [](dit_rope_plan& p) { p.axes = 5; });
    with("rope pairs < 0", [](dit_rope_plan& p) { p.pairs[0] = -1; });
    with("rope pairs over the head", [](dit_rope_plan& p) { p.pairs[1] = 17; });
    with("rope pairs overflow", [](dit_rope_plan& p) { p.pairs[1] = std::numeric_limits<int>::max(); });
    with("rope infinite frequency", [](dit_rope_plan& p) { p.freq[23] = INFINITY; });
    with("rope large frequency", [](dit_rope_plan& p) { p.freq[1] = -65537.0; });
    with("rope NaN frequency", [](dit_rope_plan& p) { p.freq[0] = NAN; });
    with("rope infinite scale", [](dit_rope_plan& p) { p.scale = 1e300; });

    double f[128];
    auto freqs = [&](int kind, int n, double base, double factor, double trained = 0, double lo = 0, double hi = 0) {
        ctx.err = "host only";
        return dit_rope_freqs(kind, n, base, factor, trained, lo, hi, f);
    };
    check("freqs", freqs(DIT_ROPE_PLAIN, 128, 1e4, 1), ok, 0);
    check("freqs kind", freqs(4, 8, 1e4, 1), bad);
    check("freqs n 0", freqs(DIT_ROPE_PLAIN, 0, 1e4, 1), bad);
    check("freqs n 129", freqs(DIT_ROPE_PLAIN, 129, 1e4, 1), bad);
    check("freqs base 0", freqs(DIT_ROPE_PLAIN, 8, 0, 1), bad);
    check("freqs base NaN", freqs(DIT_ROPE_PLAIN, 8, NAN, 1), bad);
    check("freqs factor 0.5", freqs(DIT_ROPE_LINEAR, 8, 1e4, 0.5), bad);
    check("freqs base stretched with one pair", freqs(DIT_ROPE_BASE, 1, 1e4, 2), bad);
    check("freqs bands without a length", freqs(DIT_ROPE_BANDS, 8, 1e4, 2, 0, 1, 32), bad);
    check("freqs bands low = high", freqs(DIT_ROPE_BANDS, 8, 1e4, 2, 4096, 4, 4), bad);
    check("freqs null", dit_rope_freqs(DIT_ROPE_PLAIN, 8, 1e4, 1, 0, 0, 0, (ctx.err = "host only", nullptr)), bad);

    printf("checks=%d failures=%d\n", checks, failures);
    return failures != 0;
}
