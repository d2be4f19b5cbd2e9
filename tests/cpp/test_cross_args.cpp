// The attention's entry points of dit_train.h on the CPU, beside test_train_args.cpp: csrc/dit_train.cpp is included here, the
// launches and the shared helpers are the stubs below, so that an accepted call only leaves its arguments.  Prints one line
// per failed check.
#include <cstdarg>
#include <cstdio>
#include <random>
#include <set>

#include "../../seedvr2-2b-ncnn_amd/csrc/dit_train.cpp"

static int launches, failures, checks, last_dtype;
static CrossArgs last;

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
hipError_t launch_layer_norm(int, int, const NormFwd&, hipStream_t) { return hipSuccess; }
hipError_t launch_layer_norm_grad(int, int, const NormGrad&, hipStream_t) { return hipSuccess; }
int norm_grad_groups(int M, int) { return std::min(M, 256); }
GradWeightPlan grad_weight_plan(int, int M, int, int) { return {128, 1, 1, M, 0}; }
hipError_t launch_grad_weight(int, GradWeight&, hipStream_t) { return hipSuccess; }
static hipError_t keep(int dtype, const CrossArgs& a) {
    launches++;
    last_dtype = dtype;
    last = a;
    return hipSuccess;
}
hipError_t launch_cross_forward(int dtype, const CrossArgs& a, hipStream_t) { return keep(dtype, a); }
hipError_t launch_cross_grad_queries(int dtype, const CrossArgs& a, hipStream_t) { return keep(dtype, a); }
hipError_t launch_cross_grad_keys(int dtype, const CrossArgs& a, hipStream_t) { return keep(dtype, a); }
}  // namespace awa

static awa_ctx ctx;

// want: AWA_EARG with a message and no launch, or AWA_OK with `n` launches
static void check(const char* what, int rc, int want, int n = 1) {
    checks++;
    if (rc != want || launches != (want == AWA_OK ? n : 0) || (want != AWA_OK && ctx.err.empty())) {
        failures++;
        printf("FAILED %s: rc %d (want %d), %d launches, \"%s\"\n", what, rc, want, launches, ctx.err.c_str());
    }
    launches = 0;
    ctx.err.clear();
}
static void hold(const char* what, bool ok) {
    checks++;
    if (!ok) {
        failures++;
        printf("FAILED %s\n", what);
    }
}

int main() {
    // addresses that are only compared, never read
    char* const X = (char*)0x10000000000, *const Y = (char*)0x20000000000, *const Z = (char*)0x30000000000;
    char* const W = (char*)0x40000000000, *const S = (char*)0x60000000000, *const K = (char*)0x70000000000;
    const int bad = AWA_EARG, ok = AWA_OK;
    // a plan whose tables nothing reads
    dit_cross c;
    c.heads = 4; c.kv_heads = 2; c.head_d = 64; c.q_rows = 100; c.k_rows = 50;
    for (int t = 0; t < 2; t++) c.qs[t].block = 128;
    struct A {
        int t = AWA_BF16; dit_heads q, k, v, o, dout, dq, dk, dv; const void* mask = nullptr; float scale = 0.125f; void* lse;
        int64_t ld = 100; void* work; int64_t bytes = 1 << 30;
    };
    A a0{};
    a0.q = {X, 256, 64}; a0.k = {Y, 128, 64}; a0.v = {Z, 128, 64}; a0.o = {W, 256, 64};
    a0.dout = {X + (1 << 30), 256, 64}; a0.dq = {Y + (1 << 30), 256, 64}; a0.dk = {Z + (1 << 30), 128, 64}; a0.dv = {W + (1 << 30), 128, 64};
    a0.lse = S; a0.work = K;
    auto fwd = [&](auto change) {
        A a = a0;
        change(a);
        return dit_cross_forward(&ctx, &c, a.t, &a.q, &a.k, &a.v, (const uint8_t*)a.mask, a.scale, &a.o, (float*)a.lse, a.ld, a.work,
                                 a.bytes, nullptr);
    };
    auto bwd = [&](auto change) {
        A a = a0;
        change(a);
        return dit_cross_grad(&ctx, &c, a.t, &a.dout, &a.q, &a.k, &a.v, &a.o, (const float*)a.lse, a.ld, (const uint8_t*)a.mask,
                              a.scale, &a.dq, &a.dk, &a.dv, a.work, a.bytes, nullptr);
    };

    // ---- DIT_CROSS_WHOLE
    check("forward", fwd([](A&) {}), ok);
    hold("not whole", !last.whole && last_dtype == AWA_BF16);
    check("forward whole", fwd([](A& a) { a.t = AWA_BF16 | DIT_CROSS_WHOLE; }), ok);
    hold("whole", last.whole && last_dtype == AWA_BF16);
    check("forward whole fp32", fwd([](A& a) { a.t = AWA_F32 | DIT_CROSS_WHOLE; }), ok);
    check("gradients whole", bwd([](A& a) { a.t = AWA_BF16 | DIT_CROSS_WHOLE; }), ok, 2);
    hold("gradients whole", last.whole && last_dtype == AWA_BF16);
    check("gradients not whole", bwd([](A&) {}), ok, 2);
    hold("gradients not whole", !last.whole);
    for (int t : {2, 2 | DIT_CROSS_WHOLE, AWA_BF16 | 2 * DIT_CROSS_WHOLE, AWA_BF16 | 3 * DIT_CROSS_WHOLE, -1}) {
        check("forward dtype", fwd([&](A& a) { a.t = t; }), bad);
        check("gradients dtype", bwd([&](A& a) { a.t = t; }), bad);
        hold("work dtype", dit_cross_work(&c, t, 1) < 0);
    }
    for (int t = 0; t < 2; t++)
        for (int grad = 0; grad < 2; grad++)
            hold("work whole", dit_cross_work(&c, t | DIT_CROSS_WHOLE, grad) == dit_cross_work(&c, t, grad) && dit_cross_work(&c, t, grad) >= 0);

    // ---- dropped plans go with the next one's making on their device; captured ones stay
    auto one = [&](int device, int captured) {
        dit_cross* p = new dit_cross;
        p->device = device;
        p->captured = captured;
        dit_cross_drop(p);
        return p;
    };
    one(0, 0);
    dit_cross* const other = one(1, 0);
    dit_cross* const captured = one(0, 1);
    one(0, 0);
    dit_cross_drop(nullptr);
    hold("dropped", dropped().plans.size() == 3 && dropped().plans[1] == other);
    const int64_t none = 0;
    dit_cross* made = nullptr;
    check("a bad plan frees none", dit_cross_create(&ctx, 1, &none, &none, &none, &none, 0, 1, 8, &made), bad);
    hold("a bad plan", dropped().plans.size() == 3);
    check("a plan", dit_cross_create(&ctx, 0, &none, &none, &none, &none, 1, 1, 8, &made), ok, 0);
    hold("freed", made && dropped().plans.size() == 1 && dropped().plans[0] == other);
    dit_cross_destroy(made);
    for (dit_cross* p : take_dropped(1)) dit_cross_destroy(p);
    dit_cross_destroy(captured);
    hold("none left", dropped().plans.empty());

    // ---- outputs beside inputs and each other, in one buffer
    const int64_t F = 1 << 20;  // bytes past which another tensor lies in the same buffer
    // keys' gradients with heads outermost, [2 heads][dk, dv][50 rows][64]
    check("dk, dv by heads", bwd([&](A& a) { a.dk = {Z + (1 << 30), 64, 6400}; a.dv = {Z + (1 << 30) + 6400, 64, 6400}; }), ok, 2);
    check("dk, dv by heads, dv a row early", bwd([&](A& a) { a.dk = {Z + (1 << 30), 64, 6400}; a.dv = {Z + (1 << 30) + 6400 - 128, 64, 6400}; }), bad);
    check("dk, dv by heads, another stride", bwd([&](A& a) { a.dk = {Z + (1 << 30), 64, 6400}; a.dv = {Z + (1 << 30) + 6400, 64, 6408}; }), bad);
    check("out beside v by heads", fwd([&](A& a) { a.q.row = 64; a.o = {Z, 64, 12800}; a.v = {Z + 12800, 64, 12800}; }), ok);
    c.q_rows = 1;  // one query: its stride does not matter
    a0.q.row = a0.o.row = a0.dout.row = a0.dq.row = 0;
    check("one query's gradient beside keys' rows", bwd([&](A& a) {
        a.dk = {Z + F, 512, 64}; a.dv = {Z + F + 256, 512, 64}; a.dq = {Z + F + 512, 0, 64}; }), ok, 2);
    check("one query's gradient over a key's row", bwd([&](A& a) {
        a.dk = {Z + F, 512, 64}; a.dv = {Z + F + 256, 512, 64}; a.dq = {Z + F + 768, 0, 64}; }), bad);
    c.q_rows = 100;
    a0.q.row = a0.o.row = a0.dout.row = a0.dq.row = 256;
    // against the elements themselves: nothing that overlaps is taken, and what lies side by side is
    std::mt19937 rng(3);
    auto upto = [&](int n) { return (int64_t)(rng() % (unsigned)(n + 1)); };
    int taken = 0, apart = 0;
    bool right = true;
    for (int t = 0; t < 200000; t++) {
        const int d = 8, ha = 1 + (int)upto(2), hb = 1 + (int)upto(2);
        const int64_t ra = 1 + upto(3), rb = 1 + upto(3), strides[] = {8, 16, 24, 32, 48, 64, 96};
        const bool same = upto(3) > 0;
        dit_heads a{X + 16 * upto(40), strides[upto(6)], strides[upto(6)]}, b{X + 16 * upto(40), strides[upto(6)], strides[upto(6)]};
        if (same) b.row = a.row, b.head = a.head;
        std::set<char*> in;
        for (int64_t r = 0; r < ra; r++)
            for (int h = 0; h < ha; h++) in.insert((char*)a.p + 2 * (r * a.row + h * a.head));
        bool over = false;
        for (int64_t r = 0; r < rb; r++)
            for (int h = 0; h < hb; h++) over = over || in.count((char*)b.p + 2 * (r * b.row + h * b.head));
        const bool refused = heads_collide(&a, ra, ha, &b, rb, hb, AWA_BF16, d);
        right = right && !(over && !refused) && refused == heads_collide(&b, rb, hb, &a, ra, ha, AWA_BF16, d);
        apart += !over && touches(extent(&a, AWA_BF16, ra, ha, d), extent(&b, AWA_BF16, rb, hb, d));
        taken += !over && !refused && touches(extent(&a, AWA_BF16, ra, ha, d), extent(&b, AWA_BF16, rb, hb, d));
    }
    hold("no overlap is taken", right);
    hold("what lies side by side is", taken > 1000 && taken > apart / 20);

    printf("checks=%d failures=%d\n", checks, failures);
    return failures != 0;
}
