// dit_train.h on the CPU: csrc/dit_train.cpp is included here (its plan's functions too), the launches and the
// shared helpers are the stubs below, so that an accepted call only counts.  Checks refusals, and that the plan
// of many batches covers every pair of a query row and a key once, in slots of its own.  Prints one line per
// failed check.
#include <cstdarg>
#include <cstdio>
#include <limits>
#include <random>
#include <set>

#include "../../seedvr2-2b-ncnn_amd/csrc/dit_train.cpp"

static int launches, failures, checks;

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
hipError_t launch_layer_norm(int, int, const NormFwd&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_layer_norm_grad(int, int, const NormGrad&, hipStream_t) { launches++; return hipSuccess; }
int norm_grad_groups(int M, int) { return std::min(M, 256); }
GradWeightPlan grad_weight_plan(int, int M, int, int) { return {128, 1, 1, M, M >= 1024 ? 1 << 20 : 0}; }
hipError_t launch_grad_weight(int, GradWeight&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_cross_forward(int, const CrossArgs&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_cross_grad_queries(int, const CrossArgs&, hipStream_t) { launches++; return hipSuccess; }
hipError_t launch_cross_grad_keys(int, const CrossArgs&, hipStream_t) { launches++; return hipSuccess; }
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
static void hold(const char* what, bool ok) {
    checks++;
    if (!ok) {
        failures++;
        printf("FAILED %s\n", what);
    }
}

// The tables of a batch against its lengths.
static void check_plan(const std::vector<int64_t>& qa, const std::vector<int64_t>& ql, const std::vector<int64_t>& ka,
                       const std::vector<int64_t>& kl, int heads, int kv_heads, int dtype) {
    Plan p;
    CrossQueries qs;
    CrossKeySide ks;
    plan_queries(qa, ql, ka, kl, heads, kv_heads, 64, dtype, qs, p);
    plan_keys(qa, ql, ka, kl, heads, kv_heads, 64, dtype, ks, p);
    const int per = heads / kv_heads, n = (int)ql.size();
    bool ok = (qs.block == 16 || qs.block == 32 || qs.block == 128) && (qs.pack == 1 || qs.pack == per) && qs.pack <= qs.block &&
              heads % qs.pack == 0 && qs.n_items == (int)p.items.size() && qs.n_joins == (int)p.joins.size();
    // every block of rows of a sequence over its keys, once
    size_t at = 0, join = 0;
    std::set<int> slots;
    for (int i = 0; i < n && ok; i++) {
        int64_t row = 0;
        while (row < ql[i] && ok) {
            int64_t key = 0;
            const int cols = at < p.items.size() ? p.items[at].cols : 0;
            int parts = 0;
            const int first_part = at < p.items.size() ? p.items[at].part : 0;
            do {
                if (at >= p.items.size()) { ok = false; break; }
                const CrossItem& it = p.items[at++];
                ok = ok && it.q0 == qa[i] + row && it.cols == cols && cols > 0 && cols <= qs.block && cols % qs.pack == 0 &&
                     it.k0 == ka[i] + key && it.kn >= 0 && (it.first != 0) == (key == 0) && (it.kn > 0 || kl[i] == 0);
                key += it.kn;
                parts++;
                if (it.part >= 0) ok = ok && it.part == first_part + parts - 1 && it.part < qs.n_parts && slots.insert(it.part).second;
            } while (ok && key < kl[i]);
            ok = ok && key == kl[i] && ((parts > 1) == (first_part >= 0));
            if (ok && parts > 1) {
                ok = join < p.joins.size() && p.joins[join].q0 == qa[i] + row && p.joins[join].cols == cols &&
                     p.joins[join].part0 == first_part && p.joins[join].parts == parts;
                join++;
            }
            row += cols / qs.pack;
        }
        ok = ok && row == std::max<int64_t>(ql[i], 0);
    }
    hold("plan: queries", ok && at == p.items.size() && join == p.joins.size() && (int)slots.size() == qs.n_parts);
    // every block of keys over all query rows of the sequences that have it, for every head of the group, once
    std::map<int64_t, std::pair<int64_t, std::multiset<std::pair<int64_t, int64_t>>>> want;  // key start -> length, rows
    for (int i = 0; i < n; i++)
        if (kl[i]) {
            auto& w = want[ka[i]];
            w.first = kl[i];
            if (ql[i]) w.second.insert({qa[i], ql[i]});
        }
    ok = true;
    std::set<int> kslots;
    size_t kat = 0, kjoin = 0;
    for (auto& w : want) {
        for (int64_t c = 0; c < w.second.first && ok;) {
            if (kat >= p.kitems.size()) { ok = false; break; }
            const CrossKeys f = p.kitems[kat];
            std::vector<int> seen((size_t)f.units * per, 0);
            int parts = 0;
            bool empty = w.second.second.empty();
            while (kat < p.kitems.size() && p.kitems[kat].k0 == f.k0) {
                const CrossKeys& it = p.kitems[kat++];
                // the kernel reads the run's first unit whether the run has any or not
                ok = ok && it.unit0 + it.first % it.units < (int)p.units.size();
                ok = ok && it.k0 == w.first + c && it.kn == f.kn && it.kn > 0 && it.kn <= CROSS_KEYS && it.unit0 == f.unit0 &&
                     it.units == f.units && it.count >= 0 && (empty ? it.count == 0 : it.count > 0);
                for (int u = it.first; ok && u < it.first + it.count; u++) {
                    if (u >= (int)seen.size() || seen[u]++) ok = false;
                }
                if (it.part >= 0) ok = ok && it.part == f.part + parts && it.part < ks.n_parts && kslots.insert(it.part).second;
                parts++;
            }
            ok = ok && (parts > 1) == (f.part >= 0);
            if (!empty)
                for (int s : seen) ok = ok && s == 1;
            if (ok && parts > 1) {
                ok = kjoin < p.kjoins.size() && p.kjoins[kjoin].k0 == f.k0 && p.kjoins[kjoin].kn == f.kn &&
                     p.kjoins[kjoin].part0 == f.part && p.kjoins[kjoin].parts == parts;
                kjoin++;
            }
            // the units are the sequences' rows
            std::multiset<std::pair<int64_t, int64_t>> rows;
            if (!empty)
                for (int u = f.unit0; ok && u < f.unit0 + f.units; u++) {
                    ok = u < (int)p.units.size() && p.units[u].rows > 0 && p.units[u].rows <= CROSS_QT;
                    if (ok) rows.insert({p.units[u].q0, p.units[u].rows});
                }
            int64_t total = 0, have = 0;
            for (auto& r : w.second.second) total += r.second;
            std::vector<std::pair<int64_t, int64_t>> sorted(rows.begin(), rows.end());
            for (size_t u = 0; u < sorted.size(); u++) {
                have += sorted[u].second;
                bool inside = false;
                for (auto& r : w.second.second) inside = inside || (sorted[u].first >= r.first && sorted[u].first + sorted[u].second <= r.first + r.second);
                ok = ok && inside && (u == 0 || sorted[u].first >= sorted[u - 1].first + sorted[u - 1].second);
            }
            ok = ok && have == total;
            c += f.kn;
            ok = ok && c <= w.second.first;
        }
    }
    auto check_spread = [&](auto items, int groups, const Cost& c, auto steps, auto there) {
        const size_t n = items.size() * groups;
        auto list = items;
        const int entries = spread(list, groups, c, steps);
        if (n == 0 || n > CROSS_LISTED) return entries == 0 && list.size() == items.size();
        if (entries != (int)list.size() || entries % 8) return false;
        size_t seen = 0;
        std::vector<int> per_group(groups, 0);
        int64_t work = 0, want_work = 0;
        for (int x = 0; x < 8; x++) {
            int64_t before = INT64_MAX;
            for (int i = x; i < entries; i += 8) {
                if (!there(list[i])) continue;
                if (steps(list[i]) > before || list[i].group < 0 || list[i].group >= groups) return false;
                before = steps(list[i]);
                seen++;
                per_group[list[i].group]++;
                work += steps(list[i]) * (list[i].group + 1) + list[i].k0;
            }
        }
        for (int g = 0; g < groups; g++) {
            if (per_group[g] != (int)items.size()) return false;
            for (auto& it : items) want_work += steps(it) * (g + 1) + it.k0;
        }
        return seen == n && work == want_work;
    };
    hold("plan: queries by workgroup", check_spread(p.items, heads / qs.pack, query_cost(qs.block, dtype, 64),
         [&](const CrossItem& it) { return ceil_div(it.kn, query_step(qs.block)); }, [](const CrossItem& it) { return it.cols > 0; }));
    hold("plan: keys by workgroup", check_spread(p.kitems, kv_heads, key_cost(dtype, 64), [](const CrossKeys& it) { return (int64_t)it.count; },
         [](const CrossKeys& it) { return it.kn > 0; }));
    hold("plan: keys", ok && kat == p.kitems.size() && kjoin == p.kjoins.size() && (int)kslots.size() == ks.n_parts);
}

int main() {
    // addresses that are only compared, never read
    char* const X = (char*)0x10000000000, *const Y = (char*)0x20000000000, *const Z = (char*)0x30000000000;
    char* const W = (char*)0x40000000000, *const B = (char*)0x50000000000, *const S = (char*)0x60000000000;
    char* const K = (char*)0x70000000000;
    const int bad = AWA_EARG, ok = AWA_OK;
    const int64_t big = (int64_t)1 << 40;
    const float nan = std::numeric_limits<float>::quiet_NaN(), inf = std::numeric_limits<float>::infinity();

    // ---- layer norm
    auto norm = [&](int tx, const void* x, int64_t ldx, int ty, void* y, int64_t ldy, void* st, int M, int Kc, float eps = 1e-5f,
                    const void* w = nullptr, const void* b = nullptr) {
        return dit_layer_norm(&ctx, tx, x, ldx, (const float*)w, (const float*)b, eps, ty, y, ldy, (float*)st, M, Kc, nullptr);
    };
    check("norm", norm(AWA_BF16, X, 100, AWA_F32, Y, 100, S, 7, 100), ok);
    check("norm no stats", norm(AWA_F32, X, 100, AWA_F32, Y, 100, nullptr, 7, 100, 0.f, W, B), ok);
    check("norm in place", norm(AWA_F32, X, 100, AWA_F32, X, 100, S, 7, 100), ok);
    check("norm no rows", norm(AWA_F32, nullptr, 100, AWA_F32, nullptr, 100, nullptr, 0, 100), ok, 0);
    check("norm one row, any stride", norm(AWA_F32, X, 0, AWA_F32, Y, -5, nullptr, 1, 100), ok);
    check("norm unaligned", norm(AWA_BF16, X + 2, 101, AWA_BF16, Y + 2, 103, S, 7, 100), ok);
    check("norm most columns", norm(AWA_BF16, X, DIT_NORM_COLS_MAX, AWA_BF16, Y, DIT_NORM_COLS_MAX, S, 7, DIT_NORM_COLS_MAX), ok);
    check("norm null ctx", (ctx.err = "-", dit_layer_norm(nullptr, 0, X, 1, nullptr, nullptr, 0.f, 0, Y, 1, nullptr, 1, 1, nullptr)), bad);
    check("norm too many columns", norm(AWA_BF16, X, 20000, AWA_BF16, Y, 20000, S, 7, DIT_NORM_COLS_MAX + 1), bad);
    check("norm no columns", norm(AWA_BF16, X, 20, AWA_BF16, Y, 20, S, 7, 0), bad);
    check("norm rows < 0", norm(AWA_BF16, X, 20, AWA_BF16, Y, 20, S, -1, 20), bad);
    check("norm too many rows", norm(AWA_BF16, X, 20, AWA_BF16, Y, 20, S, DIT_OPS_ROWS_MAX + 1, 20), bad);
    check("norm 8-bit x", norm(DIT_FP8, X, 128, AWA_BF16, Y, 128, S, 7, 128), bad);
    check("norm type", norm(AWA_BF16, X, 128, 3, Y, 128, S, 7, 128), bad);
    for (float e : {-1e-9f, nan, inf}) check("norm eps", norm(AWA_F32, X, 100, AWA_F32, Y, 100, S, 7, 100, e), bad);
    check("norm null x", norm(AWA_F32, nullptr, 100, AWA_F32, Y, 100, S, 7, 100), bad);
    check("norm null y", norm(AWA_F32, X, 100, AWA_F32, nullptr, 100, S, 7, 100), bad);
    check("norm misaligned x", norm(AWA_F32, X + 2, 100, AWA_F32, Y, 100, S, 7, 100), bad);
    check("norm misaligned stats", norm(AWA_F32, X, 100, AWA_F32, Y, 100, S + 4, 7, 100), bad);
    check("norm misaligned w", norm(AWA_F32, X, 100, AWA_F32, Y, 100, S, 7, 100, 0.f, W + 1), bad);
    check("norm ldx", norm(AWA_F32, X, 99, AWA_F32, Y, 100, S, 7, 100), bad);
    check("norm ldy", norm(AWA_F32, X, 100, AWA_F32, Y, 99, S, 7, 100), bad);
    check("norm far ldx", norm(AWA_F32, X, big, AWA_F32, Y, 100, S, 7, 100), bad);
    check("norm partly over x", norm(AWA_F32, X, 100, AWA_F32, X + 400, 100, S, 7, 100), bad);
    check("norm over x, other stride", norm(AWA_F32, X, 100, AWA_F32, X, 101, S, 7, 100), bad);
    check("norm over x, other type", norm(AWA_F32, X, 100, AWA_BF16, X, 100, S, 7, 100), bad);
    check("norm over w", norm(AWA_F32, X, 100, AWA_F32, Y, 100, S, 7, 100, 0.f, Y + 40), bad);
    check("norm stats over x", norm(AWA_F32, X, 100, AWA_F32, X, 100, X + 8, 7, 100), bad);
    check("norm stats over y", norm(AWA_F32, X, 100, AWA_F32, Y, 100, Y + 8, 7, 100), bad);

    // ---- its gradient
    struct G {
        int tdy = AWA_BF16; const void* dy; int64_t lddy = 100; int tx = AWA_F32; const void* x; int64_t ldx = 100;
        const void* xs = nullptr; int64_t ld_xs = 0; const void* st; const void* w = nullptr; int tdx = AWA_F32; void* dx;
        int64_t lddx = 100; void* dw; void* db; void* work; int64_t bytes = 1 << 30; int M = 7, Kc = 100;
    };
    G g0{};
    g0.dy = X; g0.x = Y; g0.st = S; g0.dx = Z; g0.dw = W; g0.db = B; g0.work = K;
    auto grad = [&](auto change) {
        G g = g0;
        change(g);
        return dit_layer_norm_grad(&ctx, g.tdy, g.dy, g.lddy, g.tx, g.x, g.ldx, (const uint32_t*)g.xs, g.ld_xs, (const float*)g.st,
                                   (const float*)g.w, g.tdx, g.dx, g.lddx, (float*)g.dw, (float*)g.db, g.work, g.bytes, g.M, g.Kc, nullptr);
    };
    auto saved = [&](G& g) { g.tx = DIT_FP8; g.ldx = 0; g.xs = (char*)0x80000000000; g.ld_xs = 7; };
    check("grad", grad([](G&) {}), ok);
    check("grad saved", grad([&](G& g) { saved(g); }), ok);
    check("grad dx alone", grad([](G& g) { g.dw = g.db = g.work = nullptr; g.bytes = 0; }), ok);
    check("grad dw alone", grad([](G& g) { g.dx = nullptr; g.db = nullptr; g.tdx = 77; g.lddx = 0; }), ok);
    check("grad no rows", grad([](G& g) { g.M = 0; g.work = nullptr; g.dy = g.x = g.st = nullptr; }), ok);
    check("grad no rows, dx alone", grad([](G& g) { g.M = 0; g.dw = g.db = nullptr; }), ok, 0);
    check("grad over dy", grad([&](G& g) { g.tdy = AWA_F32; g.dx = X; }), ok);
    check("grad over x", grad([&](G& g) { g.dx = Y; }), ok);
    check("grad exact work", grad([&](G& g) { g.bytes = dit_layer_norm_grad_work(7, 100); }), ok);
    check("grad no output", grad([](G& g) { g.dx = g.dw = g.db = nullptr; }), bad);
    check("grad saved without scales", grad([&](G& g) { saved(g); g.xs = nullptr; }), bad);
    check("grad scales without saved", grad([&](G& g) { g.xs = K; }), bad);
    check("grad ld_xs", grad([&](G& g) { saved(g); g.ld_xs = 6; }), bad);
    check("grad misaligned saved", grad([&](G& g) { saved(g); g.x = Y + 8; }), bad);
    check("grad little work", grad([&](G& g) { g.bytes = dit_layer_norm_grad_work(7, 100) - 1; }), bad);
    check("grad no work", grad([](G& g) { g.work = nullptr; }), bad);
    check("grad misaligned work", grad([&](G& g) { g.work = K + 128; }), bad);
    check("grad null dy", grad([](G& g) { g.dy = nullptr; }), bad);
    check("grad null stats", grad([](G& g) { g.st = nullptr; }), bad);
    check("grad columns", grad([](G& g) { g.Kc = DIT_NORM_COLS_MAX + 1; }), bad);
    check("grad rows", grad([](G& g) { g.M = -1; }), bad);
    check("grad type dy", grad([](G& g) { g.tdy = DIT_FP8; }), bad);
    check("grad type dx", grad([](G& g) { g.tdx = DIT_FP8; }), bad);
    check("grad lddy", grad([](G& g) { g.lddy = 99; }), bad);
    check("grad ldx", grad([](G& g) { g.ldx = 99; }), bad);
    check("grad lddx", grad([](G& g) { g.lddx = 99; }), bad);
    check("grad dx over dy, other type", grad([&](G& g) { g.dx = X; }), bad);
    check("grad dx partly over x", grad([&](G& g) { g.dx = Y + 4; }), bad);
    check("grad dx over stats", grad([&](G& g) { g.dx = S; }), bad);
    check("grad dw over db", grad([&](G& g) { g.db = g.dw; }), bad);
    check("grad dw over w", grad([&](G& g) { g.w = W + 4; }), bad);
    check("grad dw over dx", grad([&](G& g) { g.dw = Z + 400; }), bad);
    check("grad work over dy", grad([&](G& g) { g.work = X; }), bad);
    hold("grad work sizes", dit_layer_norm_grad_work(-1, 5) < 0 && dit_layer_norm_grad_work(5, 0) < 0 && dit_layer_norm_grad_work(0, 5) == 0);

    // ---- weight
    struct D {
        int tdy = AWA_BF16; const void* dy; int64_t lddy = 50; const void* q; const void* s; int64_t ld_s = 7; int tw = AWA_F32;
        void* dw; int64_t ldw = 100; void* db; int add = 0; void* work = nullptr; int64_t bytes = 0; int M = 7, N = 50, Kc = 100;
    };
    D d0{};
    d0.dy = X; d0.q = Y; d0.s = S; d0.dw = W; d0.db = B;
    auto weight = [&](auto change) {
        D d = d0;
        change(d);
        return dit_grad_weight_fp8(&ctx, d.tdy, d.dy, d.lddy, (const uint8_t*)d.q, (const uint32_t*)d.s, d.ld_s, d.tw, d.dw, d.ldw,
                                   (float*)d.db, d.add, d.work, d.bytes, d.M, d.N, d.Kc, nullptr);
    };
    check("weight", weight([](D&) {}), ok);
    check("weight no db", weight([](D& d) { d.db = nullptr; }), ok);
    check("weight no rows", weight([](D& d) { d.M = 0; d.dy = d.q = d.s = nullptr; }), ok);
    check("weight added", weight([](D& d) { d.add = 1; }), ok);
    check("weight one row of dW", weight([](D& d) { d.N = 1; d.ldw = 0; }), ok);
    check("weight with work", weight([&](D& d) { d.M = 2000; d.ld_s = 2000; d.work = K; d.bytes = dit_grad_weight_work(1, 0, 2000, 50, 100); }), ok);
    check("weight little work", weight([&](D& d) { d.M = 2000; d.ld_s = 2000; d.work = K; d.bytes = dit_grad_weight_work(1, 0, 2000, 50, 100) - 1; }), bad);
    check("weight added in bf16", weight([](D& d) { d.add = 1; d.tw = AWA_BF16; }), bad);
    check("weight type", weight([](D& d) { d.tdy = DIT_FP8; }), bad);
    check("weight null dW", weight([](D& d) { d.dw = nullptr; }), bad);
    check("weight null dy", weight([](D& d) { d.dy = nullptr; }), bad);
    check("weight misaligned q", weight([&](D& d) { d.q = Y + 8; }), bad);
    check("weight misaligned dy", weight([&](D& d) { d.dy = X + 1; }), bad);
    check("weight lddy", weight([](D& d) { d.lddy = 49; }), bad);
    check("weight far lddy", weight([](D& d) { d.lddy = DIT_OPS_COLS_MAX + 1; }), bad);
    check("weight ldw", weight([](D& d) { d.ldw = 99; }), bad);
    check("weight ld_s", weight([](D& d) { d.ld_s = 6; }), bad);
    check("weight N", weight([](D& d) { d.N = 0; }), bad);
    check("weight K", weight([](D& d) { d.Kc = DIT_OPS_COLS_MAX + 1; }), bad);
    check("weight M", weight([](D& d) { d.M = DIT_OPS_ROWS_MAX + 1; }), bad);
    check("weight dW over dy", weight([&](D& d) { d.dw = X; }), bad);
    check("weight dW over q", weight([&](D& d) { d.dw = Y + 512; }), bad);
    check("weight db over dW", weight([&](D& d) { d.db = W + 16; }), bad);
    hold("weight work sizes", dit_grad_weight_work(2, 0, 5, 5, 5) < 0 && dit_grad_weight_work(0, 0, 5, 0, 5) < 0 &&
                                  dit_grad_weight_work(0, 0, 5, 5, 5) == 0);

    // ---- plans: refusals (an accepted one would need a device)
    auto plan = [&](std::vector<int64_t> qa, std::vector<int64_t> ql, std::vector<int64_t> ka, std::vector<int64_t> kl, int h, int hk,
                    int hd) {
        dit_cross* p = nullptr;
        const int rc = dit_cross_create(&ctx, (int)qa.size(), qa.data(), ql.data(), ka.data(), kl.data(), h, hk, hd, &p);
        if (p) dit_cross_destroy(p);
        return rc;
    };
    check("plan heads", plan({0}, {1}, {0}, {1}, 0, 1, 64), bad);
    check("plan kv_heads", plan({0}, {1}, {0}, {1}, 4, 3, 64), bad);
    check("plan no kv_heads", plan({0}, {1}, {0}, {1}, 4, 0, 64), bad);
    check("plan most heads", plan({0}, {1}, {0}, {1}, DIT_CROSS_HEADS_MAX + 1, 1, 64), bad);
    for (int hd : {0, -8, 4, 12, 136, 256}) check("plan head_d", plan({0}, {1}, {0}, {1}, 4, 2, hd), bad);
    check("plan negative", plan({-1}, {1}, {0}, {1}, 4, 2, 64), bad);
    check("plan negative length", plan({0}, {1}, {0}, {-1}, 4, 2, 64), bad);
    check("plan rows", plan({DIT_OPS_ROWS_MAX}, {1}, {0}, {1}, 4, 2, 64), bad);
    check("plan far rows", plan({0}, {1}, {std::numeric_limits<int64_t>::max()}, {1}, 4, 2, 64), bad);
    check("plan far length", plan({0}, {std::numeric_limits<int64_t>::max()}, {0}, {1}, 4, 2, 64), bad);
    check("plan queries overlap", plan({0, 3}, {4, 4}, {0, 9}, {9, 9}, 4, 2, 64), bad);
    check("plan same queries", plan({0, 0}, {4, 4}, {0, 9}, {9, 9}, 4, 2, 64), bad);
    check("plan keys overlap", plan({0, 4}, {4, 4}, {0, 5}, {9, 9}, 4, 2, 64), bad);
    check("plan keys of one start", plan({0, 4}, {4, 4}, {0, 0}, {9, 8}, 4, 2, 64), bad);
    {  // a launch has fewer than 2^32 threads
        std::vector<int64_t> at(DIT_CROSS_SEQ_MAX), one(at.size(), 1), none(at.size(), 0);
        for (size_t i = 0; i < at.size(); i++) at[i] = (int64_t)i;
        check("plan blocks of queries", plan(at, one, none, none, 1024, 1024, 8), bad);
        check("plan blocks of keys", plan(none, none, at, one, 1024, 1024, 8), bad);
    }
    check("plan null out", dit_cross_create(&ctx, 0, nullptr, nullptr, nullptr, nullptr, 1, 1, 8, nullptr), bad);
    check("plan null lengths", plan({}, {}, {}, {}, 0, 1, 8), bad);

    // ---- the attention's calls, on a plan whose tables nothing reads
    dit_cross c;
    c.heads = 4; c.kv_heads = 2; c.head_d = 64; c.q_rows = 100; c.k_rows = 50;
    for (int t = 0; t < 2; t++) c.qs[t].block = 128;
    const int64_t row = 4 * 64;
    struct A {
        int t = AWA_BF16; dit_heads q, k, v, o, dout, dq, dk, dv; const void* mask = nullptr; float scale = 0.125f; void* lse;
        int64_t ld = 100; void* work; int64_t bytes = 1 << 30;
        const dit_cross* plan;
    };
    A a0{};
    a0.plan = &c;
    a0.q = {X, row, 64}; a0.k = {Y, 128, 64}; a0.v = {Z, 128, 64}; a0.o = {W, row, 64};
    a0.dout = {X + (1 << 30), row, 64}; a0.dq = {Y + (1 << 30), row, 64}; a0.dk = {Z + (1 << 30), 128, 64}; a0.dv = {W + (1 << 30), 128, 64};
    a0.lse = S; a0.work = K;
    auto fwd = [&](auto change) {
        A a = a0;
        change(a);
        return dit_cross_forward(&ctx, a.plan, a.t, &a.q, &a.k, &a.v, (const uint8_t*)a.mask, a.scale, &a.o, (float*)a.lse, a.ld, a.work,
                                 a.bytes, nullptr);
    };
    auto bwd = [&](auto change) {
        A a = a0;
        change(a);
        return dit_cross_grad(&ctx, a.plan, a.t, &a.dout, &a.q, &a.k, &a.v, &a.o, (const float*)a.lse, a.ld, (const uint8_t*)a.mask,
                              a.scale, &a.dq, &a.dk, &a.dv, a.work, a.bytes, nullptr);
    };
    check("cross", fwd([](A&) {}), ok);
    check("cross no lse", fwd([](A& a) { a.lse = nullptr; a.ld = 0; }), ok);
    check("cross beside one another", fwd([&](A& a) { a.o = {X + 512, 512, 64}; a.q = {X, 512, 64}; }), ok);
    check("cross heads outermost", fwd([](A& a) { a.q.row = 64; a.q.head = 6400; a.o.row = 64; a.o.head = 6400; }), ok);
    check("cross null plan", fwd([](A& a) { a.plan = nullptr; }), bad);
    check("cross type", fwd([](A& a) { a.t = DIT_FP8; }), bad);
    for (float s : {0.f, -1.f, 1e-31f, 2e30f, nan, inf}) check("cross scale", fwd([&](A& a) { a.scale = s; }), bad);
    check("cross ld_lse", fwd([](A& a) { a.ld = 99; }), bad);
    check("cross null q", fwd([](A& a) { a.q.p = nullptr; }), bad);
    check("cross misaligned k", fwd([&](A& a) { a.k.p = Y + 8; }), bad);
    check("cross k row stride", fwd([](A& a) { a.k.row = 132; }), bad);
    check("cross v head stride", fwd([](A& a) { a.v.head = 68; }), bad);
    check("cross negative stride", fwd([](A& a) { a.q.row = -256; }), bad);
    check("cross far rows", fwd([](A& a) { a.k.row = 2 * DIT_OPS_COLS_MAX; }), bad);
    check("cross out rows coincide", fwd([](A& a) { a.o.row = 0; }), bad);
    check("cross out heads coincide", fwd([](A& a) { a.o.head = 32; }), bad);
    check("cross out rows over heads", fwd([](A& a) { a.o.row = 128; a.o.head = 64; }), bad);
    check("cross out over q", fwd([&](A& a) { a.o = a.q; }), bad);
    check("cross out over v", fwd([&](A& a) { a.o.p = Z + 1024; }), bad);
    check("cross lse over out", fwd([&](A& a) { a.lse = W; }), bad);
    check("cross misaligned lse", fwd([&](A& a) { a.lse = S + 2; }), bad);
    check("cross out over mask", fwd([&](A& a) { a.mask = W + 5; }), bad);
    c.qs[AWA_BF16].n_parts = 3;
    check("cross work", fwd([&](A& a) { a.bytes = dit_cross_work(&c, AWA_BF16, 0); }), ok);
    check("cross little work", fwd([&](A& a) { a.bytes = dit_cross_work(&c, AWA_BF16, 0) - 1; }), bad);
    check("cross no work", fwd([](A& a) { a.work = nullptr; }), bad);
    check("cross work over q", fwd([&](A& a) { a.work = X; }), bad);
    check("cross_grad", bwd([](A&) {}), ok, 2);
    check("cross_grad exact work", bwd([&](A& a) { a.bytes = dit_cross_work(&c, AWA_BF16, 1); }), ok, 2);
    check("cross_grad little work", bwd([&](A& a) { a.bytes = dit_cross_work(&c, AWA_BF16, 1) - 1; }), bad);
    check("cross_grad dk, dv side by side", bwd([&](A& a) { a.dk = {Z + (1 << 30), 256, 64}; a.dv = {Z + (1 << 30) + 256, 256, 64}; }), ok, 2);
    check("cross_grad null lse", bwd([](A& a) { a.lse = nullptr; }), bad);
    check("cross_grad null dq", bwd([](A& a) { a.dq.p = nullptr; }), bad);
    check("cross_grad dk over dv", bwd([&](A& a) { a.dv = a.dk; }), bad);
    check("cross_grad dq over dout", bwd([&](A& a) { a.dq = a.dout; }), bad);
    check("cross_grad dk over k", bwd([&](A& a) { a.dk.p = Y; }), bad);
    check("cross_grad dq over lse", bwd([&](A& a) { a.dq.p = S; }), bad);
    check("cross_grad work over out", bwd([&](A& a) { a.work = W; }), bad);
    // one description for an input and a gradient
    check("cross_grad dq is q", dit_cross_grad(&ctx, &c, AWA_BF16, &a0.dout, &a0.q, &a0.k, &a0.v, &a0.o, (const float*)S, 100, nullptr, 1.f,
                                               &a0.q, &a0.dk, &a0.dv, K, 1 << 30, nullptr), bad);
    check("cross_grad dk is k", dit_cross_grad(&ctx, &c, AWA_BF16, &a0.dout, &a0.q, &a0.k, &a0.v, &a0.o, (const float*)S, 100, nullptr, 1.f,
                                               &a0.dq, &a0.k, &a0.dv, K, 1 << 30, nullptr), bad);
    check("cross_grad dv is dk", dit_cross_grad(&ctx, &c, AWA_BF16, &a0.dout, &a0.q, &a0.k, &a0.v, &a0.o, (const float*)S, 100, nullptr, 1.f,
                                                &a0.dq, &a0.dk, &a0.dk, K, 1 << 30, nullptr), bad);
    check("cross_grad dv rows coincide", bwd([](A& a) { a.dv.row = 64; }), bad);
    check("cross_grad misaligned dout", bwd([&](A& a) { a.dout.p = X + 4; }), bad);
    ctx.device = 1;
    check("cross plan of another device", fwd([](A&) {}), bad);
    ctx.device = 0;
    c.k_rows = 0;
    check("cross no keys", fwd([](A& a) { a.k.p = a.v.p = nullptr; }), ok);
    check("cross_grad no keys", bwd([](A& a) { a.k.p = a.v.p = a.dk.p = a.dv.p = nullptr; }), ok, 2);
    c.k_rows = 50; c.q_rows = 0;
    check("cross no queries", fwd([](A& a) { a.q.p = a.o.p = nullptr; }), ok, 0);
    check("cross_grad no queries", bwd([](A& a) { a.q.p = a.o.p = a.dq.p = a.dout.p = a.lse = nullptr; }), ok, 2);
    hold("cross work sizes", dit_cross_work(nullptr, 0, 0) < 0 && dit_cross_work(&c, 2, 0) < 0);

    // ---- plans of many batches
    std::mt19937 rng(5);
    auto upto = [&](int n) { return (int64_t)(rng() % (unsigned)(n + 1)); };
    for (int t = 0; t < 400; t++) {
        const int n = (int)upto(t % 4 == 0 ? 40 : 5), hk = 1 + (int)upto(5), h = hk * (1 << upto(t % 7 == 0 ? 6 : 2));
        const int mq = (int[]){1, 3, 40, 700, 9000}[upto(4)], mk = (int[]){1, 50, 64, 300, 5000}[upto(4)];
        std::vector<int64_t> qa, ql, ka, kl;
        int64_t q = upto(9), k = upto(9);
        for (int i = 0; i < n; i++) {
            ql.push_back(upto(mq));
            qa.push_back(q);
            q += ql.back() + upto(3);
            if (i && upto(3) == 0) {
                ka.push_back(ka.back());
                kl.push_back(kl.back());
            } else {
                kl.push_back(upto(mk));
                ka.push_back(k);
                k += kl.back() + upto(3);
            }
        }
        check_plan(qa, ql, ka, kl, h, hk, t & 1);
    }
    check_plan({0}, {1 << 24}, {0}, {200}, 4, 1, AWA_BF16);
    check_plan({0}, {1}, {0}, {1 << 24}, 1024, 1, AWA_F32);

    printf("checks=%d failures=%d\n", checks, failures);
    return failures != 0;
}
