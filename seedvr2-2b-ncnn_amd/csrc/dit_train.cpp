// dit_train.cpp — C ABI of the operators of dit_train.h: argument checks, the attention's plan, launches.
#include <algorithm>
#include <cmath>
#include <exception>
#include <map>
#include <mutex>
#include <vector>

#include "dit_train_internal.hpp"

using namespace awa;

// Lengths of a batch and the work that they make, on the device.
struct dit_cross {
    int device = 0;
    int heads = 0, kv_heads = 0, head_d = 0;
    int64_t q_rows = 0, k_rows = 0;  // past the last row of any sequence
    void* tables = nullptr;
    mutable int captured = 0;  // a graph holds a call that reads the tables
    // for AWA_F32 and AWA_BF16, whose work is worth dividing differently
    CrossQueries qs[2];
    CrossKeySide ks[2];
};

namespace {

bool dtype_ok(int dtype) { return dtype == AWA_F32 || dtype == AWA_BF16; }
size_t elem(int dtype) { return dtype == AWA_F32 ? 4 : 2; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t groups_of(int k) { return ((int64_t)k + 511) / 512; }
int padded(int k) { return (k + DIT_FP8_BLOCK - 1) / DIT_FP8_BLOCK * DIT_FP8_BLOCK; }
constexpr int64_t STRIDE_MAX = (int64_t)1 << 36;
constexpr int64_t ALIGN = 256;
int64_t align_up(int64_t x) { return (x + ALIGN - 1) / ALIGN * ALIGN; }
// bytes from the first to past the last element of rows ld elements apart
size_t span(int64_t rows, int64_t ld, int64_t cols, size_t size) {
    return rows > 0 ? (size_t)((rows - 1) * ld + cols) * size : 0;
}
bool stride_ok(int M, int64_t ld, int K) { return M <= 1 || (ld >= K && ld <= STRIDE_MAX); }

// An extent of memory that a call reads or writes.
struct Extent {
    const void* p;
    size_t bytes;
};
bool touches(const Extent& a, const Extent& b) { return a.p && b.p && a.bytes && b.bytes && overlaps(a.p, a.bytes, b.p, b.bytes); }
// whether an output lies over another output or an input
bool collide(const std::initializer_list<Extent>& outs, const std::initializer_list<Extent>& ins) {
    for (auto o = outs.begin(); o != outs.end(); o++) {
        for (auto p = outs.begin(); p != o; p++)
            if (touches(*o, *p)) return true;
        for (const Extent& i : ins)
            if (touches(*o, i)) return true;
    }
    return false;
}
int work_ok(awa_ctx* ctx, const char* who, const void* work, int64_t have, int64_t need) {
    if (need > 0 && (!work || have < need || !aligned(work, ALIGN))) {
        set_err(ctx, "%s: d_work must be %lld bytes, %lld-byte aligned (got %lld)", who, (long long)need, (long long)ALIGN,
                (long long)(work ? have : 0));
        return AWA_EARG;
    }
    return AWA_OK;
}

bool norm_sizes_ok(int M, int K) { return M >= 0 && M <= DIT_OPS_ROWS_MAX && K >= 1 && K <= DIT_NORM_COLS_MAX; }
bool weight_sizes_ok(int M, int N, int K) {
    return M >= 0 && M <= DIT_OPS_ROWS_MAX && N >= 1 && N <= DIT_OPS_COLS_MAX && K >= 1 && K <= DIT_OPS_COLS_MAX;
}
int64_t weight_work(int dtype_dy, int M, int N, int K) { return align_up(grad_weight_plan(dtype_dy, M, N, K).work); }

// ---- the attention's plan

struct Plan {
    std::vector<CrossItem> items;
    std::vector<CrossJoin> joins;
    std::vector<CrossKeys> kitems;
    std::vector<CrossKeyJoin> kjoins;
    std::vector<CrossUnit> units;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How far to divide the long axis of each block's work: the number of runs with the least estimated time, of a chip that
// takes `slots` workgroups at once, each t0 and t1 a step of its run, and then joins `part` bytes of each run (written and
// read).  `blocks`: how many blocks have how many steps.
struct Cost {
    int64_t slots;
    double t0, t1, join, part;  // us, us, us, bytes
};
int64_t runs_of(const std::map<int64_t, int64_t>& blocks, const Cost& c) {
    int64_t most = 0, best = 1;
    for (const auto& b : blocks) most = std::max(most, b.first);
    double least = 0;
    for (int64_t runs = 1; runs <= std::min<int64_t>(most, 64); runs++) {
        const int64_t run = ceil_div(most, runs);
        int64_t total = 0, parts = 0;
        for (const auto& b : blocks) {
            const int64_t n = std::max<int64_t>(1, ceil_div(b.first, run));
            total += b.second * n;
            if (n > 1) parts += b.second * n;
        }
        const double t = (double)ceil_div(total, c.slots) * (c.t0 + c.t1 * (double)run) +
                         (parts ? c.join + 2.0 * c.part * (double)parts / 4e6 : 0.0);
        if (runs == 1 || t < least) {
            least = t;
            best = runs;
        }
    }
    return most > 0 ? ceil_div(most, best) : 1;  // steps of a run
}

// A step is 64 keys, or 128 for the waves of a block of few columns.  Measured with heads of 128 channels: in bf16 a
// block of 128 columns takes 6 us and 1.6 a step where two share a CU, one of few columns 4 us and 1.5 a step; in fp32,
// one workgroup a CU, 8 us and 8 a step, and 4 us and 3.
int64_t query_step(int block) { return block < 128 ? 128 : 64; }
Cost query_cost(int block, int dtype, int head_d) {
    const bool few = block < 128, f32 = dtype == AWA_F32;
    return {few || f32 ? 256 : 512, few ? 4.0 : f32 ? 8.0 : 6.0, few ? (f32 ? 3.0 : 1.5) : f32 ? 8.0 : 1.6, 5.0, 4.0 * block * head_d};
}

void plan_queries(const std::vector<int64_t>& qa, const std::vector<int64_t>& ql, const std::vector<int64_t>& ka,
                  const std::vector<int64_t>& kl, int heads, int kv_heads, int head_d, int dtype, CrossQueries& s, Plan& p) {
    const int per = heads / kv_heads;
    int64_t most = per;
    for (int64_t n : ql) most = std::max(most, n * per);
    // Few columns: the heads that share a key head in one block, so that its keys are read once.
    s.block = most <= 16 ? 16 : most <= 32 ? 32 : 128;
    s.pack = s.block < 128 ? per : 1;
    const int rows = s.block / s.pack;
    const int64_t groups = heads / s.pack, step = query_step(s.block);
    std::map<int64_t, int64_t> made;
    for (size_t i = 0; i < ql.size(); i++)
        if (ql[i]) made[ceil_div(kl[i], step)] += ceil_div(ql[i], rows) * groups;
    const Cost cost = query_cost(s.block, dtype, head_d);
    const int64_t run = runs_of(made, cost) * step;
    for (size_t i = 0; i < ql.size(); i++) {
        for (int64_t r = 0; r < ql[i]; r += rows) {
            const int n = (int)std::min<int64_t>(rows, ql[i] - r) * s.pack;
            const int parts = (int)std::max<int64_t>(1, (kl[i] + run - 1) / run), first = s.n_parts;
            for (int c = 0; c < parts; c++) {
                CrossItem it{};
                it.q0 = (int)(qa[i] + r);
                it.cols = n;
                it.k0 = (int)(ka[i] + c * run);
                it.kn = (int)std::min(run, kl[i] - c * run);
                it.part = parts > 1 ? first + c : -1;
                it.first = c == 0;
                s.most_keys = std::max(s.most_keys, it.kn);
                p.items.push_back(it);
            }
            if (parts > 1) {
                p.joins.push_back({(int)(qa[i] + r), n, first, parts});
                s.n_parts += parts;
            }
        }
    }
    s.n_items = (int)p.items.size();
    s.n_joins = (int)p.joins.size();
}

// A step is a unit.  Measured as above: in bf16 a block takes 5 us and 2 a unit where two share a CU, in fp32 8 and 8.
Cost key_cost(int dtype, int head_d) {
    return dtype == AWA_F32 ? Cost{256, 8.0, 8.0, 5.0, 8.0 * CROSS_KEYS * head_d} : Cost{512, 5.0, 2.0, 5.0, 8.0 * CROSS_KEYS * head_d};
}

void plan_keys(const std::vector<int64_t>& qa, const std::vector<int64_t>& ql, const std::vector<int64_t>& ka,
               const std::vector<int64_t>& kl, int heads, int kv_heads, int head_d, int dtype, CrossKeySide& s, Plan& p) {
    const int per = heads / kv_heads;
    // sequences by their keys
    std::map<int64_t, std::vector<size_t>> shared;
    for (size_t i = 0; i < kl.size(); i++)
        if (kl[i]) shared[ka[i]].push_back(i);
    std::map<int64_t, int64_t> made;
    for (auto& e : shared) {
        int64_t units = 0;
        for (size_t i : e.second) units += ceil_div(ql[i], CROSS_QT);
        made[units * per] += ceil_div(kl[e.second[0]], CROSS_KEYS) * kv_heads;
    }
    const int64_t run = runs_of(made, key_cost(dtype, head_d));
    for (auto& e : shared) {
        const int unit0 = (int)p.units.size();
        for (size_t i : e.second)
            for (int64_t r = 0; r < ql[i]; r += CROSS_QT)
                p.units.push_back({(int)(qa[i] + r), (int)std::min<int64_t>(CROSS_QT, ql[i] - r)});
        const int units = (int)p.units.size() - unit0;
        const int64_t all = (int64_t)units * per, n = kl[e.second[0]];
        for (int64_t c = 0; c < n; c += CROSS_KEYS) {
            const int kn = (int)std::min<int64_t>(CROSS_KEYS, n - c), k0 = (int)(e.first + c);
            const int parts = (int)std::max<int64_t>(1, (all + run - 1) / run), first = s.n_parts;
            for (int i = 0; i < parts; i++) {
                CrossKeys it{};
                it.k0 = k0;
                it.kn = kn;
                it.unit0 = unit0;
                it.units = std::max(units, 1);
                it.first = (int)(i * run);
                it.count = (int)std::min(run, all - i * run);
                it.part = parts > 1 ? first + i : -1;
                p.kitems.push_back(it);
            }
            if (parts > 1) {
                p.kjoins.push_back({k0, kn, first, parts});
                s.n_parts += parts;
            }
        }
    }
    // a run without units still reads one: the table has one past the last
    if (!p.kitems.empty()) p.units.push_back({0, 0});
    s.n_items = (int)p.kitems.size();
    s.n_joins = (int)p.kjoins.size();
}

// Items as a table by workgroup (see CrossQueries), or as they are.  steps(item): its run's; an entry without work is Item{}.
template <typename Item, typename Steps>
int spread(std::vector<Item>& items, int groups, const Cost& c, Steps steps) {
    const int64_t n = (int64_t)items.size() * groups;
    if (n == 0 || n > CROSS_LISTED) return 0;
    auto cost = [&](const Item& it) { return c.t0 + c.t1 * (double)steps(it); };
    double all = 0, at = 0;
    for (const Item& it : items) all += cost(it) * groups;
    std::vector<Item> lists[8];
    for (int g = 0; g < groups; g++)
        for (const Item& it : items) {
            const double w = cost(it);
            lists[std::min(7, (int)((at + 0.5 * w) / all * 8.0))].push_back(it);
            lists[std::min(7, (int)((at + 0.5 * w) / all * 8.0))].back().group = g;
            at += w;
        }
    size_t longest = 0;
    for (auto& l : lists) {
        std::stable_sort(l.begin(), l.end(), [&](const Item& a, const Item& b) { return steps(a) > steps(b); });
        longest = std::max(longest, l.size());
    }
    items.assign(8 * longest, Item{});
    for (int x = 0; x < 8; x++)
        for (size_t i = 0; i < lists[x].size(); i++) items[8 * i + x] = lists[x][i];
    return (int)items.size();
}

// Whether ranges [at, at + len) of which `same` may coincide, but not overlap otherwise, do so; empty ones do not count.
bool ranges_ok(const std::vector<int64_t>& at, const std::vector<int64_t>& len, bool same) {
    std::vector<std::pair<int64_t, int64_t>> r;
    for (size_t i = 0; i < at.size(); i++)
        if (len[i]) r.push_back({at[i], len[i]});
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); i++)
        if (r[i].first < r[i - 1].first + r[i - 1].second && !(same && r[i] == r[i - 1])) return false;
    return true;
}

// Plans of dit_cross_drop, for the next plan's making to free.  Never destroyed: a plan may be dropped while the process ends.
struct Dropped {
    std::mutex lock;
    std::vector<dit_cross*> plans;
};
Dropped& dropped() {
    static Dropped* const d = new Dropped;
    return *d;
}
std::vector<dit_cross*> take_dropped(int device) {
    std::vector<dit_cross*> out, keep;
    std::lock_guard<std::mutex> hold(dropped().lock);
    for (dit_cross* p : dropped().plans) (p->device == device ? out : keep).push_back(p);
    dropped().plans.swap(keep);
    return out;
}

// notes that a graph takes a call in (the default stream cannot be captured, and is not to be asked while another one is)
void note_capture(const dit_cross* plan, hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (s && hipStreamIsCapturing(s, &status) == hipSuccess && status != hipStreamCaptureStatusNone)
        __atomic_store_n(&plan->captured, 1, __ATOMIC_RELAXED);
}

int create(awa_ctx* ctx, int n_seq, const int64_t* h_q_at, const int64_t* h_q_len, const int64_t* h_k_at,
           const int64_t* h_k_len, int heads, int kv_heads, int head_d, dit_cross** out) {
    if (!out || n_seq < 0 || n_seq > DIT_CROSS_SEQ_MAX || (n_seq && (!h_q_at || !h_q_len || !h_k_at || !h_k_len)) ||
        heads < 1 || heads > DIT_CROSS_HEADS_MAX || kv_heads < 1 || heads % kv_heads || head_d < 8 ||
        head_d > DIT_CROSS_HEAD_D_MAX || head_d % 8) {
        set_err(ctx, "dit_cross_create: bad argument (%d sequences, at most %d; %d heads, at most %d, a multiple of kv_heads=%d; "
                "head_d=%d, a multiple of 8 up to %d)",
                n_seq, DIT_CROSS_SEQ_MAX, heads, DIT_CROSS_HEADS_MAX, kv_heads, head_d, DIT_CROSS_HEAD_D_MAX);
        return AWA_EARG;
    }
    std::vector<int64_t> qa(h_q_at, h_q_at + n_seq), ql(h_q_len, h_q_len + n_seq);
    std::vector<int64_t> ka(h_k_at, h_k_at + n_seq), kl(h_k_len, h_k_len + n_seq);
    int64_t q_rows = 0, k_rows = 0;
    for (int i = 0; i < n_seq; i++) {
        const int64_t top = DIT_OPS_ROWS_MAX;
        if (qa[i] < 0 || ql[i] < 0 || ka[i] < 0 || kl[i] < 0 || qa[i] > top || ql[i] > top - qa[i] || ka[i] > top ||
            kl[i] > top - ka[i]) {
            set_err(ctx, "dit_cross_create: sequence %d has queries %lld + %lld and keys %lld + %lld (rows 0 .. %d)", i,
                    (long long)qa[i], (long long)ql[i], (long long)ka[i], (long long)kl[i], DIT_OPS_ROWS_MAX);
            return AWA_EARG;
        }
        if (ql[i]) q_rows = std::max(q_rows, qa[i] + ql[i]);
        if (kl[i]) k_rows = std::max(k_rows, ka[i] + kl[i]);
    }
    if (!ranges_ok(qa, ql, false) || !ranges_ok(ka, kl, true)) {
        set_err(ctx, "dit_cross_create: query rows of two sequences overlap, or key rows do and are not the same");
        return AWA_EARG;
    }
    for (dit_cross* plan : take_dropped(ctx->device)) dit_cross_destroy(plan);
    dit_cross c;
    c.device = ctx->device;
    c.heads = heads;
    c.kv_heads = kv_heads;
    c.head_d = head_d;
    c.q_rows = q_rows;
    c.k_rows = k_rows;
    std::vector<char> host;
    size_t at[2][5];
    auto add = [&](const void* from, size_t bytes) {
        const size_t to = host.size();
        host.resize(to + (bytes + 15) / 16 * 16);
        if (bytes) std::copy_n(static_cast<const char*>(from), bytes, host.data() + to);
        return to;
    };
    for (int t = 0; t < 2; t++) {
        Plan p;
        plan_queries(qa, ql, ka, kl, heads, kv_heads, head_d, t, c.qs[t], p);
        plan_keys(qa, ql, ka, kl, heads, kv_heads, head_d, t, c.ks[t], p);
        // a workgroup (of at most 256 threads; 512 for fp32 keys) per item and head group, in launches of less than 2^32 threads
        const int64_t q_blocks = (int64_t)c.qs[t].n_items * (heads / c.qs[t].pack), k_blocks = (int64_t)c.ks[t].n_items * kv_heads;
        if (q_blocks > (1 << 24) - 8 || k_blocks > (t == AWA_F32 ? 1 << 23 : 1 << 24) - 8) {  // grids are multiples of 8
            set_err(ctx, "dit_cross_create: too many blocks for one launch");
            return AWA_EARG;
        }
        const int64_t step = query_step(c.qs[t].block);
        c.qs[t].n_listed = spread(p.items, heads / c.qs[t].pack, query_cost(c.qs[t].block, t, head_d),
                                  [&](const CrossItem& it) { return ceil_div(it.kn, step); });
        c.ks[t].n_listed = spread(p.kitems, kv_heads, key_cost(t, head_d), [](const CrossKeys& it) { return (int64_t)it.count; });
        at[t][0] = add(p.items.data(), p.items.size() * sizeof(CrossItem));
        at[t][1] = add(p.joins.data(), p.joins.size() * sizeof(CrossJoin));
        at[t][2] = add(p.kitems.data(), p.kitems.size() * sizeof(CrossKeys));
        at[t][3] = add(p.kjoins.data(), p.kjoins.size() * sizeof(CrossKeyJoin));
        at[t][4] = add(p.units.data(), p.units.size() * sizeof(CrossUnit));
    }
    dit_cross* made = new dit_cross(c);
    if (!host.empty()) {
        DeviceGuard dg(ctx->device);
        hipError_t e = hipMalloc(&made->tables, host.size());
        if (e == hipSuccess) e = hipMemcpy(made->tables, host.data(), host.size(), hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            set_err(ctx, "dit_cross_create: tables of %zu bytes: %s", host.size(), hipGetErrorString(e));
            if (made->tables) (void)hipFree(made->tables);
            delete made;
            return AWA_EHIP;
        }
    }
    const char* base = static_cast<const char*>(made->tables);
    for (int t = 0; t < 2; t++) {
        made->qs[t].items = reinterpret_cast<const CrossItem*>(base + at[t][0]);
        made->qs[t].joins = reinterpret_cast<const CrossJoin*>(base + at[t][1]);
        made->ks[t].items = reinterpret_cast<const CrossKeys*>(base + at[t][2]);
        made->ks[t].joins = reinterpret_cast<const CrossKeyJoin*>(base + at[t][3]);
        made->ks[t].units = reinterpret_cast<const CrossUnit*>(base + at[t][4]);
    }
    *out = made;
    return AWA_OK;
}

// the parts of the workspace, each aligned
struct CrossWork {
    int64_t qpart, kpart, dsum, lse2, total;
};
CrossWork cross_work(const dit_cross& c, int dtype, bool grad) {
    const CrossQueries& qs = c.qs[dtype];
    const CrossKeySide& ks = c.ks[dtype];
    CrossWork w{};
    int64_t at = 0;
    auto take = [&](int64_t floats) {
        const int64_t p = at;
        at += align_up(4 * floats);
        return p;
    };
    w.qpart = take((int64_t)qs.n_parts * (c.heads / qs.pack) * cross_query_part(qs.block, c.head_d));
    if (grad) {
        w.kpart = take((int64_t)ks.n_parts * c.kv_heads * cross_key_part(CROSS_KEYS, c.head_d));
        w.dsum = take((int64_t)c.heads * c.q_rows);
        w.lse2 = take((int64_t)c.heads * c.q_rows);
    }
    w.total = at;
    return w;
}

const char* const HEADS_RULE = "%s: %s must be 16-byte aligned with strides of whole 16 bytes, rows at most %d and heads at most "
                               "2^36 elements apart (got %lld and %lld)";
// checks a tensor's address and strides, and that its elements are apart where it is written
int heads_ok(awa_ctx* ctx, const char* who, const char* name, const dit_heads* t, int dtype, int64_t rows, int heads, int d,
             bool written) {
    const int64_t unit = 16 / (int64_t)elem(dtype);
    if (!t || !t->p || !aligned(t->p, 16) || t->row < 0 || t->row > DIT_OPS_COLS_MAX || t->head < 0 || t->head > STRIDE_MAX ||
        t->row % unit || t->head % unit) {
        set_err(ctx, HEADS_RULE, who, name, DIT_OPS_COLS_MAX, t ? (long long)t->row : 0, t ? (long long)t->head : 0);
        return AWA_EARG;
    }
    if (written) {
        // rows within a head's span, or heads within a row's
        const bool inner_head = heads == 1 || t->head >= d, inner_row = rows <= 1 || t->row >= d;
        const bool rows_out = rows <= 1 || heads == 1 || t->row >= (heads - 1) * t->head + d;
        const bool heads_out = rows <= 1 || heads == 1 || t->head >= (rows - 1) * t->row + d;
        if (!inner_head || !inner_row || (!rows_out && !heads_out)) {
            set_err(ctx, "%s: rows or heads of %s coincide (strides %lld and %lld)", who, name, (long long)t->row, (long long)t->head);
            return AWA_EARG;
        }
    }
    return AWA_OK;
}
Extent extent(const dit_heads* t, int dtype, int64_t rows, int heads, int d) {
    return {t->p, rows > 0 ? (size_t)((rows - 1) * t->row + (heads - 1) * t->head + d) * elem(dtype) : 0};
}
// Tensors side by side in the same rows (queries, keys and values of one projection), or with heads outermost in the same heads,
// are apart although their extents are not.
bool heads_collide(const dit_heads* a, int64_t a_rows, int a_heads, const dit_heads* b, int64_t b_rows, int b_heads, int dtype, int d) {
    if (!touches(extent(a, dtype, a_rows, a_heads, d), extent(b, dtype, b_rows, b_heads, d))) return false;
    const int64_t size = (int64_t)elem(dtype);
    const intptr_t pa = reinterpret_cast<intptr_t>(a->p), pb = reinterpret_cast<intptr_t>(b->p);
    // na and nb pieces of wa and wb elements, sa and sb apart (one piece: any)
    auto beside = [&](int64_t na, int64_t sa, int64_t wa, int64_t nb, int64_t sb, int64_t wb) {
        const int64_t step = (na > 1 ? sa : sb) * size;
        if ((na > 1 && nb > 1 && sa != sb) || wa * size > step || wb * size > step) return false;
        const int64_t off = (int64_t)((pb - pa) % step + step) % step;
        return off >= wa * size && off + wb * size <= step;
    };
    return !beside(a_rows, a->row, (a_heads - 1) * a->head + d, b_rows, b->row, (b_heads - 1) * b->head + d) &&
           !beside(a_heads, a->head, (a_rows - 1) * a->row + d, b_heads, b->head, (b_rows - 1) * b->row + d);
}

void place(const dit_heads* t, int dtype, const char*& p, int64_t& row, int64_t& head) {
    p = static_cast<const char*>(t->p);
    row = t->row * (int64_t)elem(dtype);
    head = t->head * (int64_t)elem(dtype);
}
void place(const dit_heads* t, int dtype, char*& p, int64_t& row, int64_t& head) {
    p = static_cast<char*>(t->p);
    row = t->row * (int64_t)elem(dtype);
    head = t->head * (int64_t)elem(dtype);
}

// takes DIT_CROSS_WHOLE off a dtype that may have it
bool take_whole(int& dtype) {
    const bool whole = dtype == (AWA_F32 | DIT_CROSS_WHOLE) || dtype == (AWA_BF16 | DIT_CROSS_WHOLE);
    if (whole) dtype &= ~DIT_CROSS_WHOLE;
    return whole;
}

int cross_args_ok(awa_ctx* ctx, const char* who, const dit_cross* plan, int dtype, float scale, bool with_lse, int64_t ld_lse) {
    if (!plan || !dtype_ok(dtype) || !(scale >= 1e-30f && scale <= 1e30f)) {
        set_err(ctx, "%s: bad argument (plan, dtype=%d, scale=%g: 1e-30 .. 1e30)", who, dtype, (double)scale);
        return AWA_EARG;
    }
    if (plan->device != ctx->device) {
        set_err(ctx, "%s: the plan is of device %d, the context of %d", who, plan->device, ctx->device);
        return AWA_EARG;
    }
    if (with_lse && (ld_lse < plan->q_rows || ld_lse > STRIDE_MAX)) {
        set_err(ctx, "%s: ld_lse=%lld (at least %lld, at most 2^36)", who, (long long)ld_lse, (long long)plan->q_rows);
        return AWA_EARG;
    }
    return AWA_OK;
}

}  // namespace

extern "C" {

int dit_layer_norm(awa_ctx* ctx, int dtype_x, const void* d_x, int64_t ldx, const float* d_w, const float* d_b, float eps,
                   int dtype_y, void* d_y, int64_t ldy, float* d_stats, int M, int K, awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    if (!dtype_ok(dtype_x) || !dtype_ok(dtype_y) || !norm_sizes_ok(M, K) || !(eps >= 0.f) || !std::isfinite(eps)) {
        set_err(ctx, "dit_layer_norm: bad argument dtypes=%d, %d M=%d K=%d eps=%g (M <= %d, 1 <= K <= %d, eps >= 0)", dtype_x,
                dtype_y, M, K, (double)eps, DIT_OPS_ROWS_MAX, DIT_NORM_COLS_MAX);
        return AWA_EARG;
    }
    if (M == 0) return AWA_OK;
    if (!d_x || !d_y || !aligned(d_x, elem(dtype_x)) || !aligned(d_y, elem(dtype_y)) || !aligned(d_w, 4) || !aligned(d_b, 4) ||
        !aligned(d_stats, 8)) {
        set_err(ctx, "dit_layer_norm: null or misaligned pointer (elements; stats 8 bytes)");
        return AWA_EARG;
    }
    if (!stride_ok(M, ldx, K) || !stride_ok(M, ldy, K)) {
        set_err(ctx, "dit_layer_norm: ldx=%lld, ldy=%lld (at least K=%d, at most 2^36)", (long long)ldx, (long long)ldy, K);
        return AWA_EARG;
    }
    NormFwd a{};
    a.x = d_x; a.ldx = M > 1 ? ldx : K;
    a.w = d_w; a.b = d_b; a.eps = eps;
    a.y = d_y; a.ldy = M > 1 ? ldy : K;
    a.stats = reinterpret_cast<float2*>(d_stats);
    a.M = M; a.K = K;
    const bool same = d_x == d_y && dtype_x == dtype_y && a.ldx == a.ldy;
    const Extent x{same ? nullptr : d_x, span(M, a.ldx, K, elem(dtype_x))}, y{d_y, span(M, a.ldy, K, elem(dtype_y))};
    const Extent w{d_w, (size_t)K * 4}, b{d_b, (size_t)K * 4}, st{d_stats, (size_t)M * 8};
    if (collide({y, st}, {x, w, b}) || touches(st, {d_x, span(M, a.ldx, K, elem(dtype_x))})) {
        set_err(ctx, "dit_layer_norm: outputs lie over an input (other than y = x) or each other");
        return AWA_EARG;
    }
    DeviceGuard dg(ctx->device);
    HIPCK(ctx, launch_layer_norm(dtype_x, dtype_y, a, reinterpret_cast<hipStream_t>(stream)));
    return AWA_OK;
}

int64_t dit_layer_norm_grad_work(int M, int K) {
    if (!norm_sizes_ok(M, K)) return AWA_EARG;
    return align_up((int64_t)norm_grad_groups(M, K) * 2 * K * 4);
}

int dit_layer_norm_grad(awa_ctx* ctx, int dtype_dy, const void* d_dy, int64_t lddy, int dtype_x, const void* d_x, int64_t ldx,
                        const uint32_t* d_xs, int64_t ld_xs, const float* d_stats, const float* d_w, int dtype_dx, void* d_dx,
                        int64_t lddx, float* d_dw, float* d_db, void* d_work, int64_t work_bytes, int M, int K,
                        awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    const bool saved = dtype_x == DIT_FP8;
    if (!dtype_ok(dtype_dy) || !(dtype_ok(dtype_x) || saved) || (d_dx && !dtype_ok(dtype_dx)) || !norm_sizes_ok(M, K) ||
        saved != (d_xs != nullptr) || (!d_dx && !d_dw && !d_db)) {
        set_err(ctx, "dit_layer_norm_grad: bad argument dtypes=%d, %d, %d M=%d K=%d (M <= %d, 1 <= K <= %d; scale words with 8-bit "
                "x, and only with it; at least one output)",
                dtype_dy, dtype_x, dtype_dx, M, K, DIT_OPS_ROWS_MAX, DIT_NORM_COLS_MAX);
        return AWA_EARG;
    }
    const size_t xsize = saved ? 1 : elem(dtype_x);
    if ((M && (!d_dy || !d_x || !d_stats)) || !aligned(d_dy, elem(dtype_dy)) || !aligned(d_x, saved ? 16 : xsize) ||
        !aligned(d_xs, 4) || !aligned(d_stats, 8) || !aligned(d_w, 4) || (d_dx && !aligned(d_dx, elem(dtype_dx))) ||
        !aligned(d_dw, 4) || !aligned(d_db, 4)) {
        set_err(ctx, "dit_layer_norm_grad: null or misaligned pointer (elements; 8-bit x 16 bytes, stats 8)");
        return AWA_EARG;
    }
    if (!stride_ok(M, lddy, K) || (!saved && !stride_ok(M, ldx, K)) || (d_dx && !stride_ok(M, lddx, K)) ||
        (saved && (ld_xs < M || ld_xs > STRIDE_MAX))) {
        set_err(ctx, "dit_layer_norm_grad: lddy=%lld, ldx=%lld, lddx=%lld (at least K=%d), ld_xs=%lld (at least M=%d; all at most 2^36)",
                (long long)lddy, (long long)ldx, (long long)lddx, K, (long long)ld_xs, M);
        return AWA_EARG;
    }
    const bool params = d_dw || d_db;
    const int64_t need = params && M ? dit_layer_norm_grad_work(M, K) : 0;
    if (int rc = work_ok(ctx, "dit_layer_norm_grad", d_work, work_bytes, need)) return rc;
    if (M == 0 && !params) return AWA_OK;
    NormGrad a{};
    a.dy = d_dy; a.lddy = M > 1 ? lddy : K;
    a.x = d_x; a.ldx = saved ? padded(K) : M > 1 ? ldx : K;
    a.xs = d_xs; a.ld_xs = ld_xs;
    a.stats = reinterpret_cast<const float2*>(d_stats);
    a.w = d_w;
    a.dx = d_dx; a.lddx = M > 1 ? lddx : K; a.dx_f32 = dtype_dx == AWA_F32;
    a.dw = d_dw; a.db = d_db;
    a.part = params && M ? static_cast<float*>(d_work) : nullptr;
    a.groups = M ? norm_grad_groups(M, K) : 0;
    a.M = M; a.K = K;
    const Extent dy{d_dy, span(M, a.lddy, K, elem(dtype_dy))}, x{d_x, span(M, a.ldx, saved ? a.ldx : K, xsize)};
    const Extent xs{d_xs, saved ? span(groups_of(K), ld_xs, M, 4) : 0}, st{d_stats, (size_t)M * 8}, w{d_w, (size_t)K * 4};
    const Extent dx{d_dx, d_dx ? span(M, a.lddx, K, elem(dtype_dx)) : 0};
    const Extent dw{d_dw, (size_t)K * 4}, db{d_db, (size_t)K * 4}, wk{d_work, (size_t)need};
    const bool over_dy = d_dx == d_dy && dtype_dx == dtype_dy && a.lddx == a.lddy;
    const bool over_x = d_dx == d_x && dtype_dx == dtype_x && a.lddx == a.ldx;
    if (collide({dw, db, wk}, {dy, x, xs, st, w, dx}) || collide({dx}, {xs, st, w}) || (!over_dy && touches(dx, dy)) ||
        (!over_x && touches(dx, x))) {
        set_err(ctx, "dit_layer_norm_grad: outputs or d_work lie over an input (other than dx = dy or x) or each other");
        return AWA_EARG;
    }
    DeviceGuard dg(ctx->device);
    HIPCK(ctx, launch_layer_norm_grad(dtype_dy, dtype_x, a, reinterpret_cast<hipStream_t>(stream)));
    return AWA_OK;
}

int64_t dit_grad_weight_work(int dtype_dy, int dtype_w, int M, int N, int K) {
    if (!dtype_ok(dtype_dy) || !dtype_ok(dtype_w) || !weight_sizes_ok(M, N, K)) return AWA_EARG;
    return weight_work(dtype_dy, M, N, K);
}

int dit_grad_weight_fp8(awa_ctx* ctx, int dtype_dy, const void* d_dy, int64_t lddy, const uint8_t* d_q, const uint32_t* d_s,
                        int64_t ld_s, int dtype_w, void* d_dw, int64_t ldw, float* d_db, int add, void* d_work,
                        int64_t work_bytes, int M, int N, int K, awa_stream_t stream) {
    if (!ctx) return AWA_EARG;
    if (!dtype_ok(dtype_dy) || !dtype_ok(dtype_w) || !weight_sizes_ok(M, N, K) || !d_dw || (add && dtype_w != AWA_F32)) {
        set_err(ctx, "dit_grad_weight_fp8: bad argument dtypes=%d, %d M=%d N=%d K=%d add=%d (M <= %d, 1 <= N, K <= %d; add with fp32 dW)",
                dtype_dy, dtype_w, M, N, K, add, DIT_OPS_ROWS_MAX, DIT_OPS_COLS_MAX);
        return AWA_EARG;
    }
    if ((M && (!d_dy || !d_q || !d_s)) || !aligned(d_dy, elem(dtype_dy)) || !aligned(d_q, 16) || !aligned(d_s, 4) ||
        !aligned(d_dw, elem(dtype_w)) || !aligned(d_db, 4)) {
        set_err(ctx, "dit_grad_weight_fp8: null or misaligned pointer (d_q 16 bytes, words and db 4, others their elements)");
        return AWA_EARG;
    }
    if (!stride_ok(M, lddy, N) || (M > 1 && lddy > DIT_OPS_COLS_MAX) || !stride_ok(N, ldw, K) || ld_s < M || ld_s > STRIDE_MAX) {
        set_err(ctx, "dit_grad_weight_fp8: lddy=%lld (%d .. %d), ldw=%lld (at least %d), ld_s=%lld (at least %d; both at most 2^36)",
                (long long)lddy, N, DIT_OPS_COLS_MAX, (long long)ldw, K, (long long)ld_s, M);
        return AWA_EARG;
    }
    const int64_t need = weight_work(dtype_dy, M, N, K);
    if (int rc = work_ok(ctx, "dit_grad_weight_fp8", d_work, work_bytes, need)) return rc;
    GradWeight a{};
    a.dy = d_dy; a.lddy = M > 1 ? lddy : N;
    a.q = d_q; a.s = d_s; a.ld_s = ld_s;
    a.dw = d_dw; a.ldw = N > 1 ? ldw : K;
    a.db = d_db;
    a.add = add != 0; a.w_f32 = dtype_w == AWA_F32;
    a.part = static_cast<float*>(d_work);
    a.M = M; a.N = N; a.K = K; a.kp = padded(K);
    const Extent dy{d_dy, span(M, a.lddy, N, elem(dtype_dy))}, q{d_q, (size_t)M * a.kp}, s{d_s, span(groups_of(K), ld_s, M, 4)};
    const Extent dw{d_dw, span(N, a.ldw, K, elem(dtype_w))}, db{d_db, (size_t)N * 4}, wk{d_work, (size_t)need};
    if (collide({dw, db, wk}, {dy, q, s})) {
        set_err(ctx, "dit_grad_weight_fp8: outputs or d_work lie over an input or each other");
        return AWA_EARG;
    }
    DeviceGuard dg(ctx->device);
    HIPCK(ctx, launch_grad_weight(dtype_dy, a, reinterpret_cast<hipStream_t>(stream)));
    return AWA_OK;
}

int dit_cross_create(awa_ctx* ctx, int n_seq, const int64_t* h_q_at, const int64_t* h_q_len, const int64_t* h_k_at,
                     const int64_t* h_k_len, int heads, int kv_heads, int head_d, dit_cross** out) {
    if (!ctx) return AWA_EARG;
    if (out) *out = nullptr;
    try {
        return create(ctx, n_seq, h_q_at, h_q_len, h_k_at, h_k_len, heads, kv_heads, head_d, out);
    } catch (const std::exception& e) {  // memory: no exception leaves a C entry
        try {
            set_err(ctx, "dit_cross_create: %s", e.what());
        } catch (...) {
        }
        return AWA_EHIP;
    }
}

void dit_cross_destroy(dit_cross* plan) {
    if (!plan) return;
    if (plan->tables) {
        DeviceGuard dg(plan->device);
        (void)hipFree(plan->tables);
    }
    delete plan;
}

void dit_cross_drop(dit_cross* plan) {
    if (!plan || __atomic_load_n(&plan->captured, __ATOMIC_RELAXED)) return;
    try {
        std::lock_guard<std::mutex> hold(dropped().lock);
        dropped().plans.push_back(plan);
    } catch (const std::exception&) {  // memory: kept
    }
}

int64_t dit_cross_work(const dit_cross* plan, int dtype, int grad) {
    take_whole(dtype);
    if (!plan || !dtype_ok(dtype)) return AWA_EARG;
    return cross_work(*plan, dtype, grad != 0).total;
}

int dit_cross_forward(awa_ctx* ctx, const dit_cross* plan, int dtype, const dit_heads* q, const dit_heads* k,
                      const dit_heads* v, const uint8_t* d_mask, float scale, const dit_heads* out, float* d_lse, int64_t ld_lse,
                      void* d_work, int64_t work_bytes, awa_stream_t stream) {
    const char* who = "dit_cross_forward";
    if (!ctx) return AWA_EARG;
    const bool whole = take_whole(dtype);
    if (int rc = cross_args_ok(ctx, who, plan, dtype, scale, d_lse != nullptr, ld_lse)) return rc;
    if (plan->q_rows == 0) return AWA_OK;
    const int64_t qr = plan->q_rows, kr = plan->k_rows;
    const int h = plan->heads, hk = plan->kv_heads, d = plan->head_d;
    if (int rc = heads_ok(ctx, who, "q", q, dtype, qr, h, d, false)) return rc;
    if (int rc = heads_ok(ctx, who, "out", out, dtype, qr, h, d, true)) return rc;
    const dit_heads none{out->p, 0, 0};  // without keys k and v are not read
    if (kr == 0) k = v = &none;
    if (int rc = heads_ok(ctx, who, "k", k, dtype, kr, hk, d, false)) return rc;
    if (int rc = heads_ok(ctx, who, "v", v, dtype, kr, hk, d, false)) return rc;
    if (!aligned(d_lse, 4)) {
        set_err(ctx, "%s: d_lse must be 4-byte aligned", who);
        return AWA_EARG;
    }
    const CrossWork w = cross_work(*plan, dtype, false);
    if (int rc = work_ok(ctx, who, d_work, work_bytes, w.total)) return rc;
    const Extent lse{d_lse, d_lse ? span(h, ld_lse, qr, 4) : 0}, wk{d_work, (size_t)w.total}, mask{d_mask, (size_t)kr};
    const Extent eo = extent(out, dtype, qr, h, d), eq = extent(q, dtype, qr, h, d), ek = extent(k, dtype, kr, hk, d),
                 ev = extent(v, dtype, kr, hk, d);
    if (collide({lse, wk}, {eo, eq, ek, ev, mask}) || touches(eo, mask) || heads_collide(out, qr, h, q, qr, h, dtype, d) ||
        heads_collide(out, qr, h, k, kr, hk, dtype, d) || heads_collide(out, qr, h, v, kr, hk, dtype, d)) {
        set_err(ctx, "%s: outputs or d_work lie over an input or each other", who);
        return AWA_EARG;
    }
    CrossArgs a{};
    place(q, dtype, a.q, a.q_row, a.q_head);
    place(k, dtype, a.k, a.k_row, a.k_head);
    place(v, dtype, a.v, a.v_row, a.v_head);
    place(out, dtype, a.o, a.o_row, a.o_head);
    a.mask = d_mask;
    a.scale = scale;
    a.c = (float)((double)scale * 1.4426950408889634);
    a.lse = d_lse;
    a.ld_lse = ld_lse;
    a.heads = h; a.kv_heads = hk; a.head_d = d;
    a.whole = whole;
    a.qs = plan->qs[dtype]; a.ks = plan->ks[dtype];
    a.qpart = reinterpret_cast<float*>(static_cast<char*>(d_work) + w.qpart);
    DeviceGuard dg(ctx->device);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    note_capture(plan, s);
    HIPCK(ctx, launch_cross_forward(dtype, a, s));
    return AWA_OK;
}

int dit_cross_grad(awa_ctx* ctx, const dit_cross* plan, int dtype, const dit_heads* dout, const dit_heads* q,
                   const dit_heads* k, const dit_heads* v, const dit_heads* out, const float* d_lse, int64_t ld_lse,
                   const uint8_t* d_mask, float scale, const dit_heads* dq, const dit_heads* dk, const dit_heads* dv,
                   void* d_work, int64_t work_bytes, awa_stream_t stream) {
    const char* who = "dit_cross_grad";
    if (!ctx) return AWA_EARG;
    const bool whole = take_whole(dtype);
    if (int rc = cross_args_ok(ctx, who, plan, dtype, scale, true, ld_lse)) return rc;
    const int64_t qr = plan->q_rows, kr = plan->k_rows;
    const int h = plan->heads, hk = plan->kv_heads, d = plan->head_d;
    if (qr == 0 && kr == 0) return AWA_OK;
    // tensors of a side without rows are neither read nor written
    const dit_heads* const any = qr ? q : dk;
    const dit_heads none{any ? any->p : nullptr, 0, 0};
    if (qr == 0) dout = q = out = dq = &none;
    if (kr == 0) k = v = dk = dv = &none;
    const struct { const char* name; const dit_heads* t; int64_t rows; int heads; bool written; } all[] = {
        {"dout", dout, qr, h, false}, {"q", q, qr, h, false},   {"k", k, kr, hk, false},  {"v", v, kr, hk, false},
        {"out", out, qr, h, false},   {"dq", dq, qr, h, true}, {"dk", dk, kr, hk, true}, {"dv", dv, kr, hk, true}};
    for (const auto& t : all)
        if (int rc = heads_ok(ctx, who, t.name, t.t, dtype, t.rows, t.heads, d, t.written && t.rows > 0)) return rc;
    if ((qr && !d_lse) || !aligned(d_lse, 4)) {
        set_err(ctx, "%s: d_lse must not be NULL, and 4-byte aligned", who);
        return AWA_EARG;
    }
    const CrossWork w = cross_work(*plan, dtype, true);
    if (int rc = work_ok(ctx, who, d_work, work_bytes, w.total)) return rc;
    const Extent lse{d_lse, qr ? span(h, ld_lse, qr, 4) : 0}, wk{d_work, (size_t)w.total}, mask{d_mask, (size_t)kr};
    bool bad = touches(wk, lse) || touches(wk, mask);
    for (const auto& o : all) {
        const Extent e = extent(o.t, dtype, o.rows, o.heads, d);
        bad = bad || touches(wk, e);
        if (!o.written || !o.rows) continue;
        bad = bad || touches(e, lse) || touches(e, mask);
        for (const auto& t : all)
            if (&t != &o && t.rows) bad = bad || heads_collide(o.t, o.rows, o.heads, t.t, t.rows, t.heads, dtype, d);
    }
    if (bad) {
        set_err(ctx, "%s: outputs or d_work lie over an input or each other", who);
        return AWA_EARG;
    }
    CrossArgs a{};
    place(dout, dtype, a.dout, a.dout_row, a.dout_head);
    place(q, dtype, a.q, a.q_row, a.q_head);
    place(k, dtype, a.k, a.k_row, a.k_head);
    place(v, dtype, a.v, a.v_row, a.v_head);
    place(out, dtype, a.out, a.out_row, a.out_head);
    place(dq, dtype, a.dq, a.dq_row, a.dq_head);
    place(dk, dtype, a.dk, a.dk_row, a.dk_head);
    place(dv, dtype, a.dv, a.dv_row, a.dv_head);
    a.mask = d_mask;
    a.scale = scale;
    a.c = (float)((double)scale * 1.4426950408889634);
    a.lse = const_cast<float*>(d_lse);
    a.ld_lse = ld_lse;
    a.heads = h; a.kv_heads = hk; a.head_d = d;
    a.whole = whole;
    a.qs = plan->qs[dtype]; a.ks = plan->ks[dtype];
    char* base = static_cast<char*>(d_work);
    a.qpart = reinterpret_cast<float*>(base + w.qpart);
    a.kpart = reinterpret_cast<float*>(base + w.kpart);
    a.dsum = reinterpret_cast<float*>(base + w.dsum);
    a.lse2 = reinterpret_cast<float*>(base + w.lse2);
    a.ld_dsum = qr;
    DeviceGuard dg(ctx->device);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    note_capture(plan, s);
    HIPCK(ctx, launch_cross_grad_queries(dtype, a, s));
    HIPCK(ctx, launch_cross_grad_keys(dtype, a, s));
    return AWA_OK;
}

}  // extern "C"
