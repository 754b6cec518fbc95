// Native host path of the operators on token sequences: checks, views, allocation and autograd nodes.
//
// Tensors are Julia-shaped, (D, heads, N, B) or (D, heads, T).  Any strides are taken as they are when the features are
// contiguous and the others are multiples of 16 bytes (slices of a packed projection, a transposed batch); anything else is
// copied into column-major order first.
#include "host_common.h"

#include "../../include/circatt_b200_tokens.h"

using namespace circatt;

namespace {

int dtype_code(const Tensor& t) {
    const auto d = t.scalar_type();
    if (d == at::kFloat) return CA_F32;
    if (d == at::kBFloat16) return CA_BF16;
    if (d == at::kHalf) return CA_F16;
    raise(PyExc_TypeError, std::string("only Float32, BFloat16 and Float16 are supported, got ") + c10::toString(d));
}

std::string shape_text(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

[[noreturn]] void mismatch(const std::string& what) { raise(PyExc_AssertionError, what); }

void require_like(const Tensor& t, const Tensor& q, const char* name) {
    require_cuda(t);
    if (t.device() != q.device()) raise(PyExc_RuntimeError, std::string(name) + " is on " + t.device().str() + ", not on " + q.device().str());
    if (t.scalar_type() != q.scalar_type())
        raise(PyExc_TypeError, std::string(name) + " is " + c10::toString(t.scalar_type()) + ", not " + c10::toString(q.scalar_type()));
}

void require_ints(const Tensor& t, const Tensor& q, at::ScalarType want, const char* name) {
    require_cuda(t);
    if (t.device() != q.device()) raise(PyExc_RuntimeError, std::string(name) + " is on " + t.device().str() + ", not on " + q.device().str());
    if (t.scalar_type() != want) raise(PyExc_TypeError, std::string(name) + " must be " + c10::toString(want) + ", got " + c10::toString(t.scalar_type()));
}

bool as_it_is(const Tensor& t) {
    const int64_t piece = 16 / t.element_size();
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
    if (t.stride(0) != 1 && t.size(0) != 1) return false;
    for (int64_t i = 1; i < t.dim(); ++i)
        if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % piece)) return false;
    return true;
}
Tensor ready(const Tensor& t) { return as_it_is(t) ? t : colmajor(t); }

// Strides of a (D, heads, tokens[, batch]) tensor; those of extents below 2 are never used and set to a legal value.
ca_seq_view view(const Tensor& t) {
    auto st = [&](int64_t i) { return i < t.dim() && t.size(i) > 1 ? t.stride(i) : 16 / (int64_t)t.element_size(); };
    return ca_seq_view{t.data_ptr(), st(1), st(2), st(3)};
}
ca_page_view page_view(const Tensor& t) {
    auto st = [&](int64_t i) { return t.size(i) > 1 ? t.stride(i) : 16 / (int64_t)t.element_size(); };
    return ca_page_view{t.data_ptr(), st(1), st(2), st(3)};
}

int32_t int_of(int64_t n, const char* name) {
    if (n < INT32_MIN || n > INT32_MAX) raise(PyExc_OverflowError, std::string(name) + " = " + std::to_string(n) + " does not fit into 32 bits");
    return (int32_t)n;
}

// ---------------------------------------------------------------- rotary positions
struct Rotation {
    Tensor positions, turns;
    std::vector<int64_t> sections;
    bool interleaved;
};

// Checks the positions (axes, N[, B]) and turns against x (D, heads, N[, B]).
ca_rotary_desc rotary_desc(const Tensor& x, const Rotation& r, bool inverse) {
    ca_rotary_desc d{};
    d.dtype = dtype_code(x);
    require_ints(r.positions, x, at::kInt, "positions");
    require_ints(r.turns, x, at::kLong, "turns");
    if (r.turns.dim() != 1 || !r.turns.is_contiguous()) mismatch("turns must be a vector, one entry for each pair of features");
    const Tensor& p = r.positions;
    const int64_t B = x.dim() == 4 ? x.size(3) : 1;
    if ((p.dim() != 2 && p.dim() != 3) || p.size(1) != x.size(2) || (p.dim() == 3 && p.size(2) != B && p.size(2) != 1))
        mismatch("positions of size " + shape_text(p) + " do not fit " + shape_text(x) + ": (axes, N) or (axes, N, B) expected");
    if ((int64_t)r.sections.size() != p.size(0)) mismatch("positions of " + std::to_string(p.size(0)) + " axes, but " + std::to_string(r.sections.size()) + " sections");
    if (p.size(0) > CA_MAX_AXES) mismatch("at most " + std::to_string(CA_MAX_AXES) + " axes are supported");
    d.dim = int_of(x.size(0), "D");
    d.pairs = int_of(r.turns.size(0), "pairs");
    d.interleaved = r.interleaved;
    d.inverse = inverse;
    d.axes = (int32_t)p.size(0);
    for (int i = 0; i < d.axes; ++i) d.sections[i] = int_of(r.sections[i], "section");
    d.tokens = int_of(x.size(2), "N");
    d.batch = int_of(B, "B");
    d.positions = static_cast<const int32_t*>(p.data_ptr());
    d.axis_stride = p.stride(0);
    d.token_stride = p.stride(1);
    d.batch_stride = p.dim() == 3 && p.size(2) > 1 ? p.stride(2) : 0;
    d.turns = r.turns.data_ptr<int64_t>();
    return d;
}

void check_tokens(const Tensor& x, const char* name, bool packed_only = false) {
    require_cuda(x);
    if (packed_only ? x.dim() != 3 : (x.dim() != 3 && x.dim() != 4))
        mismatch(std::string(name) + " of size " + shape_text(x) + (packed_only ? ": (D, heads, T) expected" : ": (D, heads, N, B) or (D, heads, T) expected"));
}

std::tuple<Tensor, Tensor> rotate(const Tensor& x1_, const Tensor& x2_, const Rotation& r, bool inverse) {
    const Tensor x1 = ready(x1_), x2 = x2_.defined() ? ready(x2_) : Tensor();
    Call call(x1, "circatt.rotary");
    const ca_rotary_desc d = rotary_desc(x1, r, inverse);
    Tensor y1 = empty_cm(x1.sizes(), x1, x1.scalar_type()), y2;
    const ca_seq_view vx1 = view(x1), vy1 = view(y1);
    ca_seq_view vx2{}, vy2{};
    if (x2.defined()) {
        y2 = empty_cm(x2.sizes(), x2, x2.scalar_type());
        vx2 = view(x2);
        vy2 = view(y2);
    }
    check(ca_rotary(&d, &vx1, &vy1, int_of(x1.size(1), "heads"), x2.defined() ? &vx2 : nullptr, x2.defined() ? &vy2 : nullptr,
                    x2.defined() ? int_of(x2.size(1), "heads") : 0, call.stream));
    return {y1, y2};
}

// The gradient of a rotation is the rotation back.
struct RotaryFn : public Function<RotaryFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x1, const std::optional<Tensor>& x2, const Tensor& positions,
                                 const Tensor& turns, std::vector<int64_t> sections, bool interleaved) {
        const Rotation r{positions, turns, sections, interleaved};
        auto [y1, y2] = rotate(x1, x2 ? *x2 : Tensor(), r, false);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, turns});
        ctx->saved_data["sections"] = sections;
        ctx->saved_data["interleaved"] = interleaved;
        return x2 ? variable_list{y1, y2} : variable_list{y1};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Rotation r{s[0], s[1], ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool()};
        Tensor d1, d2;
        const bool two = g.size() > 1 && g[1].defined();
        if (g[0].defined()) std::tie(d1, d2) = rotate(g[0], two ? g[1] : Tensor(), r, true);
        else if (two) d2 = std::get<0>(rotate(g[1], Tensor(), r, true));
        return {d1, d2, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, std::optional<Tensor>> rotary(const Tensor& x1, const std::optional<Tensor>& x2, const Tensor& positions, const Tensor& turns,
                                                 std::vector<int64_t> sections, bool interleaved) {
    check_tokens(x1, "x");
    if (x2) {
        check_tokens(*x2, "the second tensor");
        require_like(*x2, x1, "the second tensor");
        if (x2->dim() != x1.dim() || x2->size(0) != x1.size(0) || x2->size(2) != x1.size(2) || (x1.dim() == 4 && x2->size(3) != x1.size(3)))
            mismatch("tensors of sizes " + shape_text(x1) + " and " + shape_text(*x2) + " differ in more than their heads");
    }
    if (!tracked({&x1}) && !(x2 && tracked({&*x2}))) {
        auto [y1, y2] = rotate(x1, x2 ? *x2 : Tensor(), Rotation{positions, turns, sections, interleaved}, false);
        return {y1, x2 ? std::optional<Tensor>(y2) : std::nullopt};
    }
    variable_list o = RotaryFn::apply(x1, x2, positions, turns, sections, interleaved);
    return {o[0], x2 ? std::optional<Tensor>(o[1]) : std::nullopt};
}

// ---------------------------------------------------------------- paged cache
// The cache is written in place or read by address: a copy would lose the writes, so its strides have to fit.
void check_cache(const Tensor& pool, const Tensor& q, const Tensor& other, const char* name) {
    require_like(pool, q, name);
    if (pool.dim() != 4 || pool.size(0) != q.size(0)) mismatch(std::string(name) + " of size " + shape_text(pool) + ": (D, page, heads, pages) expected, with the D of " + shape_text(q));
    if (pool.sizes() != other.sizes()) mismatch("k_pages and v_pages differ in size: " + shape_text(pool) + " and " + shape_text(other));
    if (!as_it_is(pool)) mismatch(std::string(name) + ": features must be contiguous, and the address and other strides multiples of 16 bytes");
}

ca_pages pages_of(const Tensor& q, const Tensor& pool, const Tensor& table, const Tensor& starts, const Tensor& lengths) {
    require_ints(table, q, at::kInt, "table");
    require_ints(starts, q, at::kInt, "starts");
    require_ints(lengths, q, at::kInt, "lengths");
    if (lengths.dim() != 1 || starts.dim() != 1 || starts.size(0) != lengths.size(0) + 1 || table.dim() != 2 || table.size(1) != lengths.size(0))
        mismatch("table of size " + shape_text(table) + ", starts of size " + shape_text(starts) + ", lengths of size " + shape_text(lengths) +
                 ": (width, S), (S + 1) and (S) expected");
    if (!lengths.is_contiguous() || !starts.is_contiguous() || !is_colmajor(table)) mismatch("table, starts and lengths must be dense (table column-major)");
    ca_pages p{};
    p.table = table.data_ptr<int32_t>();
    p.starts = starts.data_ptr<int32_t>();
    p.lengths = lengths.data_ptr<int32_t>();
    p.width = int_of(table.size(0), "width");
    p.page = int_of(pool.size(1), "page");
    p.pages = int_of(pool.size(3), "pages");
    p.sequences = int_of(lengths.size(0), "S");
    return p;
}

Tensor rotary_append(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                     const Tensor& starts, const Tensor& lengths, const Tensor& positions, const Tensor& turns,
                     std::vector<int64_t> sections, bool interleaved) {
    check_tokens(q_, "q", true);
    check_tokens(k_, "k", true);
    check_tokens(v_, "v", true);
    require_like(k_, q_, "k");
    require_like(v_, q_, "v");
    if (k_.sizes() != v_.sizes() || k_.size(0) != q_.size(0) || k_.size(2) != q_.size(2))
        mismatch("q, k, v of sizes " + shape_text(q_) + ", " + shape_text(k_) + ", " + shape_text(v_) + " do not belong together");
    check_cache(k_pages, q_, v_pages, "k_pages");
    check_cache(v_pages, q_, k_pages, "v_pages");
    if (k_pages.size(2) != k_.size(1)) mismatch("a cache of " + std::to_string(k_pages.size(2)) + " heads, but k has " + std::to_string(k_.size(1)));
    const Tensor q = ready(q_.detach()), k = ready(k_.detach()), v = ready(v_.detach());
    Call call(q, "circatt.append");
    const ca_rotary_desc d = rotary_desc(q, Rotation{positions, turns, sections, interleaved}, false);
    const ca_pages p = pages_of(q, k_pages, table, starts, lengths);
    Tensor out = empty_cm(q.sizes(), q, q.scalar_type());
    const ca_seq_view vq = view(q), vo = view(out), vk = view(k), vv = view(v);
    const ca_page_view kp = page_view(k_pages), vp = page_view(v_pages);
    check(ca_rotary_append(&d, &vq, &vo, int_of(q.size(1), "heads"), &vk, &vv, int_of(k.size(1), "heads"), &kp, &vp, &p, call.stream));
    return out;
}

// ---------------------------------------------------------------- other scores and masks
struct Form {
    double cap;                         // 0: none
    Tensor slopes, spans, prefix;       // undefined: none
    ca_seq_form view() const {
        return ca_seq_form{(float)cap, fptr(slopes), static_cast<const int32_t*>(ptr(spans)), static_cast<const int32_t*>(ptr(prefix))};
    }
};

// Checks them against q, whose heads and tokens they belong to.
Form form_of(const Tensor& q, std::optional<double> cap, const std::optional<Tensor>& slopes, const std::optional<Tensor>& spans,
             const std::optional<Tensor>& prefix) {
    Form f;
    if (cap && !(*cap > 0.0)) mismatch("cap (" + std::to_string(*cap) + ") must be positive: None leaves the scores as they are");
    f.cap = cap ? *cap : 0.0;
    if (cap && (float)f.cap == 0.f) mismatch("cap is too small for 32 bits");
    if (slopes) {
        require_ints(*slopes, q, at::kFloat, "slopes");
        if (slopes->dim() != 1 || slopes->size(0) != q.size(1) || !slopes->is_contiguous())
            mismatch("slopes of size " + shape_text(*slopes) + ": one for each of the " + std::to_string(q.size(1)) + " query heads expected");
        if (tracked({&*slopes})) raise(PyExc_NotImplementedError, "slopes have no gradient: detach them");
        f.slopes = *slopes;
    }
    if (spans) {
        require_ints(*spans, q, at::kInt, "spans");
        if (spans->dim() != 3 || spans->size(0) != 4 || spans->size(1) != q.size(2) || spans->size(2) != q.size(3) || !is_colmajor(*spans))
            mismatch("spans of size " + shape_text(*spans) + ": those of token_spans for " + std::to_string(q.size(2)) + " tokens and a batch of " + std::to_string(q.size(3)) + " expected");
        f.spans = *spans;
    }
    if (prefix) {
        require_ints(*prefix, q, at::kInt, "prefix");
        f.prefix = *prefix;
    }
    return f;
}

Tensor token_spans(const Tensor& documents_, const std::optional<Tensor>& groups_) {
    require_cuda(documents_);
    require_ints(documents_, documents_, at::kInt, "documents");
    if (documents_.dim() != 1 && documents_.dim() != 2) mismatch("documents of size " + shape_text(documents_) + ": (N, B) or (N) expected");
    if (groups_) {
        require_ints(*groups_, documents_, at::kInt, "groups");
        if (groups_->sizes() != documents_.sizes()) mismatch("groups of size " + shape_text(*groups_) + ", but documents of size " + shape_text(documents_));
    }
    const Tensor documents = colmajor(documents_), groups = groups_ ? colmajor(*groups_) : Tensor();
    Call call(documents, "circatt.spans");
    const int64_t N = documents.size(0), B = documents.dim() == 2 ? documents.size(1) : 1;
    Tensor spans = empty_cm({4, N, B}, documents, at::kInt);
    check(ca_token_spans(static_cast<const int32_t*>(ptr(documents)), static_cast<const int32_t*>(ptr(groups)), int_of(N, "N"), int_of(B, "B"),
                         static_cast<int32_t*>(ptr(spans)), call.stream));
    return spans;
}

Tensor paged_window(const Tensor& q_, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& starts,
                    const Tensor& lengths, int64_t left, int64_t sinks, std::optional<double> scale, std::optional<double> cap,
                    const std::optional<Tensor>& slopes, const std::optional<Tensor>& prefix) {
    check_tokens(q_, "q", true);
    const Form form = form_of(q_, cap, slopes, std::nullopt, prefix);
    if (prefix && (prefix->dim() != 1 || prefix->sizes() != lengths.sizes() || !prefix->is_contiguous()))
        mismatch("prefix of size " + shape_text(*prefix) + ": one for each sequence expected");
    check_cache(k_pages, q_, v_pages, "k_pages");
    check_cache(v_pages, q_, k_pages, "v_pages");
    const Tensor q = ready(q_.detach());
    Call call(q, "circatt.paged");
    ca_seq_desc d{};
    d.dtype = dtype_code(q);
    d.dim = int_of(q.size(0), "D");
    d.heads_q = int_of(q.size(1), "heads");
    d.heads_kv = int_of(k_pages.size(2), "heads");
    d.tokens = int_of(q.size(2), "T");
    d.batch = 1;
    d.left = int_of(left, "left");
    d.sinks = int_of(sinks, "sinks");
    d.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)q.size(0)));
    const ca_pages p = pages_of(q, k_pages, table, starts, lengths);
    Tensor y = empty_cm(q.sizes(), q, q.scalar_type());
    const ca_seq_view vq = view(q), vy = view(y);
    const ca_page_view kp = page_view(k_pages), vp = page_view(v_pages);
    const ca_seq_form vf = form.view();
    check(ca_paged_window_form(&d, &vf, &vq, &kp, &vp, &p, &vy, call.stream));
    return y;
}

// ---------------------------------------------------------------- the pages of a cache
ca_table table_of(const Tensor& table, const Tensor& refs, const Tensor& lengths, int64_t page) {
    require_cuda(table);
    require_ints(table, table, at::kInt, "table");
    require_ints(refs, table, at::kInt, "refs");
    if (table.dim() != 2 || refs.dim() != 1) mismatch("table of size " + shape_text(table) + ", refs of size " + shape_text(refs) + ": (width, S) and (pages) expected");
    if ((table.numel() && !is_colmajor(table)) || !refs.is_contiguous()) mismatch("table and refs must be dense (table column-major)");
    if (lengths.defined()) {
        require_ints(lengths, table, at::kInt, "lengths");
        if (lengths.dim() != 1 || lengths.size(0) != table.size(1) || !lengths.is_contiguous()) mismatch("lengths of size " + shape_text(lengths) + ": one for each sequence expected");
    }
    return ca_table{static_cast<const int32_t*>(ptr(table)), static_cast<const int32_t*>(ptr(refs)), static_cast<const int32_t*>(ptr(lengths)),
                    int_of(table.size(0), "width"), int_of(table.size(1), "S"), int_of(page, "page"), int_of(refs.size(0), "pages")};
}

// Their strides in bytes; pools are written in place, so that they have to lie as they are needed.
std::vector<ca_pool> pools_of(const std::vector<Tensor>& pools, const Tensor& table, const Tensor& refs) {
    if (pools.empty()) mismatch("no pools: at least one tensor (D, page, heads, pages) expected");
    std::vector<ca_pool> out;
    for (const Tensor& p : pools) {
        require_cuda(p);
        if (p.device() != table.device()) raise(PyExc_RuntimeError, "a pool is on " + p.device().str() + ", not on " + table.device().str());
        if (p.dim() != 4 || p.size(3) != refs.size(0)) mismatch("a pool of size " + shape_text(p) + ": (D, page, heads, pages) with " + std::to_string(refs.size(0)) + " pages expected");
        if (p.size(1) != pools[0].size(1)) mismatch("pools with pages of " + std::to_string(pools[0].size(1)) + " and " + std::to_string(p.size(1)) + " tokens");
        const int64_t e = p.element_size();
        if (!as_it_is(p) || p.size(0) * e % 16) mismatch("a pool's features must be contiguous, and its address, strides and the features of a head multiples of 16 bytes");
        auto st = [&](int64_t i) { return p.size(i) > 1 ? p.stride(i) * e : 16; };
        out.push_back(ca_pool{p.data_ptr(), st(1), st(2), st(3), int_of(p.size(0) * e, "D"), int_of(p.size(1), "page"), int_of(p.size(2), "heads")});
    }
    return out;
}

Tensor like_ints(const Tensor& t) { return empty_cm(t.sizes(), t, at::kInt); }

std::tuple<Tensor, Tensor, Tensor> advance_pages(const Tensor& table, const Tensor& refs, const Tensor& starts, const Tensor& lengths, int64_t page,
                                                 int64_t left, int64_t sinks) {
    const ca_table t = table_of(table, refs, lengths, page);
    require_ints(starts, table, at::kInt, "starts");
    if (starts.dim() != 1 || starts.size(0) != table.size(1) + 1 || !starts.is_contiguous()) mismatch("starts of size " + shape_text(starts) + ": (S + 1) expected");
    Call call(table, "circatt.pages.advance");
    const Tensor out = like_ints(table), counts = like_ints(refs), missing = at::empty({1}, table.options()), work = scratch(ca_pages_workspace(&t), table);
    check(ca_advance_pages(&t, starts.data_ptr<int32_t>(), int_of(left, "left"), int_of(sinks, "sinks"), static_cast<int32_t*>(ptr(out)), static_cast<int32_t*>(ptr(counts)),
                           missing.data_ptr<int32_t>(), ptr(work), call.stream));
    return {out, counts, missing};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> fork_pages(const std::vector<Tensor>& pools_, const Tensor& table, const Tensor& refs, const Tensor& lengths,
                                                      const Tensor& parents) {
    const std::vector<ca_pool> pools = pools_of(pools_, table, refs);
    const ca_table t = table_of(table, refs, lengths, pools[0].tokens);
    require_ints(parents, table, at::kInt, "parents");
    if (parents.dim() != 1 || parents.size(0) != table.size(1) || !parents.is_contiguous()) mismatch("parents of size " + shape_text(parents) + ": one for each sequence expected");
    Call call(table, "circatt.pages.fork");
    const Tensor out = like_ints(table), counts = like_ints(refs), n = like_ints(lengths), missing = at::empty({1}, table.options()),
                 work = scratch(ca_pages_workspace(&t), table);
    check(ca_fork_pages(&t, static_cast<const int32_t*>(ptr(parents)), pools.data(), (int32_t)pools.size(), static_cast<int32_t*>(ptr(out)), static_cast<int32_t*>(ptr(counts)),
                        static_cast<int32_t*>(ptr(n)), missing.data_ptr<int32_t>(), ptr(work), call.stream));
    return {out, counts, n, missing};
}

std::tuple<Tensor, Tensor, Tensor> compact_pages(const std::vector<Tensor>& pools_, const Tensor& table, const Tensor& refs) {
    const std::vector<ca_pool> pools = pools_of(pools_, table, refs);
    const ca_table t = table_of(table, refs, Tensor(), pools[0].tokens);
    Call call(table, "circatt.pages.compact");
    const Tensor out = like_ints(table), counts = like_ints(refs), live = at::empty({1}, table.options()), work = scratch(ca_pages_workspace(&t), table);
    check(ca_compact_pages(&t, pools.data(), (int32_t)pools.size(), static_cast<int32_t*>(ptr(out)), static_cast<int32_t*>(ptr(counts)), live.data_ptr<int32_t>(), ptr(work),
                           call.stream));
    return {out, counts, live};
}

// ---------------------------------------------------------------- window attention
struct Window {
    int64_t left, right, sinks;
    double scale;
};

ca_seq_desc window_desc(const Tensor& q, const Tensor& k, const Window& w) {
    ca_seq_desc d{};
    d.dtype = dtype_code(q);
    d.dim = int_of(q.size(0), "D");
    d.heads_q = int_of(q.size(1), "heads");
    d.heads_kv = int_of(k.size(1), "heads");
    d.tokens = int_of(q.size(2), "N");
    d.batch = int_of(q.size(3), "B");
    d.left = int_of(w.left, "left");
    d.right = int_of(w.right, "right");
    d.sinks = int_of(w.sinks, "sinks");
    d.scale = (float)w.scale;
    return d;
}

struct WindowOut { Tensor y, rest, lse; };

// `train`: also what the backward needs, the rows' sums and (16-bit types) what rounding took from y.
WindowOut window_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Window& w, const Form& form, bool train) {
    Call call(q, "circatt.window");
    const ca_seq_desc d = window_desc(q, k, w);
    WindowOut o;
    o.y = empty_cm(q.sizes(), q, q.scalar_type());
    if (train) o.lse = at::empty({q.size(1) * q.size(2) * q.size(3)}, q.options().dtype(at::kFloat));
    if (train && q.element_size() == 2) o.rest = empty_cm(q.sizes(), q, q.scalar_type());
    const ca_seq_view vq = view(q), vk = view(k), vv = view(v), vy = view(o.y), vr = o.rest.defined() ? view(o.rest) : ca_seq_view{};
    const ca_seq_form vf = form.view();
    check(ca_window_form_fwd(&d, &vf, &vq, &vk, &vv, static_cast<const int32_t*>(ptr(lengths)), &vy, o.rest.defined() ? &vr : nullptr, fptr(o.lse), call.stream));
    return o;
}

struct WindowFn : public Function<WindowFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const std::optional<Tensor>& lengths,
                          int64_t left, int64_t right, int64_t sinks, double scale, double cap, const std::optional<Tensor>& slopes_,
                          const std::optional<Tensor>& spans_) {
        const Tensor slopes = slopes_ ? *slopes_ : Tensor(), spans = spans_ ? *spans_ : Tensor();
        const Tensor q = ready(q_), k = ready(k_), v = ready(v_), n = lengths ? *lengths : Tensor();
        const WindowOut o = window_fwd(q, k, v, n, Window{left, right, sinks, scale}, Form{cap, slopes, spans, Tensor()}, true);
        ctx->save_for_backward({q, k, v, o.y, o.lse, n, o.rest, slopes, spans});
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["left"] = left;
        ctx->saved_data["right"] = right;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &y = s[3], &lse = s[4], &n = s[5], &rest = s[6], dy = ready(g[0]);
        const Window w{ctx->saved_data["left"].toInt(), ctx->saved_data["right"].toInt(), ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble()};
        Call call(q, "circatt.window.bwd");
        const ca_seq_desc d = window_desc(q, k, w);
        Tensor dq = empty_cm(q.sizes(), q, q.scalar_type()), dk = empty_cm(k.sizes(), k, k.scalar_type()), dv = empty_cm(v.sizes(), v, v.scalar_type());
        const Tensor work = scratch(ca_window_bwd_workspace(&d), q);
        const ca_seq_view vq = view(q), vk = view(k), vv = view(v), vy = view(y), vdy = view(dy), vdq = view(dq), vdk = view(dk), vdv = view(dv),
                          vr = rest.defined() ? view(rest) : ca_seq_view{};
        const ca_seq_form vf = Form{ctx->saved_data["cap"].toDouble(), s[7], s[8], Tensor()}.view();
        check(ca_window_form_bwd(&d, &vf, &vq, &vk, &vv, &vy, rest.defined() ? &vr : nullptr, &vdy, static_cast<const int32_t*>(ptr(n)), fptr(lse), &vdq, &vdk, &vdv, ptr(work), call.stream));
        return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor window(const Tensor& q, const Tensor& k, const Tensor& v, int64_t left, int64_t right, int64_t sinks, const std::optional<Tensor>& lengths,
              std::optional<double> scale_, std::optional<double> cap, const std::optional<Tensor>& slopes, const std::optional<Tensor>& spans) {
    require_cuda(q);
    require_like(k, q, "k");
    require_like(v, q, "v");
    if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(2) != k.size(2) || q.size(3) != k.size(3))
        mismatch("q, k, v of sizes " + shape_text(q) + ", " + shape_text(k) + ", " + shape_text(v) + ": (D, heads, N, B) expected, k and v alike");
    if (lengths) {
        require_ints(*lengths, q, at::kInt, "lengths");
        if (lengths->dim() != 1 || lengths->size(0) != q.size(3) || !lengths->is_contiguous()) mismatch("lengths of size " + shape_text(*lengths) + ": one for each of the batch expected");
    }
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)q.size(0));
    const Form form = form_of(q, cap, slopes, spans, std::nullopt);
    if (!tracked({&q, &k, &v}))
        return window_fwd(ready(q), ready(k), ready(v), lengths ? *lengths : Tensor(), Window{left, right, sinks, scale}, form, false).y;
    return WindowFn::apply(q, k, v, lengths, left, right, sinks, scale, form.cap, slopes, spans);
}

}  // namespace

void bind_tokens(py::module_& m) {
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("rotary", &rotary, release());
    m.def("rotary_append", &rotary_append, release());
    m.def("token_spans", &token_spans, release());
    m.def("advance_pages", &advance_pages, release());
    m.def("fork_pages", &fork_pages, release());
    m.def("compact_pages", &compact_pages, release());
    m.def("window_attention", &window, release());
    m.def("paged_window_attention", &paged_window, release());
}
