// Host binding of rotary positions and the paged cache (part of na_torch.cpp):
// the checks and the C call of an ordinary call, in C++.  Each function
// returns None for anything it does not take as it is (another device or
// dtype, a copy to make, gradients where there are none, an argument to
// refuse): positions.py and paged.py then check it and name what is wrong.
#pragma once

#include <torch/csrc/autograd/custom_function.h>

namespace {

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? NATTEN_F32 : t == at::kHalf ? NATTEN_F16 : t == at::kBFloat16 ? NATTEN_BF16 : -1;
}

// A plain strided device tensor with elements (no subclass, no pending
// conjugation or negation, no forward-mode tangent), sizes that fit the
// descriptors.
bool plain(const at::Tensor& t) {
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.numel() == 0) return false;
    const auto ks = t.unsafeGetTensorImpl()->key_set();
    if (ks.has(c10::DispatchKey::Python) || ks.has(c10::DispatchKey::FuncTorchBatched) ||
        ks.has(c10::DispatchKey::FuncTorchGradWrapper) || t.is_conj() || t.is_neg() || t._fw_grad(0).defined())
        return false;
    for (int64_t n : t.sizes())
        if (n > INT32_MAX) return false;
    return true;
}

// plain, unit innermost stride, the device and dtype of `like`
bool operand(const at::Tensor& t, const at::Tensor& like) {
    return plain(t) && t.stride(-1) == 1 && t.device() == like.device() && t.scalar_type() == like.scalar_type();
}

bool index_rows(const at::Tensor& t, const at::Tensor& like) {
    return plain(t) && t.device() == like.device() && t.scalar_type() == at::kInt && t.stride(-1) == 1;
}

// [B, *sp, H, D] (trailing 1) or [B, *sp, H] (trailing 0)
natten_layout_t layout_of(const at::Tensor& t, int trailing) {
    natten_layout_t l{};
    const auto st = t.strides();
    const int rank = static_cast<int>(t.dim()) - 2 - trailing;
    l.batch = st[0];
    for (int i = 0; i < rank; ++i) l.axis[3 - rank + i] = st[1 + i];
    l.head = st[1 + rank];
    return l;
}

struct DeviceOf {
    c10::OptionalDeviceGuard guard;
    explicit DeviceOf(const at::Tensor& t) {
        if (FusedCall::current_index() != t.get_device()) guard.reset_device(t.device());
    }
};

// ---------------------------------------------------------------------------
// rotary
// ---------------------------------------------------------------------------

struct TurnParams {
    int64_t turned, axes;
    bool interleaved;
    double magnitude;
};

std::vector<at::Tensor> turn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                             const at::Tensor& table, const TurnParams& p, bool inverse) {
    const DeviceOf dev(q);
    const int rank = static_cast<int>(q.dim()) - 3;
    natten_rotary_t r{};
    r.batch = static_cast<int32_t>(q.size(0));
    for (int i = 0; i < 3; ++i) r.length[i] = 1;
    for (int i = 0; i < rank; ++i) r.length[3 - rank + i] = static_cast<int32_t>(q.size(1 + i));
    r.dim = static_cast<int32_t>(q.size(-1));
    r.dtype = dtype_code(q.scalar_type());
    r.heads_q = static_cast<int32_t>(q.size(-2));
    r.heads_k = k.defined() ? static_cast<int32_t>(k.size(-2)) : 0;
    r.axes = static_cast<int32_t>(p.axes);
    r.turned = static_cast<int32_t>(p.turned);
    r.interleaved = p.interleaved;
    r.inverse = inverse;
    r.magnitude = static_cast<float>(p.magnitude);
    if (positions.defined()) {
        const int64_t lead = positions.dim() - (p.axes > 1 ? 1 : 0);
        r.position_bits = positions.scalar_type() == at::kInt ? 32 : 64;
        r.position_stride[0] =
            lead == rank + 1 && positions.size(0) > 1 ? positions.numel() / positions.size(0) : 0;
        r.position_stride[1] = p.axes;
        r.position_stride[2] = 1;
    }
    std::vector<at::Tensor> out{alloc(q.sizes(), q.scalar_type(), q.device())};
    if (k.defined()) out.push_back(alloc(k.sizes(), k.scalar_type(), k.device()));
    const natten_layout_t lq = layout_of(q, 1), lqo = layout_of(out[0], 1);
    natten_layout_t lk{}, lko{};
    if (k.defined()) {
        lk = layout_of(k, 1);
        lko = layout_of(out[1], 1);
    }
    const int rc = natten_hip_rotary(
        &r, reinterpret_cast<const uint64_t*>(table.data_ptr()), positions.defined() ? positions.data_ptr() : nullptr,
        q.data_ptr(), &lq, out[0].data_ptr(), &lqo, k.defined() ? k.data_ptr() : nullptr, k.defined() ? &lk : nullptr,
        k.defined() ? out[1].data_ptr() : nullptr, k.defined() ? &lko : nullptr,
        reinterpret_cast<void*>(current_stream(q)));
    if (rc != NATTEN_OK) raise_status(rc, "rotary");
    return out;
}

// The gradient of a turn is the turn back, through this node again.
struct TurnFunction : public torch::autograd::Function<TurnFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                  const std::optional<at::Tensor>& key,
                                                  const std::optional<at::Tensor>& at_positions,
                                                  const at::Tensor& table, int64_t turned, int64_t axes,
                                                  bool interleaved, double magnitude, bool inverse) {
        const at::Tensor k = key.value_or(at::Tensor()), positions = at_positions.value_or(at::Tensor());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({positions, table});
        ctx->saved_data["p"] = c10::List<int64_t>({turned, axes, interleaved, inverse});
        ctx->saved_data["m"] = magnitude;
        return turn(q, k, positions, table, {turned, axes, interleaved, magnitude}, inverse);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto p = ctx->saved_data["p"].toIntVector();
        const double m = ctx->saved_data["m"].toDouble();
        std::vector<at::Tensor> given;
        for (at::Tensor& g : grads)
            if (g.defined()) given.push_back(g.stride(-1) == 1 ? g : g.contiguous());
        torch::autograd::variable_list res(9);
        if (given.empty()) return res;
        const std::optional<at::Tensor> second = given.size() > 1 ? std::make_optional(given[1]) : std::nullopt;
        const std::optional<at::Tensor> positions = saved[0].defined() ? std::make_optional(saved[0]) : std::nullopt;
        const auto back = apply(given[0], second, positions, saved[1], p[0], p[1], p[2] != 0, m, p[3] == 0);
        size_t next = 0;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined()) res[i] = back[next++];
        return res;
    }
};

// (turned q,) or (q, k); None: not taken.
pybind11::object rotary(const at::Tensor& q, const std::optional<at::Tensor>& k,
                        const std::optional<at::Tensor>& positions, const at::Tensor& table, int64_t turned,
                        int64_t axes, bool interleaved, double magnitude) {
    if (!plain(q) || q.dim() < 4 || q.dim() > 6 || !operand(q, q) || dtype_code(q.scalar_type()) < 0 ||
        q.size(-1) > 256 || turned > q.size(-1) || !plain(table))
        return pybind11::none();
    if (k.has_value()) {
        if (!operand(*k, q) || k->dim() != q.dim() || k->size(-1) != q.size(-1)) return pybind11::none();
        for (int64_t i = 0; i < q.dim() - 2; ++i)
            if (k->size(i) != q.size(i)) return pybind11::none();
    }
    const int64_t rank = q.dim() - 3;
    at::Tensor pos;
    if (positions.has_value()) {
        pos = *positions;
        const int64_t tail = axes > 1 ? 1 : 0, lead = pos.dim() - tail;
        if (!plain(pos) || pos.device() != q.device() || !pos.is_contiguous() ||
            (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) || (lead != rank && lead != rank + 1) ||
            (tail && pos.size(-1) != axes) || (lead == rank + 1 && pos.size(0) != 1 && pos.size(0) != q.size(0)))
            return pybind11::none();
        for (int64_t i = 0; i < rank; ++i)
            if (pos.size(lead - rank + i) != q.size(1 + i)) return pybind11::none();
    } else if (axes != rank) {
        return pybind11::none();
    }
    const at::Tensor key = k.has_value() ? *k : at::Tensor();
    std::vector<at::Tensor> out;
    if (at::GradMode::is_enabled() && (q.requires_grad() || (key.defined() && key.requires_grad())))
        out = TurnFunction::apply(q, k, positions, table, turned, axes, interleaved, magnitude, false);
    else
        out = turn(q, key, pos, table, {turned, axes, interleaved, magnitude}, false);
    if (out.size() == 1) return pybind11::make_tuple(std::move(out[0]));
    return pybind11::make_tuple(std::move(out[0]), std::move(out[1]));
}

// ---------------------------------------------------------------------------
// paged cache
// ---------------------------------------------------------------------------

bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : ts)
        if (t && t->requires_grad()) return true;
    return false;
}

// The cache's own tensors, for a batch like `x`'s.
bool cache_ok(const at::Tensor& x, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table,
              const at::Tensor& lens, const std::optional<at::Tensor>& news) {
    if (!plain(x) || x.dim() != 4 || !operand(x, x) || dtype_code(x.scalar_type()) < 0 || !operand(kp, x) ||
        !operand(vp, x) || kp.dim() != 4 || vp.dim() != 4)
        return false;
    for (int i = 0; i < 3; ++i)
        if (kp.size(i) != vp.size(i)) return false;
    if (!index_rows(table, x) || table.dim() != 2 || table.size(0) != x.size(0)) return false;
    if (!index_rows(lens, x) || lens.dim() != 1 || lens.size(0) != x.size(0)) return false;
    return !news.has_value() || (index_rows(*news, x) && news->dim() == 1 && news->size(0) == x.size(0));
}

natten_paged_t paged_problem(const at::Tensor& x, int64_t heads_q, const at::Tensor& kp, const at::Tensor& vp,
                             const at::Tensor& table) {
    natten_paged_t p{};
    p.batch = static_cast<int32_t>(x.size(0));
    p.tokens = static_cast<int32_t>(x.size(1));
    p.heads_q = static_cast<int32_t>(heads_q);
    p.pages = static_cast<int32_t>(kp.size(0));
    p.page_size = static_cast<int32_t>(kp.size(1));
    p.heads_kv = static_cast<int32_t>(kp.size(2));
    p.dim_qk = static_cast<int32_t>(kp.size(3));
    p.dim_v = static_cast<int32_t>(vp.size(3));
    p.dtype = dtype_code(x.scalar_type());
    p.table_width = static_cast<int32_t>(table.size(1));
    p.table_stride = table.stride(0);
    for (int i = 0; i < 3; ++i) {
        p.key_stride[i] = kp.stride(i);
        p.value_stride[i] = vp.stride(i);
    }
    p.dilation = 1;
    return p;
}

const int32_t* rows_of(const std::optional<at::Tensor>& t) {
    return t.has_value() ? t->data_ptr<int32_t>() : nullptr;
}

// (turned q,) or (); None: not taken.
pybind11::object paged_append(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kp,
                              const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens,
                              const std::optional<at::Tensor>& news, const std::optional<at::Tensor>& query,
                              const std::optional<at::Tensor>& turns, int64_t turned, int64_t axes, bool interleaved,
                              double magnitude) {
    if (!cache_ok(key, kp, vp, table, lens, news) || !operand(value, key) || value.dim() != 4) return pybind11::none();
    for (int i = 0; i < 3; ++i)
        if (value.size(i) != key.size(i)) return pybind11::none();
    if (key.size(2) != kp.size(2) || key.size(3) != kp.size(3) || value.size(3) != vp.size(3))
        return pybind11::none();
    for (int i = 0; i < 3; ++i)
        if ((kp.stride(i) == 0 && kp.size(i) > 1) || (vp.stride(i) == 0 && vp.size(i) > 1)) return pybind11::none();
    if (query.has_value() && (!operand(*query, key) || query->dim() != 4 || query->size(0) != key.size(0) ||
                              query->size(1) != key.size(1) || query->size(3) != key.size(3)))
        return pybind11::none();
    if (turns.has_value() && (axes != 1 || turned > key.size(3) || !plain(*turns))) return pybind11::none();
    if (needs_grad({&key, &value, &kp, &vp, query.has_value() ? &*query : nullptr})) return pybind11::none();
    const DeviceOf dev(key);
    const natten_paged_t p = paged_problem(key, query.has_value() ? query->size(2) : 0, kp, vp, table);
    natten_rotary_t r{};
    r.axes = 1;
    r.turned = static_cast<int32_t>(turned);
    r.interleaved = interleaved;
    r.magnitude = static_cast<float>(magnitude);
    at::Tensor out;
    natten_layout_t lq{}, lqo{};
    const natten_layout_t lk = layout_of(key, 1), lv = layout_of(value, 1);
    if (query.has_value()) {
        out = alloc(query->sizes(), query->scalar_type(), query->device());
        lq = layout_of(*query, 1);
        lqo = layout_of(out, 1);
    }
    const bool q = query.has_value();
    const int rc = natten_hip_paged_append(
        &p, turns.has_value() ? &r : nullptr,
        turns.has_value() ? reinterpret_cast<const uint64_t*>(turns->data_ptr()) : nullptr, table.data_ptr<int32_t>(),
        lens.data_ptr<int32_t>(), rows_of(news), key.data_ptr(), &lk, value.data_ptr(), &lv,
        q ? query->data_ptr() : nullptr, q ? &lq : nullptr, q ? out.data_ptr() : nullptr, q ? &lqo : nullptr,
        kp.data_ptr(), vp.data_ptr(), reinterpret_cast<void*>(current_stream(key)));
    if (rc != NATTEN_OK) raise_status(rc, "paged_append");
    return q ? pybind11::make_tuple(std::move(out)) : pybind11::make_tuple();
}

// A positive int, or a tuple of one: 0 when it is something else.
int64_t positive(pybind11::handle h) {
    PyObject* o = h.ptr();
    if (PyTuple_CheckExact(o) && PyTuple_GET_SIZE(o) == 1) o = PyTuple_GET_ITEM(o, 0);
    if (!PyLong_CheckExact(o)) return 0;
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) PyErr_Clear();
    return x > 0 && x <= INT32_MAX ? x : 0;
}

// (out, lse); None: not taken.
pybind11::object paged_forward(const at::Tensor& query, const at::Tensor& kp, const at::Tensor& vp,
                               const at::Tensor& table, const at::Tensor& lens, const std::optional<at::Tensor>& news,
                               pybind11::handle kernel, pybind11::handle dilation, pybind11::handle scale) {
    if (!cache_ok(query, kp, vp, table, lens, news) || query.size(3) != kp.size(3) ||
        query.size(2) % kp.size(2) != 0 || needs_grad({&query, &kp, &vp}))
        return pybind11::none();
    natten_paged_t p = paged_problem(query, query.size(2), kp, vp, table);
    const bool windowed = kernel.ptr() != Py_None;
    const int64_t k = windowed ? positive(kernel) : 0, d = positive(dilation);
    if (d == 0 || (windowed ? k == 0 : d != 1)) return pybind11::none();
    p.kernel = static_cast<int32_t>(k);
    p.dilation = static_cast<int32_t>(d);
    if (scale.ptr() == Py_None) p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(query.size(3))));
    else if (PyFloat_CheckExact(scale.ptr())) p.scale = static_cast<float>(PyFloat_AS_DOUBLE(scale.ptr()));
    else return pybind11::none();
    const DeviceOf dev(query);
    const int64_t out_shape[4] = {query.size(0), query.size(1), query.size(2), vp.size(3)};
    Block blk;
    blk.add(numel(out_shape) * static_cast<int64_t>(c10::elementSize(query.scalar_type())));
    blk.add(numel({out_shape, 3}) * static_cast<int64_t>(sizeof(float)));
    blk.allocate(query.device());
    at::Tensor out = blk.part(0, out_shape, query.scalar_type());
    at::Tensor lse = blk.part(1, {out_shape, 3}, at::kFloat);
    const int64_t stream = current_stream(query);
    const int64_t need = std::max<int64_t>(natten_hip_paged_workspace(&p), 0);
    const Workspace work(static_cast<size_t>(need), reinterpret_cast<hipStream_t>(stream));
    const natten_layout_t lq = layout_of(query, 1), lo = layout_of(out, 1), ll = layout_of(lse, 0);
    const int rc = natten_hip_paged_forward(&p, table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), rows_of(news),
                                            query.data_ptr(), &lq, kp.data_ptr(), vp.data_ptr(), out.data_ptr(), &lo,
                                            lse.data_ptr<float>(), &ll, work.ptr, need,
                                            reinterpret_cast<void*>(stream));
    if (rc != NATTEN_OK) raise_status(rc, "paged_forward");
    return pybind11::make_tuple(std::move(out), std::move(lse));
}

}  // namespace
