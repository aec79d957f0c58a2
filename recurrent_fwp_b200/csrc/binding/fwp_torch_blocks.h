// Host path of the operators of a state-space layer: causal_conv, selective_scan, block_norm.  Included by fwp_torch.cpp inside its
// anonymous namespace; the division of labour with the Python modules is the one described there.  Optional arguments are None.

// Borrowed arguments, null where None; false when one of them is neither None nor a plain tensor (see tensors()).
template <size_t K>
bool optional_tensors(PyObject* const* args, std::array<const Tensor*, K>& out) {
    if (at::tracer::impl::is_dispatch_enabled()) return false;
    constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
    for (size_t i = 0; i < K; i++) {
        out[i] = nullptr;
        if (args[i] == Py_None) continue;
        if (!THPVariable_Check(args[i])) return false;
        const Tensor& t = THPVariable_Unpack(args[i]);
        const auto* impl = t.unsafeGetTensorImpl();
        if (impl->key_set().has_any(wrappers) || (impl->autograd_meta() && torch::autograd::isFwGradDefined(t))) return false;
        out[i] = &t;
    }
    return true;
}
template <size_t K>
bool any_needs_grad(const std::array<const Tensor*, K>& in) {
    if (!at::GradMode::is_enabled()) return false;
    for (auto* t : in)
        if (t && t->requires_grad()) return true;
    return false;
}
// A state is not saved: no backward reads it, and its owner may overwrite it before.
template <class NodeT, size_t K>
std::shared_ptr<NodeT> optional_node(const std::array<const Tensor*, K>& in, size_t state = K) {
    auto node = std::shared_ptr<NodeT>(new NodeT(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    edges.reserve(K);
    for (auto* t : in) edges.push_back(t && t->requires_grad() ? torch::autograd::impl::gradient_edge(*t) : torch::autograd::Edge());
    node->set_next_edges(std::move(edges));
    for (size_t i = 0; i < K; i++) node->save(in[i] && i != state ? *in[i] : Tensor());
    return node;
}

constexpr int64_t kMaxSize = 0x7fffffff;

// a (N, L, D) stream of the first one's type, device and shape with unit inner stride
bool rows_like(const Tensor& t, at::ScalarType type, const at::Device& dev, at::IntArrayRef shape) {
    return t.defined() && t.layout() == at::kStrided && t.scalar_type() == type && t.device() == dev && t.sizes() == shape &&
           (t.size(-1) == 1 || t.stride(-1) == 1);
}
bool first_rows(const Tensor& t) {
    if (!t.defined() || t.dim() < 2 || t.dim() > 3 || !t.is_cuda() || t.layout() != at::kStrided) return false;
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) return false;
    for (int64_t s : t.sizes())
        if (s > kMaxSize) return false;
    return t.size(-1) == 1 || t.stride(-1) == 1;
}
// fp32 weights: contiguous, of this shape
bool weight_like(const Tensor* t, const at::Device& dev, at::IntArrayRef shape) {
    return !t || (t->layout() == at::kStrided && t->scalar_type() == at::kFloat && t->device() == dev && t->sizes() == shape && t->is_contiguous());
}
// an fp32 state that is written in place: no two of its elements share memory through an expanded dimension
bool state_like(const Tensor* t, const at::Device& dev, at::IntArrayRef shape) {
    if (!t) return true;
    if (!rows_like(*t, at::kFloat, dev, shape)) return false;
    for (int64_t i = 0; i < t->dim(); i++)
        if (t->size(i) > 1 && t->stride(i) == 0) return false;
    return true;
}
bool lengths_like(const Tensor* t, const at::Device& dev, int64_t N) {
    return !t || (t->layout() == at::kStrided && t->scalar_type() == at::kInt && t->device() == dev && t->dim() == 1 && t->size(0) == N &&
                  t->is_contiguous());
}

// an (N, L, D) or (L, D) tensor as the C interface's descriptor
struct RowsDesc {
    fwp_tensor d;
    explicit RowsDesc(const Tensor& t) : d{nullptr, {0, 0, 0, 1}} {
        if (!t.defined()) return;
        d.data = t.data_ptr();
        const int64_t k = t.dim();
        d.stride[0] = k == 3 ? t.stride(0) : 0;
        d.stride[2] = t.stride(k - 2);
    }
    explicit RowsDesc(const Tensor* t) : RowsDesc(t ? *t : Tensor()) {}
    operator const fwp_tensor*() const { return &d; }
};
// B or C, (N, L, S) or (N, L, G, S), in the order (N, G, L, S)
struct GroupDesc {
    fwp_tensor d;
    explicit GroupDesc(const Tensor& t) : d{t.data_ptr(), {t.stride(0), t.dim() == 4 ? t.stride(2) : 0, t.stride(1), 1}} {}
    operator const fwp_tensor*() const { return &d; }
};
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const float* floats(const Tensor* t) { return t ? t->data_ptr<float>() : nullptr; }
const int* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int>() : nullptr; }
const int* ints(const Tensor* t) { return t ? t->data_ptr<int>() : nullptr; }

// a tensor of x's shape whose rows lie in x's order of sequences and steps, so that a (len, batch, ...) model stays in its order
Tensor rows_as(const Tensor& x, at::ScalarType type) {
    if (x.dim() == 3) {
        if (x.stride(0) < x.stride(1) && x.size(0) > 1) return empty({x.size(1), x.size(0), x.size(2)}, type, x).transpose(0, 1);
        return empty({x.size(0), x.size(1), x.size(2)}, type, x);
    }
    return empty({x.size(0), x.size(1)}, type, x);
}
Tensor empty_as(const Tensor& t) { return Tensor(at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), std::nullopt)); }
Tensor vector_for(const Tensor& w) { return w.defined() ? empty_as(w) : Tensor(); }
Tensor scratch_of(int64_t n, const Tensor& like) { return n > 0 ? empty({n}, at::kFloat, like) : Tensor(); }
int flag(PyObject* o) { return PyObject_IsTrue(o); }

// ------------------------------------------------------------------ causal convolution
struct ConvNode final : public OpNode {
    int silu = 1;
    std::string name() const override { return "CausalConvBackward"; }
    variable_list apply(variable_list&& g) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const auto t = unpack(user), o = unpack(own);
        const Tensor &x = t[0], &w = t[1], &b = t[2], &lengths = t[4], &start = o[0];
        const int64_t N = x.size(0), L = x.size(1), D = x.size(2), K = w.size(1);
        const Tensor gy = incoming(g[0], x, x.sizes());
        Tensor gx = rows_as(x, x.scalar_type()), gw = vector_for(w), gb = vector_for(b);
        const int64_t need = fwp_causal_conv_backward_scratch_floats(N, L, D, K);
        const Tensor scratch = scratch_of(need, x);
        check(fwp_causal_conv_backward(N, L, D, K, RowsDesc(x), floats(w), floats(b), RowsDesc(start), ints(lengths), RowsDesc(gy), RowsDesc(gx),
                                       floats(gw), floats(gb), floats(scratch), need, silu, dtype_code(x), stream_of(x), x.device().index()),
              "causal_conv_backward");
        return {gx, gw, gb, Tensor(), Tensor()};
    }
};

// x, weight, bias, state, lengths, silu
PyObject* causal_conv(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    std::array<const Tensor*, 5> in;
    if (n != 6 || !optional_tensors(args, in) || !in[0] || !in[1]) return not_implemented();
    const int silu = flag(args[5]);
    if (silu < 0) return nullptr;
    const Tensor &x = *in[0], &w = *in[1];
    if (!first_rows(x) || x.dim() != 3 || w.dim() != 2) return not_implemented();
    const int64_t N = x.size(0), L = x.size(1), D = x.size(2), K = w.size(1);
    const auto dev = x.device();
    if (!weight_like(&w, dev, {D, K}) || !weight_like(in[2], dev, {D}) || !state_like(in[3], dev, {N, K - 1, D}) || !lengths_like(in[4], dev, N))
        return not_implemented();
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        const bool grad = any_needs_grad(in);
        out = rows_as(x, x.scalar_type());
        Tensor start;
        if (grad && in[3]) start = in[3]->detach().clone(at::MemoryFormat::Contiguous);
        check(fwp_causal_conv_forward(N, L, D, K, RowsDesc(x), floats(&w), floats(in[2]), RowsDesc(K > 1 ? in[3] : nullptr), ints(in[4]),
                                      RowsDesc(out), silu, dtype_code(x), stream_of(x), dev.index()), "causal_conv_forward");
        if (grad) {
            auto node = optional_node<ConvNode>(in, 3);
            node->silu = silu;
            node->keep({start});
            torch::autograd::create_gradient_edge(out, node);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------- selective scan
struct ScanNode final : public OpNode {
    int softplus = 1;
    std::string name() const override { return "SelectiveScanBackward"; }
    variable_list apply(variable_list&& g) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const auto t = unpack(user), o = unpack(own);
        const Tensor &x = t[0], &dt = t[1], &A = t[2], &B = t[3], &C = t[4], &skip = t[5], &z = t[6], &bias = t[7], &lengths = t[9];
        const int64_t N = x.size(0), L = x.size(1), D = x.size(2), S = A.size(1), G = B.dim() == 4 ? B.size(2) : 1;
        const int dev = x.device().index();
        const Tensor gy = incoming(g[0], x, x.sizes());
        Tensor gx = rows_as(x, x.scalar_type()), gdt = rows_as(dt, x.scalar_type()), gz;
        if (z.defined()) gz = rows_as(z, x.scalar_type());
        Tensor gA = vector_for(A), gB, gC, gskip = vector_for(skip),
               gbias = vector_for(bias);
        for (Tensor* q : {&gB, &gC}) *q = x.numel() ? empty_as(B) : at::zeros(B.sizes(), B.options());
        const int64_t need = fwp_selective_scan_backward_scratch_floats(N, L, D, S, G, dev);
        const Tensor scratch = scratch_of(need, x);
        check(fwp_selective_scan_backward(N, L, D, S, G, RowsDesc(x), RowsDesc(dt), floats(A), GroupDesc(B), GroupDesc(C), floats(skip), RowsDesc(z),
                                          floats(bias), ints(lengths), floats(o[0]), RowsDesc(gy), RowsDesc(gx), RowsDesc(gdt), floats(gA),
                                          GroupDesc(gB), GroupDesc(gC), floats(gskip), RowsDesc(gz), floats(gbias), floats(scratch), need, softplus,
                                          dtype_code(x), stream_of(x), dev), "selective_scan_backward");
        return {gx, gdt, gA, gB, gC, gskip, gz, gbias, Tensor(), Tensor()};
    }
};

bool group_like(const Tensor& t, const Tensor& x, int64_t S) {
    return t.layout() == at::kStrided && t.scalar_type() == x.scalar_type() && t.device() == x.device() && (t.dim() == 3 || t.dim() == 4) &&
           t.size(0) == x.size(0) && t.size(1) == x.size(1) && t.size(-1) == S && (S == 1 || t.stride(-1) == 1) &&
           (t.dim() == 3 || (t.size(2) > 0 && x.size(2) % t.size(2) == 0));
}

// x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus
PyObject* selective_scan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    std::array<const Tensor*, 10> in;
    if (n != 11 || !optional_tensors(args, in)) return not_implemented();
    for (int i = 0; i < 5; i++)
        if (!in[i]) return not_implemented();
    const int softplus = flag(args[10]);
    if (softplus < 0) return nullptr;
    const Tensor &x = *in[0], &dt = *in[1], &A = *in[2], &B = *in[3], &C = *in[4];
    if (!first_rows(x) || x.dim() != 3 || A.dim() != 2) return not_implemented();
    const int64_t N = x.size(0), L = x.size(1), D = x.size(2), S = A.size(1);
    const auto dev = x.device();
    const auto ty = x.scalar_type();
    if (S < 1 || !rows_like(dt, ty, dev, x.sizes()) || (in[6] && !rows_like(*in[6], ty, dev, x.sizes())) || !group_like(B, x, S) || !group_like(C, x, S) ||
        B.sizes() != C.sizes() || !weight_like(&A, dev, {D, S}) || !weight_like(in[5], dev, {D}) || !weight_like(in[7], dev, {D}) ||
        !state_like(in[8], dev, {N, D, S}) || !lengths_like(in[9], dev, N))
        return not_implemented();
    const int64_t G = B.dim() == 4 ? B.size(2) : 1;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        const bool grad = any_needs_grad(in);
        out = rows_as(x, ty);
        Tensor keep;
        if (grad) keep = scratch_of(fwp_selective_scan_checkpoint_floats(N, L, D, S), x);
        const int64_t need = fwp_selective_scan_scratch_floats(N, L, D, S, G, dev.index());
        const Tensor scratch = scratch_of(need, x);
        check(fwp_selective_scan_forward(N, L, D, S, G, RowsDesc(x), RowsDesc(dt), floats(&A), GroupDesc(B), GroupDesc(C), floats(in[5]),
                                         RowsDesc(in[6]), floats(in[7]), RowsDesc(in[8]), ints(in[9]), RowsDesc(out), floats(keep),
                                         floats(scratch), need, softplus, dtype_code(x), stream_of(x), dev.index()), "selective_scan_forward");
        if (grad) {
            auto node = optional_node<ScanNode>(in, 8);
            node->softplus = softplus;
            node->keep({keep});
            torch::autograd::create_gradient_edge(out, node);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// --------------------------------------------------------------- norms between two blocks
struct NormNode final : public OpNode {
    double scale = 1;
    int rms = 0, act = 0;
    std::string name() const override { return "BlockNormBackward"; }
    variable_list apply(variable_list&& g) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const auto t = unpack(user), o = unpack(own);
        const Tensor &x = t[0], &w = t[1], &b = t[2], &res = t[3], &sv = t[4], &gate = t[5], &pw = t[6], &pb = t[7];
        const auto ty = x.scalar_type(), rty = res.defined() ? res.scalar_type() : ty;
        const int64_t N = x.dim() == 3 ? x.size(0) : 1, L = x.size(-2), D = x.size(-1);
        Tensor gy, gr;
        if (g[0].defined()) gy = incoming(g[0], x, x.sizes());
        if (g[1].defined()) gr = incoming(g[1], res.defined() ? res : x, x.sizes());
        // the residual's gradient is the sum's; with nothing but the sum in between the block's is the same tensor
        const bool same = res.defined() && ty == rty && !gate.defined() && !pw.defined() && !sv.defined() && scale == 1.;
        Tensor gx = rows_as(x, ty), gres, ggate;
        if (res.defined() && !same) gres = rows_as(res, rty);
        if (gate.defined()) ggate = rows_as(gate, ty);
        Tensor gw = vector_for(w), gb = vector_for(b), gpw = vector_for(pw), gpb = vector_for(pb), gs = vector_for(sv);
        const int64_t need = fwp_block_norm_backward_scratch_floats(N, L, D);
        const Tensor scratch = scratch_of(need, x);
        check(fwp_block_norm_backward(N, L, D, RowsDesc(x), RowsDesc(res), RowsDesc(gate), floats(sv), (float)scale, floats(pw), floats(pb), floats(w),
                                      floats(b), floats(o[0]), RowsDesc(gy), RowsDesc(gr), RowsDesc(gx), RowsDesc(gres), RowsDesc(ggate), floats(gs),
                                      floats(gpw), floats(gpb), floats(gw), floats(gb), floats(scratch), need, rms, act, dtype_code(x),
                                      rty == at::kFloat ? FWP_F32 : FWP_BF16, stream_of(x), x.device().index()), "block_norm_backward");
        return {gx, gw, gb, same ? gx : gres, gs, ggate, gpw, gpb};
    }
};

// x, weight, bias, residual, scale (a tensor, a number or None), gate, post_weight, post_bias, gate_act (0, 1, 2), eps, rms
PyObject* block_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11) return not_implemented();
    PyObject* a[8] = {args[0], args[1], args[2], args[3], args[4], args[5], args[6], args[7]};
    double scale = 1;
    if (PyFloat_Check(a[4]) || PyLong_Check(a[4])) {
        scale = PyFloat_AsDouble(a[4]);
        if (scale == -1. && PyErr_Occurred()) return nullptr;
        a[4] = Py_None;
    }
    std::array<const Tensor*, 8> in;
    if (!optional_tensors(a, in) || !in[0] || !in[1]) return not_implemented();
    const long act = PyLong_AsLong(args[8]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    const double eps = PyFloat_AsDouble(args[9]);
    if (eps == -1. && PyErr_Occurred()) return nullptr;
    const int rms = flag(args[10]);
    if (rms < 0) return nullptr;
    const Tensor& x = *in[0];
    if (!first_rows(x)) return not_implemented();
    const auto ty = x.scalar_type();
    const auto dev = x.device();
    const int64_t N = x.dim() == 3 ? x.size(0) : 1, L = x.size(-2), D = x.size(-1);
    const Tensor* res = in[3];
    if (res && !rows_like(*res, at::kFloat, dev, x.sizes()) && !rows_like(*res, ty, dev, x.sizes())) return not_implemented();
    if (in[5] && !rows_like(*in[5], ty, dev, x.sizes())) return not_implemented();
    for (int i : {1, 2, 4, 6, 7})
        if (!weight_like(in[i], dev, {D})) return not_implemented();
    if (in[7] && !in[6]) return not_implemented();
    const auto rty = res ? res->scalar_type() : ty;
    Tensor y, r;
    {
        pybind11::gil_scoped_release no_gil;
        const bool grad = any_needs_grad(in);
        y = rows_as(x, ty);
        r = rows_as(x, rty);
        Tensor stats;
        if (grad) stats = scratch_of(N * L * 4, x);
        check(fwp_block_norm_forward(N, L, D, RowsDesc(x), RowsDesc(res), RowsDesc(in[5]), floats(in[4]), (float)scale, floats(in[6]), floats(in[7]),
                                     floats(in[1]), floats(in[2]), RowsDesc(y), RowsDesc(r), floats(stats), (float)eps, rms, (int)act, dtype_code(x),
                                     rty == at::kFloat ? FWP_F32 : FWP_BF16, stream_of(x), dev.index()), "block_norm_forward");
        if (grad) {
            auto node = optional_node<NormNode>(in);
            node->scale = scale;
            node->rms = rms;
            node->act = (int)act;
            node->keep({stats});
            torch::autograd::create_gradient_edge(y, node);
            torch::autograd::create_gradient_edge(r, node);
        }
    }
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(y)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(r)));
    return pair;
    END_HANDLE_TH_ERRORS
}
