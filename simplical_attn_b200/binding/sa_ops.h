// Rotary positions and causal attention on torch tensors (included by sa_torch.cpp, inside its namespace): argument
// checks, output allocation, the C-ABI call and the autograd node, in the manner of the 2-simplicial operator there.

sa_dtype dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? SA_BF16 : t.scalar_type() == at::kHalf ? SA_F16 : SA_F32; }
// (b, n, h) strides of a [B, N, heads, D] tensor, or of a packed [T, heads, D] one
sa_strides row_strides(const Tensor& t) {
    if (!t.defined()) return sa_strides{0, 0, 0};
    return t.dim() == 4 ? sa_strides{t.stride(0), t.stride(1), t.stride(2)} : sa_strides{0, t.stride(0), t.stride(1)};
}
int32_t int32_of(int64_t v, const char* what) {
    TORCH_CHECK_VALUE(v >= 0 && v <= std::numeric_limits<int32_t>::max(), what, " does not fit 32 bits: ", v);
    return (int32_t)v;
}
void check_type_of(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "simplical_attn_b200 runs on CUDA tensors only; there is no CPU path");
    const auto st = t.scalar_type();
    TORCH_CHECK_TYPE(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, "unsupported dtype ", st);
}

// A second backward pass through `grads` raises: the kernels have no derivative of the gradient.
torch::autograd::variable_list no_second_derivative(torch::autograd::variable_list grads, const char* name) {
    for (Tensor& g : grads)
        if (g.defined()) g.requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", (int64_t)grads.size());
    return (*error)(std::move(grads));
}

// ---------------------------------------------------------------------------------------- rotary positions
struct RotaryConfig {
    int64_t offset;
    double magnitude;
    bool interleaved, inverse;
};
using Tensors = std::vector<Tensor>;
constexpr size_t kMaxRotary = 4;

// [first, last) element addresses that a tensor's elements lie in
std::pair<const char*, const char*> extent(const Tensor& t) {
    int64_t lo = 0, hi = 0;
    for (int64_t d = 0; d < t.dim(); ++d) (t.stride(d) < 0 ? lo : hi) += (t.size(d) - 1) * t.stride(d);
    const char* base = static_cast<const char*>(t.data_ptr());
    return {base + lo * t.element_size(), base + (hi + 1) * t.element_size()};
}
// Whether two tensors certainly share no element: apart in memory, or different heads of equally laid out rows (views cut out
// of one projection's output).
bool disjoint(const Tensor& x, const Tensor& y) {
    const auto ex = extent(x), ey = extent(y);
    if (ex.second <= ey.first || ey.second <= ex.first) return true;
    const sa_strides sx = row_strides(x), sy = row_strides(y);
    if (sx.b != sy.b || sx.n != sy.n || sx.n <= 0 || sx.h < 0 || sy.h < 0) return false;
    if (x.dim() == 4 && x.size(0) > 1 && sx.b < x.size(1) * sx.n) return false;
    const int64_t es = x.element_size();
    const char *px = static_cast<const char*>(x.data_ptr()), *py = static_cast<const char*>(y.data_ptr());
    const bool x_first = px < py;
    const Tensor &a = x_first ? x : y, &b = x_first ? y : x;
    const int64_t gap = (x_first ? py - px : px - py);
    auto row = [&](const Tensor& t) { return ((t.size(-2) - 1) * t.stride(-2) + t.size(-1)) * es; };
    return row(a) <= gap && gap + row(b) <= sx.n * es;
}

void check_rotary(const Tensors& xs, const Tensors& outs, const Tensor& frequencies, const Tensor& positions) {
    TORCH_CHECK_VALUE(xs.size() >= 1 && xs.size() <= kMaxRotary, "rotary_positions takes one to four tensors, got ", xs.size());
    const Tensor& x = xs[0];
    check_type_of(x);
    for (const Tensor& t : xs) {
        TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() && t.device() == x.device(), "the tensors must share dtype and device");
        TORCH_CHECK_VALUE(t.dim() == 4 || t.dim() == 3, "tensors must be [batch, seq_len, heads, head_dim] or packed [rows, heads, head_dim], got ", t.sizes());
        TORCH_CHECK_VALUE(t.dim() == x.dim() && t.size(0) == x.size(0) && (t.dim() == 3 || t.size(1) == x.size(1)) && t.size(-1) == x.size(-1),
                          "the tensors must share every extent but the heads, got ", x.sizes(), " and ", t.sizes());
    }
    TORCH_CHECK_TYPE(frequencies.device() == x.device() && (frequencies.scalar_type() == at::kDouble || frequencies.scalar_type() == at::kFloat),
                     "frequencies must be float32 or float64 on the tensors' device");
    TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.size(0) >= 1 && 2 * frequencies.size(0) <= x.size(-1),
                      "frequencies must be [rotary_dim / 2] with 2 <= rotary_dim <= head_dim, got ", frequencies.sizes());
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && frequencies.requires_grad()), "there is no gradient for the frequencies");
    if (positions.defined()) {
        TORCH_CHECK_TYPE(positions.device() == x.device() && (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
                         "positions must be int32 or int64 on the tensors' device");
        const int64_t n = x.size(x.dim() - 3);
        TORCH_CHECK_VALUE((positions.dim() == 1 && positions.size(0) == n) ||
                              (x.dim() == 4 && positions.dim() == 2 && positions.size(0) == x.size(0) && positions.size(1) == n),
                          "positions must be one per row, or [batch, seq_len], got ", positions.sizes(), " for ", x.sizes());
    }
    if (outs.empty()) return;
    TORCH_CHECK_VALUE(outs.size() == xs.size(), "as many outputs as tensors, got ", outs.size(), " for ", xs.size());
    for (size_t i = 0; i < xs.size(); ++i) {
        const Tensor& o = outs[i];
        TORCH_CHECK_TYPE(o.scalar_type() == x.scalar_type() && o.device() == x.device(), "an output must match its tensor's dtype and device");
        TORCH_CHECK_VALUE(o.sizes() == xs[i].sizes(), "an output must have its tensor's shape, got ", o.sizes(), " for ", xs[i].sizes());
        TORCH_CHECK_VALUE(o.stride(-1) == 1 || o.size(-1) == 1, "an output's innermost stride must be 1");
        if (o.numel() == 0) continue;
        for (int64_t d = 0; d < o.dim(); ++d) TORCH_CHECK_VALUE(o.size(d) == 1 || o.stride(d) != 0, "an output's elements must not share memory");
        for (size_t j = 0; j < xs.size(); ++j) {
            const bool same = i == j && o.data_ptr() == xs[i].data_ptr() && o.strides() == xs[i].strides();
            TORCH_CHECK_VALUE(same || disjoint(o, xs[j]), "output ", i, " may overlap tensor ", j, "; in place an output is its own tensor");
            TORCH_CHECK_VALUE(i == j || disjoint(o, outs[j]), "outputs ", i, " and ", j, " may overlap");
        }
    }
}

// `outs` empty: new tensors.
Tensors rotary_call(const Tensors& xs_, Tensors outs, const Tensor& frequencies_, const Tensor& positions, const RotaryConfig& c) {
    check_rotary(xs_, outs, frequencies_, positions);
    const Tensor frequencies = frequencies_.contiguous();
    const c10::cuda::CUDAGuard guard(xs_[0].device());
    Tensors xs;
    for (const Tensor& t : xs_) xs.push_back(unit_inner(t));
    if (outs.empty())
        for (const Tensor& t : xs) outs.push_back(at::empty_like(t));
    sa_rotary_params p{};
    const Tensor& x = xs[0];
    const void* in[kMaxRotary];
    void* out[kMaxRotary];
    for (size_t i = 0; i < xs.size(); ++i) {
        if (xs[i].size(-2) == 0) continue;                 // no heads: nothing to turn
        const int k = p.tensors++;
        p.heads[k] = int32_of(xs[i].size(-2), "the number of heads");
        p.in[k] = row_strides(xs[i]);
        p.out[k] = row_strides(outs[i]);
        in[k] = xs[i].data_ptr();
        out[k] = outs[i].data_ptr();
    }
    if (p.tensors == 0 || x.size(0) == 0 || x.size(x.dim() - 3) == 0) return outs;
    p.B = x.dim() == 4 ? int32_of(x.size(0), "the batch") : 1;
    p.N = int32_of(x.size(x.dim() - 3), "the sequence length");
    p.D = int32_of(x.size(-1), "head_dim");
    p.rotary_dim = (int32_t)(2 * frequencies.size(0));
    p.interleaved = c.interleaved;
    p.inverse = c.inverse;
    p.dtype = dtype_of(x);
    p.frequency_bits = frequencies.scalar_type() == at::kDouble ? 64 : 32;
    p.offset = c.offset;
    p.magnitude = (float)c.magnitude;
    if (positions.defined()) {
        p.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
        p.position_b = positions.dim() == 2 ? positions.stride(0) : 0;
        p.position_n = positions.stride(-1);
    }
    const int rc = sa_rotary(&p, in, out, positions.defined() ? positions.data_ptr() : nullptr, frequencies.data_ptr(),
                             at::cuda::getCurrentCUDAStream(x.device().index()).stream());
    if (rc != SA_OK) raise_status("sa_rotary", rc);
    return outs;
}

Tensors rotary(const Tensors& xs, const Tensor& frequencies, const Tensor& positions, const RotaryConfig& c);

struct RotaryBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable frequencies, positions;
    RotaryConfig cfg;
    size_t n = 0;

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list out(n);
        Tensors in;
        for (size_t i = 0; i < n; ++i)
            if (grads[i].defined() && task_should_compute_output(i)) in.push_back(grads[i]);
        if (in.empty()) return out;
        RotaryConfig back = cfg;
        back.inverse = !back.inverse;
        Tensors g = rotary(in, frequencies.unpack(), positions.unpack(), back);      // (with a history of its own under create_graph)
        for (size_t i = 0, k = 0; i < n; ++i)
            if (grads[i].defined() && task_should_compute_output(i)) out[i] = std::move(g[k++]);
        return out;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        frequencies.reset_data();
        positions.reset_data();
    }
    std::string name() const override { return "RotaryPositionsBackward"; }
};

Tensors rotary(const Tensors& xs, const Tensor& frequencies, const Tensor& positions, const RotaryConfig& c) {
    std::shared_ptr<RotaryBackward> node;
    bool any = false;
    for (const Tensor& t : xs) any |= t.requires_grad();
    if (any && at::GradMode::is_enabled()) {
        node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
        torch::autograd::edge_list edges;
        for (const Tensor& t : xs) edges.push_back(torch::autograd::impl::gradient_edge(t));
        node->set_next_edges(std::move(edges));
        node->cfg = c;
        node->n = xs.size();
        node->frequencies = torch::autograd::SavedVariable(frequencies, false);
        node->positions = torch::autograd::SavedVariable(positions, false);
    }
    Tensors r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = rotary_call(xs, {}, frequencies, positions, c);
    }
    if (node)
        for (Tensor& t : r) torch::autograd::set_history(t, node);
    return r;
}

// ---------------------------------------------------------------------------------------- causal attention
struct CausalConfig {
    double scale;
    int64_t max_q, max_k;
    int algo;
};

void check_causal(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k) {
    check_type_of(q);
    const bool packed = cu_q.defined();
    TORCH_CHECK_VALUE(packed ? q.dim() == 3 : q.dim() == 4, packed ? "q must be packed [rows, num_heads, head_dim] with cu_q"
                                                                   : "q must be [batch, seq_len, num_heads, head_dim] (packed tensors need cu_q)",
                      ", got ", q.sizes());
    const int64_t H = q.size(-2), D = q.size(-1);
    const Tensor* const kv[2] = {&k, &v};
    static const char* const names[2] = {"k", "v"};
    for (int i = 0; i < 2; ++i) {
        const Tensor& t = *kv[i];
        TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type() && t.device() == q.device(), names[i], " must match q's dtype and device");
        TORCH_CHECK_VALUE(t.dim() == q.dim() && t.sizes() == k.sizes() && t.size(-1) == D && (packed || t.size(0) == q.size(0)), names[i], " must be ",
                          packed ? "[rows, kv_heads, head_dim]" : "[batch, key_len, kv_heads, head_dim]", " like the other of the two, got ", t.sizes());
    }
    TORCH_CHECK_VALUE(k.size(-2) > 0 && H > 0 && H % k.size(-2) == 0, "K and V must have a head count that divides the query head count");
    TORCH_CHECK_VALUE(D > 0, "head_dim must be positive");
    if (!packed) {
        TORCH_CHECK_VALUE(!cu_k.defined(), "cu_k without cu_q");
        return;
    }
    const Tensor* const cu[2] = {&cu_q, &cu_k};
    static const char* const cu_names[2] = {"cu_q", "cu_k"};
    for (int i = 0; i < 2; ++i) {
        TORCH_CHECK_TYPE(cu[i]->scalar_type() == at::kInt && cu[i]->device() == q.device(), cu_names[i], " must be int32 on q's device");
        TORCH_CHECK_VALUE(cu[i]->dim() == 1 && cu[i]->size(0) >= 2 && cu[i]->size(0) == cu_q.size(0) && cu[i]->is_contiguous(), cu_names[i],
                          " must be contiguous [sequences + 1] with at least one sequence, as many as cu_q has, got ", cu[i]->sizes());
    }
}

sa_causal_params causal_params(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& cu_q, const CausalConfig& c) {
    sa_causal_params p{};
    const bool packed = cu_q.defined();
    p.B = packed ? 1 : int32_of(q.size(0), "the batch");
    p.Nq = int32_of(q.size(packed ? 0 : 1), "the number of queries");
    p.Nk = int32_of(k.size(packed ? 0 : 1), "the number of keys");
    p.H = int32_of(q.size(-2), "the number of heads");
    p.Hkv = int32_of(k.size(-2), "the number of KV heads");
    p.D = int32_of(q.size(-1), "head_dim");
    p.sequences = packed ? int32_of(cu_q.size(0) - 1, "the number of sequences") : 0;
    p.max_q = int32_of(c.max_q, "max_q");
    p.max_k = int32_of(c.max_k, "max_k");
    p.dtype = dtype_of(q);
    p.algo = c.algo;
    p.scale = (float)c.scale;
    p.q = row_strides(q); p.k = row_strides(k); p.v = row_strides(v); p.o = row_strides(o);
    return p;
}

// A workspace from torch's allocator (the status word is elsewhere).
struct Scratch {
    Tensor t;
    void* ptr = nullptr;
    size_t bytes = 0;
    Scratch(size_t need, const Tensor& like) {
        if (need == 0) return;
        t = at::empty({(int64_t)need}, like.options().dtype(at::kByte));
        ptr = t.data_ptr();
        bytes = need;
    }
};
const int32_t* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

// O, LSE, and with `low` what rounding took from a 16-bit O (else, and for fp32, undefined).
std::array<Tensor, 3> causal_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu_q, const Tensor& cu_k, const CausalConfig& c,
                                     bool low) {
    check_causal(q_, k_, v_, cu_q, cu_k);
    const c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = unit_inner(q_), k = unit_inner(k_), v = unit_inner(v_);
    const int device = q.device().index();
    poll_device(device);
    Tensor o = at::empty_like(q);
    Tensor lse = q.dim() == 4 ? at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat))
                              : at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    if (q.numel() == 0 || k.numel() == 0) {                // no query, or none that sees a key
        o.zero_();
        lse.fill_(-std::numeric_limits<float>::infinity());
        return {std::move(o), std::move(lse), Tensor()};
    }
    Tensor o_low;
    if (low && q.scalar_type() != at::kFloat) o_low = at::empty_like(o);
    const sa_causal_params p = causal_params(q, k, v, o, cu_q, c);
    const Scratch ws(sa_causal_forward_workspace_size(&p), q);
    const int rc = sa_causal_forward(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), o_low.defined() ? o_low.data_ptr() : nullptr,
                                     (float*)lse.data_ptr(), ints(cu_q), ints(cu_k), ws.ptr, ws.bytes, status_word(device, kCausalForward), at::cuda::getCurrentCUDAStream(device).stream());
    if (rc != SA_OK) raise_status("sa_causal_forward", rc);
    return {std::move(o), std::move(lse), std::move(o_low)};
}

std::array<Tensor, 3> causal_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o_, const Tensor& o_low, const Tensor& lse,
                                      const Tensor& d_o_, const Tensor& cu_q, const Tensor& cu_k, const CausalConfig& c, const std::array<bool, 3>& need) {
    check_causal(q_, k_, v_, cu_q, cu_k);
    TORCH_CHECK_TYPE(d_o_.scalar_type() == q_.scalar_type() && d_o_.device() == q_.device() && o_.scalar_type() == q_.scalar_type() && o_.device() == q_.device(),
                     "o and its gradient must match q's dtype and device");
    TORCH_CHECK_VALUE(d_o_.sizes() == q_.sizes() && o_.sizes() == q_.sizes(), "o and its gradient must have q's shape");
    TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.device() == q_.device() && lse.is_contiguous() &&
                          lse.numel() == (q_.size(-1) == 0 ? 0 : q_.numel() / q_.size(-1)),
                      "lse must be the forward's");
    const c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = unit_inner(q_), k = unit_inner(k_), v = unit_inner(v_), o = unit_inner(o_), d_o = unit_inner(d_o_);
    TORCH_CHECK_VALUE(!o_low.defined() || (o_low.sizes() == o.sizes() && o_low.strides() == o.strides() && o_low.scalar_type() == o.scalar_type() &&
                                           o_low.device() == o.device()),
                      "o_low must be the forward's");
    const int device = q.device().index();
    poll_device(device);
    const Tensor* const in[3] = {&q, &k, &v};
    std::array<Tensor, 3> g;
    void* gp[3];
    const bool none = q.numel() == 0 || k.numel() == 0;
    for (int i = 0; i < 3; ++i) {
        if (need[i]) g[i] = none ? at::zeros_like(*in[i]) : at::empty_like(*in[i]);
        gp[i] = need[i] ? g[i].data_ptr() : nullptr;
    }
    if (none) return g;
    sa_causal_params p = causal_params(q, k, v, o, cu_q, c);
    p.d_o = row_strides(d_o);
    p.dq = row_strides(g[0]); p.dk = row_strides(g[1]); p.dv = row_strides(g[2]);
    const Scratch ws(sa_causal_backward_workspace_size(&p), q);
    const int rc = sa_causal_backward(&p, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), o_low.defined() ? o_low.data_ptr() : nullptr,
                                      (const float*)lse.data_ptr(), d_o.data_ptr(), gp[0], gp[1], gp[2], ints(cu_q), ints(cu_k), ws.ptr, ws.bytes, status_word(device, kCausalBackward),
                                      at::cuda::getCurrentCUDAStream(device).stream());
    if (rc != SA_OK) raise_status("sa_causal_backward", rc);
    return g;
}

struct CausalBackward : public torch::autograd::Node {
    torch::autograd::SavedVariable q, k, v, o, o_low, lse, cu_q, cu_k;
    CausalConfig cfg;

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        torch::autograd::variable_list out(3);
        if (!grads[0].defined()) return out;
        std::array<bool, 3> need;
        bool any = false;
        for (int i = 0; i < 3; ++i) any |= need[i] = task_should_compute_output(i);
        if (!any) return out;
        const auto self = getptr();
        const Tensor q_ = q.unpack(), k_ = k.unpack(), v_ = v.unpack(), o_ = o.unpack(self), low_ = o_low.unpack(), lse_ = lse.unpack(), cq = cu_q.unpack(), ck = cu_k.unpack();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            std::array<Tensor, 3> g = causal_backward(q_, k_, v_, o_, low_, lse_, grads[0], cq, ck, cfg, need);
            for (int i = 0; i < 3; ++i) out[i] = std::move(g[i]);
        }
        return at::GradMode::is_enabled() ? no_second_derivative(std::move(out), "causal_attention") : out;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto* x : {&q, &k, &v, &o, &o_low, &lse, &cu_q, &cu_k}) x->reset_data();
    }
    std::string name() const override { return "CausalAttentionBackward"; }
};

std::pair<Tensor, Tensor> causal_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k, const CausalConfig& c) {
    std::shared_ptr<CausalBackward> node;
    if (torch::autograd::compute_requires_grad(q, k, v)) {
        node = std::shared_ptr<CausalBackward>(new CausalBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
        node->cfg = c;
        node->q = torch::autograd::SavedVariable(q, false);
        node->k = torch::autograd::SavedVariable(k, false);
        node->v = torch::autograd::SavedVariable(v, false);
        node->cu_q = torch::autograd::SavedVariable(cu_q, false);
        node->cu_k = torch::autograd::SavedVariable(cu_k, false);
    }
    std::array<Tensor, 3> r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = causal_forward(q, k, v, cu_q, cu_k, c, node != nullptr);
    }
    if (node) {
        torch::autograd::set_history(r[0], node);
        node->o = torch::autograd::SavedVariable(r[0], true);
        node->lse = torch::autograd::SavedVariable(r[1], false);
        node->o_low = torch::autograd::SavedVariable(r[2], false);
    }
    return {std::move(r[0]), std::move(r[1])};
}

// ---------------------------------------------------------------------------------------- Python entry points
Tensor optional_tensor(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }
Tensors tensors_arg(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(PyTuple_Check(o), name, " must be a tuple of tensors");
    Tensors r;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) r.push_back(tensor_arg(PyTuple_GET_ITEM(o, i), name));
    return r;
}
// Whether plain() holds for the tensors of a tuple, and whatever else is a tensor is one itself.
bool plain_tuple(PyObject* t) {
    if (!PyTuple_Check(t)) return false;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(t); ++i)
        if (!plain(&PyTuple_GET_ITEM(t, i), 1)) return false;
    return true;
}
bool plain_or_none(PyObject* o) { return o == Py_None || plain(&o, 1); }
PyObject* wrap_tuple(Tensors&& ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    for (size_t i = 0; i < ts.size(); ++i) {
        if (ts[i].defined()) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(std::move(ts[i])));
        else PyTuple_SET_ITEM(r, (Py_ssize_t)i, Py_NewRef(Py_None));
    }
    return r;
}

// tensors, outputs or None, frequencies, positions or None, offset, interleaved, magnitude, inverse
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 8);
    if (!plain_tuple(a[0]) || (a[1] != Py_None && !plain_tuple(a[1])) || !plain(a + 2, 1) || !plain_or_none(a[3])) Py_RETURN_NONE;
    const Tensors xs = tensors_arg(a[0], "tensors"), outs = a[1] == Py_None ? Tensors{} : tensors_arg(a[1], "out");
    const Tensor frequencies = tensor_arg(a[2], "frequencies"), positions = optional_tensor(a[3], "positions");
    const RotaryConfig c{int_arg(a[4]), float_arg(a[6]), int_arg(a[5]) != 0, int_arg(a[7]) != 0};
    Tensors r;
    {
        pybind11::gil_scoped_release no_gil;
        if (a[1] == Py_None) r = rotary(xs, frequencies, positions, c);
        else {
            if (at::GradMode::is_enabled())
                for (const Tensors* ts : {&xs, &outs})
                    for (const Tensor& t : *ts) TORCH_CHECK(!t.requires_grad(), "rotary_positions with out= records no gradient: call it under no_grad, or without out=");
            {
                at::AutoDispatchBelowADInplaceOrView below;
                r = rotary_call(xs, outs, frequencies, positions, c);
            }
            for (const Tensor& t : outs) torch::autograd::impl::bump_version(t);
        }
    }
    return wrap_tuple(std::move(r));
    END_HANDLE_TH_ERRORS
}

// q, k, v, cu_q or None, cu_k or None, scale, max_q, max_k, algo
CausalConfig causal_config(PyObject* const* a) { return CausalConfig{float_arg(a[0]), int_arg(a[1]), int_arg(a[2]), (int)int_arg(a[3])}; }

PyObject* py_causal(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    if (!plain(a, 3) || !plain_or_none(a[3]) || !plain_or_none(a[4])) Py_RETURN_NONE;
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v");
    const Tensor cu_q = optional_tensor(a[3], "cu_q"), cu_k = optional_tensor(a[4], "cu_k");
    const CausalConfig c = causal_config(a + 5);
    std::pair<Tensor, Tensor> r;
    {
        pybind11::gil_scoped_release no_gil;
        r = causal_attention(q, k, v, cu_q, cu_k, c);
    }
    return wrap_tuple({std::move(r.first), std::move(r.second)});
    END_HANDLE_TH_ERRORS
}

// the same and whether O's low part is wanted; without a history
PyObject* py_causal_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    if (!exact(a, 3)) Py_RETURN_NONE;
    const Tensor &q = tensor_arg(a[0], "q"), &k = tensor_arg(a[1], "k"), &v = tensor_arg(a[2], "v");
    const Tensor cu_q = optional_tensor(a[3], "cu_q"), cu_k = optional_tensor(a[4], "cu_k");
    const CausalConfig c = causal_config(a + 5);
    const bool low = int_arg(a[9]) != 0;
    std::array<Tensor, 3> r;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        r = causal_forward(q, k, v, cu_q, cu_k, c, low);
    }
    return wrap_tuple({std::move(r[0]), std::move(r[1]), std::move(r[2])});
    END_HANDLE_TH_ERRORS
}

// q, k, v, o, lse, d_o, o_low or None, cu_q or None, cu_k or None, scale, max_q, max_k, algo, need (bit i: gradient i)
PyObject* py_causal_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 14);
    if (!exact(a, 6)) Py_RETURN_NONE;
    static const char* const names[6] = {"q", "k", "v", "o", "lse", "d_o"};
    const Tensor* t[6];
    for (int i = 0; i < 6; ++i) t[i] = &tensor_arg(a[i], names[i]);
    const Tensor o_low = optional_tensor(a[6], "o_low"), cu_q = optional_tensor(a[7], "cu_q"), cu_k = optional_tensor(a[8], "cu_k");
    const CausalConfig c = causal_config(a + 9);
    const int64_t bits = int_arg(a[13]);
    const std::array<bool, 3> need{(bits & 1) != 0, (bits & 2) != 0, (bits & 4) != 0};
    std::array<Tensor, 3> g;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        g = causal_backward(*t[0], *t[1], *t[2], *t[3], o_low, *t[4], *t[5], cu_q, cu_k, c, need);
    }
    return wrap_tuple({std::move(g[0]), std::move(g[1]), std::move(g[2])});
    END_HANDLE_TH_ERRORS
}
