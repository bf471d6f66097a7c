// Native host path of the selective state space mixer and the norms round a block (part of binding.cpp, whose helpers it
// uses): the ordinary case in one call from Python, NotImplemented for the rest, which ssm.py and layer_ops.py serve.
#pragma once

namespace {

struct SsmAbi {
    decltype(&hdla_short_conv_fwd) conv_fwd;
    decltype(&hdla_short_conv_bwd_workspace_bytes) conv_bwd_bytes;
    decltype(&hdla_short_conv_bwd) conv_bwd;
    decltype(&hdla_short_conv_step) conv_step;
    decltype(&hdla_selective_scan_checkpoint_bytes) scan_checkpoint_bytes;
    decltype(&hdla_selective_scan_workspace_bytes) scan_bytes;
    decltype(&hdla_selective_scan_fwd) scan_fwd;
    decltype(&hdla_selective_scan_bwd) scan_bwd;
    decltype(&hdla_selective_scan_step) scan_step;
    decltype(&hdla_norm_residual_fwd) norm_fwd;
    decltype(&hdla_norm_residual_bwd_workspace_bytes) norm_bwd_bytes;
    decltype(&hdla_norm_residual_bwd) norm_bwd;
} ssm{};

void bind_ssm(void* h) {
    look_up(h, "hdla_short_conv_fwd", ssm.conv_fwd);
    look_up(h, "hdla_short_conv_bwd_workspace_bytes", ssm.conv_bwd_bytes);
    look_up(h, "hdla_short_conv_bwd", ssm.conv_bwd);
    look_up(h, "hdla_short_conv_step", ssm.conv_step);
    look_up(h, "hdla_selective_scan_checkpoint_bytes", ssm.scan_checkpoint_bytes);
    look_up(h, "hdla_selective_scan_workspace_bytes", ssm.scan_bytes);
    look_up(h, "hdla_selective_scan_fwd", ssm.scan_fwd);
    look_up(h, "hdla_selective_scan_bwd", ssm.scan_bwd);
    look_up(h, "hdla_selective_scan_step", ssm.scan_step);
    look_up(h, "hdla_norm_residual_fwd", ssm.norm_fwd);
    look_up(h, "hdla_norm_residual_bwd_workspace_bytes", ssm.norm_bwd_bytes);
    look_up(h, "hdla_norm_residual_bwd", ssm.norm_bwd);
}

const float* read(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
// Rows may lie anywhere as long as a row's last dimension is dense: slices of a wider projection are read where they are.
Tensor rows_of(const Tensor& t) { return !t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
// the stride of dimension d; one that is never stepped over may hold anything
int64_t step_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
Tensor space(size_t bytes, const Tensor& like) {
    return bytes ? dense({static_cast<int64_t>(bytes)}, at::kByte, like.device()) : Tensor();
}
Tensor as_type(const Tensor& t, at::ScalarType st) { return t.defined() && t.scalar_type() != st ? t.to(st) : t; }
// The type that weights used together have in a kernel: the widest among them (all products and sums are fp32 either way).
at::ScalarType weights_type(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->scalar_type() != at::kBFloat16) return at::kFloat;
    return at::kBFloat16;
}
Tensor grad_in(const Tensor& g, at::ScalarType st) { return g.defined() ? g.to(st).contiguous() : g; }
bool is_float(const Tensor& t) { return !t.defined() || t.is_floating_point(); }
bool shape3(const Tensor& t, int64_t a, int64_t b, int64_t c) { return t.dim() == 3 && t.size(0) == a && t.size(1) == b && t.size(2) == c; }
bool vector_of(const Tensor& t, int64_t n) { return !t.defined() || (t.dim() == 1 && t.size(0) == n && t.is_floating_point()); }
bool offsets_tensor(const Tensor& cu, int64_t B) {
    return !cu.defined() || (B == 1 && cu.dim() == 1 && cu.size(0) >= 2 && cu.size(0) <= 0x7fffffff && cu.scalar_type() == at::kLong && cu.is_contiguous());
}
int64_t sequences(const Tensor& cu, int64_t B) { return cu.defined() ? cu.size(0) - 1 : B; }
// A saved tensor as it was, strides included (Saved::get would make it contiguous); one that was changed since is an error.
Tensor unpack_saved(const Saved& s, const char* node) {
    const Tensor t = s.var.unpack();
    if (!s.defined) return t;
    if (!t.defined() || t.device() != s.device || t.scalar_type() != s.type || t.sizes() != at::IntArrayRef(s.size) || t.layout() != at::kStrided)
        throw std::runtime_error(std::string(node) + ": a saved-tensor hook returned a tensor of another shape, type or device "
                                 "than the saved one's");
    return rows_of(t);
}

// ------------------------------------------------------------------------------------------ short convolution
struct ConvIn { Tensor x, w, b, h0, cu; bool silu = false; };      // (w and b of one type)

HdlaConvArgs conv_args(const ConvIn& i) {
    HdlaConvArgs a{};
    a.B = (int)i.x.size(0); a.T = (int)i.x.size(1); a.D = (int)i.x.size(2); a.W = (int)i.w.size(1);
    a.dtype = dtype_code(i.x); a.w_dtype = dtype_code(i.w); a.activation = i.silu ? HDLA_ACT_SILU : HDLA_ACT_NONE;
    a.n_seqs = i.cu.defined() ? (int)i.cu.size(0) - 1 : 0;
    a.cu_seqlens = static_cast<const int64_t*>(ptr(i.cu));
    a.x_batch = step_of(i.x, 0); a.x_token = step_of(i.x, 1);
    a.x = ptr(i.x); a.weight = ptr(i.w); a.bias = ptr(i.b); a.h0 = ptr(i.h0);
    return a;
}
std::pair<Tensor, Tensor> conv_forward(const ConvIn& i, bool want_ht) {
    HdlaConvArgs a = conv_args(i);
    const Tensor y = dense(i.x.sizes(), i.x.scalar_type(), i.x.device());
    Tensor ht;
    if (want_ht) ht = dense({sequences(i.cu, a.B), a.W - 1, a.D}, i.x.scalar_type(), i.x.device());
    a.y = mptr(y); a.ht = mptr(ht);
    check(ssm.conv_fwd(&a, stream_of(i.x)), "hdla_short_conv_fwd");
    return {y, ht};
}
struct ConvGrads { Tensor dx, dw, db, dh0; };
ConvGrads conv_backward(const ConvIn& i, const Tensor& dy_, const Tensor& dht_) {
    c10::cuda::CUDAGuard guard(i.x.device());
    HdlaConvArgs a = conv_args(i);
    const Tensor dy = grad_in(dy_, i.x.scalar_type()), dht = grad_in(dht_, i.x.scalar_type());
    ConvGrads g;
    g.dx = dense(i.x.sizes(), i.x.scalar_type(), i.x.device());
    g.dw = dense_like(i.w);
    if (i.b.defined()) g.db = dense_like(i.b);
    if (i.h0.defined()) g.dh0 = dense_like(i.h0);
    const size_t n = ssm.conv_bwd_bytes(&a);
    const Tensor ws = space(n, i.x);
    a.dy = ptr(dy); a.dht = ptr(dht);
    a.dx = mptr(g.dx); a.dh0 = mptr(g.dh0); a.dweight = mptr(g.dw); a.dbias = mptr(g.db);
    check(ssm.conv_bwd(&a, mptr(ws), n, stream_of(i.x)), "hdla_short_conv_bwd");
    return g;
}

struct ConvNode : torch::autograd::Node {
    Saved x, w, b, h0, cu;
    bool silu = false;
    at::ScalarType w_type = at::kFloat, b_type = at::kFloat;
    std::string name() const override { return "HdlaShortConvBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved* s : {&x, &w, &b, &h0, &cu}) s->var.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const Tensor dht = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !dht.defined()) return variable_list(4);
        const char* me = "HdlaShortConvBackward";
        ConvGrads g = conv_backward({unpack_saved(x, me), w.get(me), b.get(me), h0.get(me), cu.get(me), silu}, grads[0], dht);
        return {g.dx, as_type(g.dw, w_type), as_type(g.db, b_type), g.dh0};
    }
};

ConvIn conv_in(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& h0, const Tensor& cu, bool silu) {
    const auto type = weights_type({&w, &b});
    return {rows_of(x), as_type(w, type).contiguous(), b.defined() ? as_type(b, type).contiguous() : b, h0.defined() ? h0.contiguous() : h0, cu, silu};
}

std::pair<Tensor, Tensor> conv_op(const Tensor& x_, const Tensor& w_, const Tensor& b_, const Tensor& h0_, const Tensor& cu, bool silu, bool want_ht) {
    const bool grad = needs_grad({&x_, &w_, &b_, &h0_});
    std::pair<Tensor, Tensor> r;
    std::shared_ptr<ConvNode> node;
    {
        at::NoGradGuard no_grad;
        c10::cuda::CUDAGuard guard(x_.device());
        const ConvIn i = conv_in(x_, w_, b_, h0_, cu, silu);
        r = conv_forward(i, want_ht);
        if (grad) {
            node = make_node<ConvNode>();
            node->x.save(i.x); node->w.save(i.w); node->b.save(i.b); node->h0.save(i.h0); node->cu.save(i.cu);
            node->silu = silu;
            node->w_type = w_.scalar_type();
            if (b_.defined()) node->b_type = b_.scalar_type();
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(x_, w_, b_, h0_));
        torch::autograd::create_gradient_edge(r.first, node);
        if (r.second.defined()) torch::autograd::create_gradient_edge(r.second, node);
    }
    return r;
}

// (x [B,T,D], weight [D,W], bias or None, silu, h0 or None, cu_seqlens or None) at av; false: not the ordinary case
struct ConvCall { const Tensor *x, *w, *b, *h0, *cu; bool silu; };
bool conv_call(PyObject* const* av, ConvCall& c) {
    c.x = arg(av[0]); c.w = arg(av[1]); c.b = arg(av[2], true); c.h0 = arg(av[4], true); c.cu = arg(av[5], true);
    if (!ssm.conv_fwd || !c.x || !c.w || !c.b || !c.h0 || !c.cu || transforms_active()) return false;
    const int silu = PyObject_IsTrue(av[3]);
    if (silu < 0) { PyErr_Clear(); return false; }
    c.silu = silu;
    const Tensor& x = *c.x;
    if (x.dim() != 3 || c.w->dim() != 2 || dtype_code(x) < 0 || dtype_code(*c.w) < 0) return false;
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), W = c.w->size(1);
    if (!fits_int({B, T, D, W}) || W > 8 || T > (1 << 30) || c.w->size(0) != D || !vector_of(*c.b, D) || !offsets_tensor(*c.cu, B)) return false;
    if (c.h0->defined() && !(shape3(*c.h0, sequences(*c.cu, B), W - 1, D) && c.h0->scalar_type() == x.scalar_type())) return false;
    return same_device(x, {c.w, c.b, c.h0, c.cu});
}

// short_conv(x, weight, bias or None, silu, h0 or None, cu_seqlens or None, output_final_state, bare) -> (y, final state or None);
// bare: without a graph, which the Python autograd function makes
PyObject* py_short_conv(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "short_conv takes 8 arguments"); return nullptr; }
    ConvCall c;
    const bool bare = av[7] == Py_True;
    const int want = PyObject_IsTrue(av[6]);
    if (want < 0) { PyErr_Clear(); NOT_MINE(); }
    if ((!bare && tracing()) || !conv_call(av, c)) NOT_MINE();
    std::pair<Tensor, Tensor> r;
    if (!guarded([&] {
            if (bare) {
                at::NoGradGuard no_grad;
                c10::cuda::CUDAGuard guard(c.x->device());
                r = conv_forward(conv_in(*c.x, *c.w, *c.b, *c.h0, *c.cu, c.silu), want);
            } else {
                r = conv_op(*c.x, *c.w, *c.b, *c.h0, *c.cu, c.silu, want);
            }
        }))
        return nullptr;
    return tuple_of({&r.first, &r.second});
}
// short_conv_backward(x, weight, bias, silu, h0, cu_seqlens, dy or None, dht or None) -> (dx, dweight, dbias, dh0)
PyObject* py_short_conv_backward(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "short_conv_backward takes 8 arguments"); return nullptr; }
    ConvCall c;
    const Tensor *dy = arg(av[6], true), *dht = arg(av[7], true);
    if (!conv_call(av, c) || !dy || !dht) {
        PyErr_SetString(PyExc_TypeError, "short_conv_backward: arguments of another kind than the forward call's");
        return nullptr;
    }
    ConvGrads g;
    if (!guarded([&] {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(c.x->device());
            g = conv_backward(conv_in(*c.x, *c.w, *c.b, *c.h0, *c.cu, c.silu), *dy, *dht);
            g.dw = as_type(g.dw, c.w->scalar_type());
            if (g.db.defined()) g.db = as_type(g.db, c.b->scalar_type());
        }))
        return nullptr;
    return tuple_of({&g.dx, &g.dw, &g.db, &g.dh0});
}
// short_conv_step(x [B,D], state [B,W-1,D], weight, bias or None, silu) -> y; the state moves on in place
PyObject* py_short_conv_step(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "short_conv_step takes 5 arguments"); return nullptr; }
    const Tensor *x = arg(av[0]), *h = arg(av[1]), *w = arg(av[2]), *b = arg(av[3], true);
    if (!ssm.conv_step || !x || !h || !w || !b || transforms_active() || tracing()) NOT_MINE();
    const int silu = PyObject_IsTrue(av[4]);
    if (silu < 0) { PyErr_Clear(); NOT_MINE(); }
    if (x->dim() != 2 || w->dim() != 2 || dtype_code(*x) < 0 || dtype_code(*w) < 0) NOT_MINE();
    const int64_t B = x->size(0), D = x->size(1), W = w->size(1);
    if (!fits_int({B, D, W}) || W > 8 || w->size(0) != D || !vector_of(*b, D) || !shape3(*h, B, W - 1, D) || !h->is_contiguous() ||
        h->scalar_type() != x->scalar_type() || !same_device(*x, {h, w, b}) || needs_grad({x, h, w, b}))
        NOT_MINE();
    Tensor y;
    if (!guarded([&] {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(x->device());
            const auto type = weights_type({w, b});
            const Tensor xr = rows_of(*x), wc = as_type(*w, type).contiguous(), bc = b->defined() ? as_type(*b, type).contiguous() : *b;
            HdlaConvArgs a{};                                  // (filled in here: views of one token cost more than the call)
            a.B = (int)B; a.T = 1; a.D = (int)D; a.W = (int)W;
            a.dtype = dtype_code(xr); a.w_dtype = dtype_code(wc); a.activation = silu ? HDLA_ACT_SILU : HDLA_ACT_NONE;
            a.x_batch = step_of(xr, 0);
            a.x = ptr(xr); a.weight = ptr(wc); a.bias = ptr(bc); a.h0 = ptr(*h);
            y = dense({B, D}, x->scalar_type(), x->device());
            a.y = mptr(y); a.ht = mptr(*h);
            h->unsafeGetTensorImpl()->bump_version();          // (refuses what may not be changed, before it is)
            check(ssm.conv_step(&a, stream_of(*x)), "hdla_short_conv_step");
        }))
        return nullptr;
    return wrap(y);
}

// ------------------------------------------------------------------------------------------ selective scan
struct ScanIn { Tensor x, dt, A, B, C, D, z, bias, h0, cu; bool softplus = false; };

HdlaScanArgs scan_args(const ScanIn& i) {
    HdlaScanArgs a{};
    a.B = (int)i.x.size(0); a.T = (int)i.x.size(1); a.D = (int)i.x.size(2); a.N = (int)i.A.size(1); a.G = (int)i.B.size(2);
    a.dtype = dtype_code(i.x); a.softplus = i.softplus;
    a.n_seqs = i.cu.defined() ? (int)i.cu.size(0) - 1 : 0;
    a.cu_seqlens = static_cast<const int64_t*>(ptr(i.cu));
    a.x_batch = step_of(i.x, 0); a.x_token = step_of(i.x, 1);
    a.dt_batch = step_of(i.dt, 0); a.dt_token = step_of(i.dt, 1);
    if (i.z.defined()) { a.z_batch = step_of(i.z, 0); a.z_token = step_of(i.z, 1); }
    a.B_batch = step_of(i.B, 0); a.B_token = step_of(i.B, 1); a.B_group = step_of(i.B, 2);
    a.C_batch = step_of(i.C, 0); a.C_token = step_of(i.C, 1); a.C_group = step_of(i.C, 2);
    a.x = ptr(i.x); a.dt = ptr(i.dt); a.z = ptr(i.z); a.Bm = ptr(i.B); a.Cm = ptr(i.C);
    a.A = read(i.A); a.skip = read(i.D); a.dt_bias = read(i.bias); a.h0 = read(i.h0);
    return a;
}
// B and C as [B, T, G, N]
Tensor grouped(const Tensor& t) { return rows_of(t.dim() == 3 ? t.unsqueeze(2) : t); }

struct ScanOut { Tensor y, ht, ckpt; };
ScanOut scan_forward(const ScanIn& i, bool want_ht, bool keep) {
    HdlaScanArgs a = scan_args(i);
    ScanOut r;
    r.y = dense(i.x.sizes(), i.x.scalar_type(), i.x.device());
    if (want_ht) r.ht = dense({sequences(i.cu, a.B), a.D, a.N}, at::kFloat, i.x.device());
    if (keep) r.ckpt = dense({static_cast<int64_t>(ssm.scan_checkpoint_bytes(&a) / sizeof(float))}, at::kFloat, i.x.device());
    const size_t n = ssm.scan_bytes(&a, 0);
    const Tensor ws = space(n, i.x);
    a.y = mptr(r.y); a.ht = fptr(r.ht); a.checkpoints = fptr(r.ckpt);
    check(ssm.scan_fwd(&a, mptr(ws), n, stream_of(i.x)), "hdla_selective_scan_fwd");
    return r;
}
struct ScanGrads { Tensor dx, ddt, dA, dB, dC, dD, dz, dbias, dh0; };
// (without the forward pass's checkpoints it runs once more)
ScanGrads scan_backward(const ScanIn& i, Tensor ckpt, const Tensor& dy_, const Tensor& dht_) {
    c10::cuda::CUDAGuard guard(i.x.device());
    if (!ckpt.defined()) ckpt = scan_forward(i, false, true).ckpt;
    HdlaScanArgs a = scan_args(i);
    const auto st = i.x.scalar_type();
    const Tensor dy = grad_in(dy_, st), dht = grad_in(dht_, at::kFloat);
    auto like = [&](const Tensor& t) { return t.defined() ? dense(t.sizes(), t.scalar_type(), t.device()) : Tensor(); };
    ScanGrads g{like(i.x), like(i.dt), like(i.A), like(i.B), like(i.C), like(i.D), like(i.z), like(i.bias), like(i.h0)};
    const size_t n = ssm.scan_bytes(&a, 1);
    const Tensor ws = space(n, i.x);
    a.checkpoints = fptr(ckpt);
    a.dy = ptr(dy); a.dht = read(dht);
    a.dx = mptr(g.dx); a.ddt = mptr(g.ddt); a.dz = mptr(g.dz); a.dB = mptr(g.dB); a.dC = mptr(g.dC);
    a.dA = fptr(g.dA); a.dskip = fptr(g.dD); a.ddt_bias = fptr(g.dbias); a.dh0 = fptr(g.dh0);
    check(ssm.scan_bwd(&a, mptr(ws), n, stream_of(i.x)), "hdla_selective_scan_bwd");
    return g;
}

struct ScanNode : torch::autograd::Node {
    // ckpt: forward's states, the largest of these by far, so that hooks (offloading, activation checkpointing) get it too; read
    // only, a second backward finds it as it was
    Saved x, dt, A, B, C, D, z, bias, h0, cu, ckpt;
    bool softplus = false;
    at::ScalarType A_type, D_type, bias_type, h0_type;
    std::vector<int64_t> B_size, C_size;
    std::string name() const override { return "HdlaSelectiveScanBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved* s : {&x, &dt, &A, &B, &C, &D, &z, &bias, &h0, &cu, &ckpt}) s->var.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const Tensor dht = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !dht.defined()) return variable_list(9);
        const char* me = "HdlaSelectiveScanBackward";
        const ScanIn i{unpack_saved(x, me), unpack_saved(dt, me), A.get(me), grouped(unpack_saved(B, me)), grouped(unpack_saved(C, me)),
                       D.get(me), unpack_saved(z, me), bias.get(me), h0.get(me), cu.get(me), softplus};
        ScanGrads g = scan_backward(i, ckpt.get(me), grads[0], dht);
        return {g.dx, g.ddt, as_type(g.dA, A_type), g.dB.view(B_size), g.dC.view(C_size), as_type(g.dD, D_type), g.dz,
                as_type(g.dbias, bias_type), as_type(g.dh0, h0_type)};
    }
};

struct ScanCall { const Tensor *x, *dt, *A, *B, *C, *D, *z, *bias, *h0, *cu; bool softplus; };
ScanIn scan_in(const ScanCall& c) {
    return {rows_of(*c.x), rows_of(*c.dt), f32_contiguous(*c.A), grouped(*c.B), grouped(*c.C), f32_contiguous(*c.D), rows_of(*c.z),
            f32_contiguous(*c.bias), f32_contiguous(*c.h0), *c.cu, c.softplus};
}

std::pair<Tensor, Tensor> scan_op(const ScanCall& c, bool want_ht) {
    const bool grad = needs_grad({c.x, c.dt, c.A, c.B, c.C, c.D, c.z, c.bias, c.h0});
    ScanOut r;
    std::shared_ptr<ScanNode> node;
    {
        at::NoGradGuard no_grad;
        c10::cuda::CUDAGuard guard(c.x->device());
        const ScanIn i = scan_in(c);
        r = scan_forward(i, want_ht, grad && !env_is_1("HDLA_RECOMPUTE"));
        if (grad) {
            node = make_node<ScanNode>();
            node->x.save(i.x); node->dt.save(i.dt); node->A.save(i.A); node->D.save(i.D); node->z.save(i.z);
            node->B.save(*c.B); node->C.save(*c.C);
            node->bias.save(i.bias); node->h0.save(i.h0); node->cu.save(i.cu);
            node->ckpt.save(r.ckpt);
            node->softplus = c.softplus;
            auto type = [](const Tensor& t) { return t.defined() ? t.scalar_type() : at::kFloat; };
            node->A_type = type(*c.A); node->D_type = type(*c.D); node->bias_type = type(*c.bias); node->h0_type = type(*c.h0);
            node->B_size = c.B->sizes().vec(); node->C_size = c.C->sizes().vec();
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(*c.x, *c.dt, *c.A, *c.B, *c.C, *c.D, *c.z, *c.bias, *c.h0));
        torch::autograd::create_gradient_edge(r.y, node);
        if (r.ht.defined()) torch::autograd::create_gradient_edge(r.ht, node);
    }
    return {r.y, r.ht};
}

// (x, dt, A, B, C, D or None, z or None, dt_bias or None, softplus, h0 or None, cu_seqlens or None) at av, with `lead` leading
// dimensions of x ([B,T,D]: 2; [B,D]: 1)
bool scan_call(PyObject* const* av, int lead, ScanCall& c) {
    c.x = arg(av[0]); c.dt = arg(av[1]); c.A = arg(av[2]); c.B = arg(av[3]); c.C = arg(av[4]); c.D = arg(av[5], true); c.z = arg(av[6], true);
    c.bias = arg(av[7], true); c.h0 = arg(av[9], true); c.cu = arg(av[10], true);
    if (!ssm.scan_fwd || !c.x || !c.dt || !c.A || !c.B || !c.C || !c.D || !c.z || !c.bias || !c.h0 || !c.cu || transforms_active()) return false;
    const int sp = PyObject_IsTrue(av[8]);
    if (sp < 0) { PyErr_Clear(); return false; }
    c.softplus = sp;
    const Tensor& x = *c.x;
    if (x.dim() != lead + 1 || dtype_code(x) < 0 || c.A->dim() != 2 || !c.A->is_floating_point()) return false;
    const int64_t B = x.size(0), T = lead == 2 ? x.size(1) : 1, D = x.size(lead), N = c.A->size(1);
    if (!fits_int({B, T, D, N}) || N > 128 || T > (1 << 30) || c.A->size(0) != D || c.dt->sizes() != x.sizes() || c.dt->scalar_type() != x.scalar_type())
        return false;
    if (c.z->defined() && (c.z->sizes() != x.sizes() || c.z->scalar_type() != x.scalar_type())) return false;
    if (!vector_of(*c.D, D) || !vector_of(*c.bias, D) || !is_float(*c.h0) || !offsets_tensor(*c.cu, B)) return false;
    for (const Tensor* t : {c.B, c.C}) {
        if (t->scalar_type() != x.scalar_type() || (t->dim() != lead + 1 && t->dim() != lead + 2) || t->size(-1) != N) return false;
        for (int d = 0; d < lead; ++d)
            if (t->size(d) != x.size(d)) return false;
    }
    if (c.B->sizes() != c.C->sizes()) return false;
    const int64_t G = c.B->dim() == lead + 2 ? c.B->size(lead) : 1;
    if (G < 1 || D % G || (c.h0->defined() && !shape3(*c.h0, sequences(*c.cu, B), D, N))) return false;
    return same_device(x, {c.dt, c.A, c.B, c.C, c.D, c.z, c.bias, c.h0, c.cu});
}

// selective_scan(..., output_final_state, keep or None): keep None: the differentiable operator, (y, final state or None); True or
// False: a bare forward call, (y, final state or None, checkpoints or None)
PyObject* py_selective_scan(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 13) { PyErr_SetString(PyExc_TypeError, "selective_scan takes 13 arguments"); return nullptr; }
    ScanCall c;
    const bool bare = av[12] != Py_None;
    const int want = PyObject_IsTrue(av[11]);
    if (want < 0) { PyErr_Clear(); NOT_MINE(); }
    if ((!bare && tracing()) || !scan_call(av, 2, c)) NOT_MINE();
    ScanOut r;
    if (!guarded([&] {
            if (bare) {
                at::NoGradGuard no_grad;
                c10::cuda::CUDAGuard guard(c.x->device());
                r = scan_forward(scan_in(c), want, av[12] == Py_True);
            } else {
                std::tie(r.y, r.ht) = scan_op(c, want);
            }
        }))
        return nullptr;
    return bare ? tuple_of({&r.y, &r.ht, &r.ckpt}) : tuple_of({&r.y, &r.ht});
}
// selective_scan_backward(..., checkpoints or None, dy or None, dht or None) -> gradients of (x, dt, A, B, C, D, z, dt_bias, h0)
PyObject* py_selective_scan_backward(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 14) { PyErr_SetString(PyExc_TypeError, "selective_scan_backward takes 14 arguments"); return nullptr; }
    ScanCall c;
    const Tensor *ck = arg(av[11], true), *dy = arg(av[12], true), *dht = arg(av[13], true);
    if (!scan_call(av, 2, c) || !ck || !dy || !dht) {
        PyErr_SetString(PyExc_TypeError, "selective_scan_backward: arguments of another kind than the forward call's");
        return nullptr;
    }
    ScanGrads g;
    if (!guarded([&] {
            at::NoGradGuard no_grad;
            const ScanIn i = scan_in(c);
            const HdlaScanArgs a = scan_args(i);
            if (ck->defined() && (ck->scalar_type() != at::kFloat || !ck->is_contiguous() || ck->numel() * sizeof(float) < ssm.scan_checkpoint_bytes(&a)))
                throw std::runtime_error("selective_scan_backward: these are not the forward call's checkpoints");
            g = scan_backward(i, *ck, *dy, *dht);
            g.dB = g.dB.view(c.B->sizes()); g.dC = g.dC.view(c.C->sizes());
            if (g.dA.defined()) g.dA = as_type(g.dA, c.A->scalar_type());
            if (g.dD.defined()) g.dD = as_type(g.dD, c.D->scalar_type());
            if (g.dbias.defined()) g.dbias = as_type(g.dbias, c.bias->scalar_type());
            if (g.dh0.defined()) g.dh0 = as_type(g.dh0, c.h0->scalar_type());
        }))
        return nullptr;
    return tuple_of({&g.dx, &g.ddt, &g.dA, &g.dB, &g.dC, &g.dD, &g.dz, &g.dbias, &g.dh0});
}
// selective_scan_step(x [B,D], dt, A, B, C, D, z, dt_bias, softplus, state [B,D,N] fp32) -> y; the state moves on in place
PyObject* py_selective_scan_step(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 10) { PyErr_SetString(PyExc_TypeError, "selective_scan_step takes 10 arguments"); return nullptr; }
    PyObject* all[11];
    for (int i = 0; i < 10; ++i) all[i] = av[i];
    all[10] = Py_None;
    ScanCall c;
    if (tracing() || !scan_call(all, 1, c) || !c.h0->defined() || c.h0->scalar_type() != at::kFloat || !c.h0->is_contiguous() ||
        needs_grad({c.x, c.dt, c.A, c.B, c.C, c.D, c.z, c.bias, c.h0}))
        NOT_MINE();
    Tensor y;
    if (!guarded([&] {
            at::NoGradGuard no_grad;
            c10::cuda::CUDAGuard guard(c.x->device());
            const Tensor x = rows_of(*c.x), dt = rows_of(*c.dt), z = rows_of(*c.z), B = rows_of(*c.B), C = rows_of(*c.C),
                         A = f32_contiguous(*c.A), D = f32_contiguous(*c.D), bias = f32_contiguous(*c.bias);
            HdlaScanArgs a{};                                  // (filled in here: views of one token cost more than the call)
            a.B = (int)x.size(0); a.T = 1; a.D = (int)x.size(1); a.N = (int)A.size(1); a.G = B.dim() == 3 ? (int)B.size(1) : 1;
            a.dtype = dtype_code(x); a.softplus = c.softplus;
            a.x_batch = step_of(x, 0); a.dt_batch = step_of(dt, 0); a.z_batch = z.defined() ? step_of(z, 0) : 0;
            a.B_batch = step_of(B, 0); a.C_batch = step_of(C, 0);
            if (B.dim() == 3) { a.B_group = step_of(B, 1); a.C_group = step_of(C, 1); }
            a.x = ptr(x); a.dt = ptr(dt); a.z = ptr(z); a.Bm = ptr(B); a.Cm = ptr(C);
            a.A = read(A); a.skip = read(D); a.dt_bias = read(bias); a.h0 = read(*c.h0);
            y = dense({a.B, a.D}, c.x->scalar_type(), c.x->device());
            a.y = mptr(y); a.ht = fptr(*c.h0);
            c.h0->unsafeGetTensorImpl()->bump_version();
            check(ssm.scan_step(&a, stream_of(*c.x)), "hdla_selective_scan_step");
        }))
        return nullptr;
    return wrap(y);
}

// ------------------------------------------------------------------------------------------ norms round a block
struct NormIn { Tensor x, r, g, post, pre, scale; double scale_value = 1.0, eps = 0.0; int act = 0; at::ScalarType w_type = at::kFloat; };

HdlaNormResidualArgs norm_args(const NormIn& i) {
    HdlaNormResidualArgs a{};
    a.D = (int)i.x.size(-1);
    a.rows = i.x.numel() / a.D;
    a.dtype = dtype_code(i.x); a.r_dtype = i.r.defined() ? dtype_code(i.r) : a.dtype;
    a.w_dtype = i.w_type == at::kFloat ? HDLA_F32 : HDLA_BF16;
    a.activation = i.act; a.eps = static_cast<float>(i.eps); a.scale_value = static_cast<float>(i.scale_value);
    a.x = ptr(i.x); a.residual = ptr(i.r); a.gate = ptr(i.g); a.post_weight = ptr(i.post); a.pre_weight = ptr(i.pre); a.scale = ptr(i.scale);
    return a;
}
struct NormOut { Tensor r, u, factors; };
NormOut norm_forward(const NormIn& i, bool keep) {
    HdlaNormResidualArgs a = norm_args(i);
    const Tensor r = dense(i.x.sizes(), i.r.defined() ? i.r.scalar_type() : i.x.scalar_type(), i.x.device());
    Tensor u;
    if (i.pre.defined()) u = dense_like(i.x);
    Tensor factors;
    if (keep && (i.post.defined() || i.pre.defined())) factors = dense({a.rows, 2}, at::kFloat, i.x.device());
    a.r = mptr(r); a.u = mptr(u); a.factors = fptr(factors);
    check(ssm.norm_fwd(&a, stream_of(i.x)), "hdla_norm_residual_fwd");
    return {r, u, factors};
}
struct NormGrads { Tensor dx, dr, dg, dpost, dpre, dscale; };
NormGrads norm_backward(const NormIn& i, const Tensor& factors, const Tensor& dr_, const Tensor& du_) {
    c10::cuda::CUDAGuard guard(i.x.device());
    HdlaNormResidualArgs a = norm_args(i);
    const Tensor dr = grad_in(dr_, i.r.defined() ? i.r.scalar_type() : i.x.scalar_type()), du = grad_in(du_, i.x.scalar_type());
    auto like = [&](const Tensor& t) { return t.defined() ? dense_like(t) : Tensor(); };
    NormGrads g{like(i.x), like(i.r), like(i.g), like(i.post), like(i.pre), like(i.scale)};
    const size_t n = ssm.norm_bwd_bytes(&a);
    const Tensor ws = space(n, i.x);
    a.dr = ptr(dr); a.du = ptr(du); a.factors = fptr(factors);
    a.dx = mptr(g.dx); a.dresidual = mptr(g.dr); a.dgate = mptr(g.dg);
    a.dpost_weight = mptr(g.dpost); a.dpre_weight = mptr(g.dpre); a.dscale = mptr(g.dscale);
    check(ssm.norm_bwd(&a, mptr(ws), n, stream_of(i.x)), "hdla_norm_residual_bwd");
    return g;
}

struct NormCall { const Tensor *x, *r, *g, *scale, *post, *pre; double scale_value, eps; int act; };
NormIn norm_in(const NormCall& c) {
    NormIn i;
    i.w_type = weights_type({c.post, c.pre, c.scale});
    auto weight = [&](const Tensor& t) { return t.defined() ? as_type(t, i.w_type).contiguous() : t; };
    i.x = c.x->contiguous(); i.r = c.r->defined() ? c.r->contiguous() : *c.r; i.g = c.g->defined() ? c.g->contiguous() : *c.g;
    i.post = weight(*c.post); i.pre = weight(*c.pre); i.scale = weight(*c.scale);
    i.scale_value = c.scale_value; i.eps = c.eps; i.act = c.act;
    return i;
}

struct NormResidualNode : torch::autograd::Node {
    Saved x, r, g, post, pre, scale, factors;
    NormIn rest;                                     // the numbers; no tensors
    at::ScalarType post_type = at::kFloat, pre_type = at::kFloat, scale_type = at::kFloat;
    std::string name() const override { return "HdlaNormResidualBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved* s : {&x, &r, &g, &post, &pre, &scale, &factors}) s->var.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        at::NoGradGuard no_grad;
        const Tensor du = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !du.defined()) return variable_list(6);
        const char* me = "HdlaNormResidualBackward";
        NormIn i = rest;
        i.x = x.get(me); i.r = r.get(me); i.g = g.get(me); i.post = post.get(me); i.pre = pre.get(me); i.scale = scale.get(me);
        NormGrads d = norm_backward(i, factors.get(me), grads[0], du);
        return {d.dx, d.dr, d.dg, as_type(d.dscale, scale_type), as_type(d.dpost, post_type), as_type(d.dpre, pre_type)};
    }
};

std::pair<Tensor, Tensor> norm_residual_op(const NormCall& c) {
    const bool grad = needs_grad({c.x, c.r, c.g, c.scale, c.post, c.pre});
    NormOut out;
    std::shared_ptr<NormResidualNode> node;
    {
        at::NoGradGuard no_grad;
        c10::cuda::CUDAGuard guard(c.x->device());
        const NormIn i = norm_in(c);
        out = norm_forward(i, grad);
        if (grad) {
            node = make_node<NormResidualNode>();
            node->x.save(i.x); node->r.save(i.r); node->g.save(i.g); node->post.save(i.post); node->pre.save(i.pre); node->scale.save(i.scale);
            node->factors.save(out.factors);
            node->rest.scale_value = i.scale_value; node->rest.eps = i.eps; node->rest.act = i.act; node->rest.w_type = i.w_type;
            if (c.post->defined()) node->post_type = c.post->scalar_type();
            if (c.pre->defined()) node->pre_type = c.pre->scalar_type();
            if (c.scale->defined()) node->scale_type = c.scale->scalar_type();
        }
    }
    if (grad) {
        node->set_next_edges(torch::autograd::collect_next_edges(*c.x, *c.r, *c.g, *c.scale, *c.post, *c.pre));
        torch::autograd::create_gradient_edge(out.r, node);
        if (out.u.defined()) torch::autograd::create_gradient_edge(out.u, node);
    }
    return {out.r, out.u};
}

// (x, residual or None, gate or None, scale: a vector or a number, post or None, pre or None, activation code, eps) at av
bool norm_call(PyObject* const* av, NormCall& c) {
    c.x = arg(av[0]); c.r = arg(av[1], true); c.g = arg(av[2], true); c.post = arg(av[4], true); c.pre = arg(av[5], true);
    c.scale = THPVariable_Check(av[3]) ? arg(av[3]) : &kNone;
    if (!ssm.norm_fwd || !c.x || !c.r || !c.g || !c.post || !c.pre || !c.scale || transforms_active()) return false;
    c.scale_value = c.scale->defined() ? 1.0 : PyFloat_AsDouble(av[3]);
    const long act = PyLong_AsLong(av[6]);
    c.eps = PyFloat_AsDouble(av[7]);
    if (PyErr_Occurred()) { PyErr_Clear(); return false; }
    c.act = static_cast<int>(act);
    const Tensor& x = *c.x;
    if (dtype_code(x) < 0 || x.dim() < 1 || x.numel() == 0 || x.size(-1) > 8192) return false;
    const int64_t D = x.size(-1);
    for (const Tensor* t : {c.r, c.g})
        if (t->defined() && t->sizes() != x.sizes()) return false;
    if (c.g->defined() && c.g->scalar_type() != x.scalar_type()) return false;
    if (c.r->defined() && c.r->scalar_type() != x.scalar_type() && c.r->scalar_type() != at::kFloat) return false;
    if (!vector_of(*c.post, D) || !vector_of(*c.pre, D) || !vector_of(*c.scale, D)) return false;
    return same_device(x, {c.r, c.g, c.scale, c.post, c.pre});
}

// norm_residual(..., keep or None): keep None: the differentiable operator, (r, u or None); True or False: a bare forward call,
// (r, u or None, the norms' factors or None)
PyObject* py_norm_residual(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "norm_residual takes 9 arguments"); return nullptr; }
    NormCall c;
    const bool bare = av[8] != Py_None;
    if ((!bare && tracing()) || !norm_call(av, c)) NOT_MINE();
    NormOut r;
    if (!guarded([&] {
            if (bare) {
                at::NoGradGuard no_grad;
                c10::cuda::CUDAGuard guard(c.x->device());
                r = norm_forward(norm_in(c), av[8] == Py_True);
            } else {
                std::tie(r.r, r.u) = norm_residual_op(c);
            }
        }))
        return nullptr;
    return bare ? tuple_of({&r.r, &r.u, &r.factors}) : tuple_of({&r.r, &r.u});
}
// norm_residual_backward(..., factors or None, dr or None, du or None) -> gradients of (x, residual, gate, scale, post, pre)
PyObject* py_norm_residual_backward(PyObject*, PyObject* const* av, Py_ssize_t n) {
    if (n != 11) { PyErr_SetString(PyExc_TypeError, "norm_residual_backward takes 11 arguments"); return nullptr; }
    NormCall c;
    const Tensor *factors = arg(av[8], true), *dr = arg(av[9], true), *du = arg(av[10], true);
    if (!norm_call(av, c) || !factors || !dr || !du ||
        (factors->defined() && (factors->scalar_type() != at::kFloat || !factors->is_contiguous() || factors->numel() != 2 * (c.x->numel() / c.x->size(-1))))) {
        PyErr_SetString(PyExc_TypeError, "norm_residual_backward: arguments of another kind than the forward call's");
        return nullptr;
    }
    NormGrads g;
    if (!guarded([&] {
            at::NoGradGuard no_grad;
            g = norm_backward(norm_in(c), *factors, *dr, *du);
            if (g.dscale.defined()) g.dscale = as_type(g.dscale, c.scale->scalar_type());
            if (g.dpost.defined()) g.dpost = as_type(g.dpost, c.post->scalar_type());
            if (g.dpre.defined()) g.dpre = as_type(g.dpre, c.pre->scalar_type());
        }))
        return nullptr;
    return tuple_of({&g.dx, &g.dr, &g.dg, &g.dscale, &g.dpost, &g.dpre});
}

}  // namespace
