"""GPU: calls of the short convolution, the selective scan and the norms round a block that lie at the edge of what they take.

Tolerances are of the kind of test_gpu_ssm.py: an output of type t is rounded once (finfo(t).eps / 2), all else is fp32."""
import math

import pytest
import torch

from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.device("cuda:0")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rn(g, *s, dtype=F32, scale=1.0):
    return (scale * torch.randn(*s, generator=g)).to(dtype)


def off(got, ref):
    """Largest difference relative to the largest value of the definition."""
    assert got.shape == ref.shape and bool(torch.isfinite(got).all())
    return float((got.detach().cpu().double() - ref.detach()).abs().max()) / float(ref.detach().abs().max())


# --------------------------------------------------------------------------------------------- norms
@pytest.mark.parametrize("D", [64, 1001, 8192])
@pytest.mark.parametrize("which", ["post_weight", "pre_weight"])
@pytest.mark.parametrize("size,eps", [(1e12, 1e-5), (1e15, 1e-5), (1e-14, 1e-30)])
def test_norms_of_large_and_of_tiny_rows(dev, D, which, size, eps):
    """The norms' gradient takes its second term, the projection on the row, where the cube of the norm's factor is no fp32 number
    (1e-45 at rows of 1e15, 1e42 at rows of 1e-14), and so do the gradients that are small themselves (dy of 1e-3)."""
    from hdla_impl_b200 import layer_ops
    g = gen(D)
    x, w, do = rn(g, 3, D, scale=size), rn(g, D), rn(g, 3, D, scale=1e-3)
    a, v = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = [t for t in layer_ops.rms_norm_residual(a, **{which: v}, eps=eps) if t is not None][-1]
    got = torch.autograd.grad(y, [a, v], do.to(dev))
    b, c = x.double().requires_grad_(True), w.double().requires_grad_(True)
    r = [t for t in orc.norm_residual(b, **{which[:-7]: c}, eps=eps) if t is not None][-1]
    # sums of D roundings of random sign and a dozen operations: (sqrt(D) + 64) 2^-21, and the gradient is a difference: 8 times
    tol = 8 * (math.sqrt(D) + 64) * 2.0 ** -21
    assert off(y, r) <= tol
    for p, q in zip(got, torch.autograd.grad(r, [b, c], do.double())):
        assert off(p, q) <= tol


@pytest.mark.parametrize("D", [(4104, 8192), (2056, 4096)])
def test_threads_with_rows_of_different_widths(dev, D):
    """Two threads, each with its stream: widths that one kernel serves with different amounts of shared memory, forward and
    backward.  No launch is refused, and both get what they get alone."""
    import threading
    from hdla_impl_b200 import layer_ops

    def call(x, w):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        r, u = layer_ops.rms_norm_residual(x, post_weight=w, pre_weight=w)
        return [r.detach(), u.detach(), *torch.autograd.grad([r, u], [x, w], [x.detach(), x.detach()])]

    g = gen(6)
    inputs = [(rn(g, 4, d).to(dev), rn(g, d).to(dev)) for d in D]
    want = [call(*i) for i in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for i in range(1500):
                    got = call(*inputs[k])
                    if i % 100 == 0 and not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append((D[k], i, "values"))
        except Exception as e:  # noqa: BLE001
            wrong.append((D[k], repr(e)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong


@pytest.mark.parametrize("D", [(4104, 8192), (2056, 4096)])
def test_threads_with_rows_of_different_widths_at_the_c_entry_points(dev, D):
    """The same without PyTorch between the calls, so that two threads often stand between a limit and its launch."""
    import ctypes as C
    import threading
    from hdla_impl_b200 import _lib
    from test_ssm_host import Norm
    lib = C.CDLL(_lib.lib_path())                            # (prototypes of its own)
    size = lib.hdla_norm_residual_bwd_workspace_bytes
    size.restype = C.c_size_t
    wrong, keep = [], []

    def calls_of(d):
        x, w, out, f = torch.ones(2, d, device=dev), torch.ones(d, device=dev), torch.empty(8, 2, d, device=dev), torch.empty(2, 2, device=dev)
        at = lambda k: out[k].data_ptr()  # noqa: E731
        a = Norm(rows=2, D=d, eps=1e-5, scale_value=1.0, x=x.data_ptr(), post_weight=w.data_ptr(), pre_weight=w.data_ptr(), r=at(0), u=at(1),
                 factors=f.data_ptr(), dr=x.data_ptr(), du=x.data_ptr(), dx=at(2), dpost_weight=at(3), dpre_weight=at(4))
        ws = torch.empty(size(C.byref(a)), dtype=torch.uint8, device=dev)
        keep.extend((x, w, out, f, ws, a))
        return a, ws

    def work(d, a, ws, stream):
        for i in range(4000):
            rc = lib.hdla_norm_residual_fwd(C.byref(a), C.c_void_p(stream)) if i % 2 == 0 else \
                lib.hdla_norm_residual_bwd(C.byref(a), C.c_void_p(ws.data_ptr()), C.c_size_t(ws.numel()), C.c_void_p(stream))
            if rc != 0:
                wrong.append((d, i, rc))
                return

    streams = [torch.cuda.Stream(dev) for _ in D]
    threads = [threading.Thread(target=work, args=(d, *calls_of(d), s.cuda_stream)) for d, s in zip(D, streams)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong


# --------------------------------------------------------------------------------------------- short convolution
@pytest.mark.parametrize("xt", [F32, BF])
@pytest.mark.parametrize("wt,bt", [(BF, F32), (F32, BF), (BF, torch.float16), (BF, torch.float64)])
def test_taps_and_bias_of_different_types_keep_their_digits(dev, xt, wt, bt):
    """The wider of the two is not rounded to the other's type: prompts, gradients and single tokens."""
    from hdla_impl_b200 import ssm
    g = gen(4)
    x, w, b, do = rn(g, 2, 40, 16, dtype=xt), rn(g, 16, 4, dtype=wt), rn(g, 16, scale=50).to(bt), rn(g, 2, 40, 16, dtype=xt)
    h0 = torch.zeros(2, 3, 16, dtype=xt)
    t = [v.to(dev).requires_grad_(True) for v in (x, w, b)]
    y, _ = ssm.short_convolution(*t, activation=None)
    got = torch.autograd.grad(y, t, do.to(dev))
    with torch.no_grad():
        first = ssm.short_convolution_step(t[0][:, 0], h0.to(dev), *t[1:], activation=None)
    assert torch.equal(first, y[:, 0])
    ref = [v.double().requires_grad_(True) for v in (x, w, b)]
    r, _ = orc.short_conv(*ref, None)
    half = lambda t: torch.finfo(t).eps / 2  # noqa: E731
    # five roundings of fp32 a sum of taps, one to the output's type; the weights' gradients are sums of 80 terms
    assert off(y, r) <= half(xt) + 64 * 2.0 ** -24
    for a, v, q in zip(got, t, torch.autograd.grad(r, ref, do.double())):
        assert a.dtype == v.dtype and off(a, q) <= half(max(a.dtype, F32, key=lambda d: torch.finfo(d).eps)) + 80 * 2.0 ** -24


# --------------------------------------------------------------------------------------------- selective scan
def test_shares_of_few_states_take_turns(dev):
    """Eight states, sixteen groups of 68 channels (two tiles of channels each), 2^23 tokens times groups: one tile's shares of dB and
    dC take half of the limit of 1 GiB and a little more, so that the tiles of the whole batch go in two launches, the second of which
    adds to the first's shares; those of each row of the batch go in one.  Decays of a half and less a token: what a row's cuts into
    segments round differently is as small as a state's own rounding."""
    from hdla_impl_b200 import ssm
    G, per, N, T = 16, 68, 8, (1 << 18) + 8
    D = G * per
    g = torch.Generator(device=dev).manual_seed(17)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=BF)  # noqa: E731
    t = {"x": rnd(2, T, D), "dt": rnd(2, T, D).abs_(), "B": rnd(2, T, G, N), "C": rnd(2, T, G, N)}
    A = -1 - torch.rand(D, N, generator=g, device=dev)
    dy = rnd(2, T, D)

    def f(rows):
        leaves = [v[rows].detach().requires_grad_(k in "BC") for k, v in t.items()]
        y, _ = ssm.selective_scan(leaves[0], leaves[1], A, *leaves[2:])
        return torch.autograd.grad(y, leaves[2:], dy[rows])

    whole = f(slice(0, 2))
    for b in range(2):
        for name, a, c in zip(("dB", "dC"), whole, f(slice(b, b + 1))):
            # both sides are rounded to bf16; fp32 before that, over a state's memory of some ten tokens and 68 channels
            e = float((a[b].float() - c[0].float()).abs().max() / c.float().abs().max())
            assert e <= 2 * torch.finfo(BF).eps / 2 + 128 * 2.0 ** -21, (name, b, e)


# --------------------------------------------------------------------------------------------- tracing
def traceable(dev):
    """{name: (function of tensors, tensors)}: each operator for whole sequences."""
    from hdla_impl_b200 import layer_ops, ssm
    g = gen(23)
    D, N = 24, 8
    x, z, w, b = rn(g, 2, 30, D, dtype=BF), rn(g, 2, 30, D, dtype=BF), rn(g, D, 4, dtype=BF), rn(g, D, dtype=BF)
    bc, A = rn(g, 2, 30, N, dtype=BF), -torch.exp(rn(g, D, N))
    calls = {
        "conv": (lambda x, w, b: ssm.short_convolution(x, w, b, output_final_state=True), (x, w, b)),
        "scan": (lambda x, z, A, bc: ssm.selective_scan(x, z, A, bc, bc, z=z, output_final_state=True), (x, z, A, bc)),
        "norm": (lambda x, z, b: layer_ops.rms_norm_residual(x, z, gate=z, scale=b, post_weight=b, pre_weight=b), (x, z, b)),
        "norm without weights": (lambda x, z: layer_ops.rms_norm_residual(x, z, scale=0.5)[0], (x, z)),
    }
    return {k: (f, [t.to(dev) for t in ts]) for k, (f, ts) in calls.items()}


@pytest.mark.parametrize("what", ["conv", "scan", "norm", "norm without weights"])
def test_a_traced_call_runs_on_its_own_inputs(dev, what):
    """torch.jit.trace records the operators as calls: the traced function computes on what it is given, not what it was traced with."""
    f, x = traceable(dev)[what]
    y = [t.flip(1) if t.dim() == 3 else t for t in x]
    traced = torch.jit.trace(f, tuple(x), check_trace=False)
    for inputs in (y, x):
        got, want = traced(*inputs), f(*inputs)
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b)


def test_single_tokens_refuse_to_be_traced(dev):
    from hdla_impl_b200 import ssm
    x, w, A = torch.ones(2, 8, device=dev), torch.ones(8, 4, device=dev), -torch.ones(8, 4, device=dev)
    conv, state = torch.zeros(2, 3, 8, device=dev), torch.zeros(2, 8, 4, device=dev)
    for f in (lambda x: ssm.short_convolution_step(x, conv, w), lambda x: ssm.selective_scan_step(x, x, A, x[:, :4], x[:, :4], state)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
    assert float(conv.abs().max()) == 0 and float(state.abs().max()) == 0


@pytest.mark.parametrize("what", ["conv", "scan", "norm", "norm without weights"])
def test_a_compiled_function_calls_the_operators(dev, what):
    """torch.compile leaves them out of its graphs: the same bits, gradients among them, and new offsets at every call."""
    f, x = traceable(dev)[what]
    torch._dynamo.reset()

    def g(*ts):
        y = f(*[t * 1 for t in ts])
        return [t + 0 for t in (y if isinstance(y, tuple) else (y,))]

    def both(h):
        leaves = [t.detach().requires_grad_(True) for t in x]
        out = h(*leaves)
        return [*out, *torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])]

    for a, b in zip(both(torch.compile(g, backend="eager")), both(g)):
        assert torch.equal(a, b)


def test_compiled_single_tokens_and_packed_batches(dev):
    from hdla_impl_b200 import ssm
    torch._dynamo.reset()
    g = gen(29)
    x, w, A, bc = rn(g, 1, 40, 8).to(dev), rn(g, 8, 4).to(dev), -torch.exp(rn(g, 8, 4)).to(dev), rn(g, 1, 40, 4).to(dev)

    def step(x, bc, conv, scan):
        c = ssm.short_convolution_step(x * 2, conv, w)
        return ssm.selective_scan_step(c, x, A, bc, bc, scan) + 1

    def packed(x, bc, cu):
        c, _ = ssm.short_convolution(x * 2, w, cu_seqlens=cu)
        return ssm.selective_scan(c, x, A, bc, bc, cu_seqlens=cu)[0] + 1

    fast = torch.compile(step, backend="eager"), torch.compile(packed, backend="eager")
    states = [[torch.zeros(1, 3, 8, device=dev), torch.zeros(1, 8, 4, device=dev)] for _ in range(2)]
    for t in range(4):
        assert torch.equal(fast[0](x[:, t], bc[:, t], *states[0]), step(x[:, t], bc[:, t], *states[1]))
    assert all(torch.equal(a, b) for a, b in zip(*states))
    for cut in range(3, 15):
        assert torch.equal(fast[1](x, bc, [0, cut, 40]), packed(x, bc, [0, cut, 40]))


# --------------------------------------------------------------------------------------------- what is kept for backward
def scan_for_memory(dev):
    """A scan whose checkpoints (8 bytes a token and channel) outweigh all else: (function, leaves, gradient of y, bytes of y, of them)."""
    from hdla_impl_b200 import ssm
    g = torch.Generator(device=dev).manual_seed(3)
    B, T, D, N = 2, 1024, 512, 16
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    t = [rnd(B, T, D), rnd(B, T, D), -torch.exp(rnd(D, N)), rnd(B, T, N), rnd(B, T, N)]
    for v in t:
        v.requires_grad_(True)
    return (lambda *t: ssm.selective_scan(*t)[0]), t, rnd(B, T, D), B * T * D * 4, B * T // 8 * D * N * 4


def kept(f):
    """(what f returns, the bytes that it has left allocated)"""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = f()
    torch.cuda.synchronize()
    return y, torch.cuda.memory_allocated() - before


@pytest.mark.parametrize("how", ["checkpoint", "save_on_cpu", "subclass on cpu"])
def test_the_scans_checkpoints_go_through_saved_tensor_hooks(dev, how):
    """Activation checkpointing and offloading leave nothing of them on the GPU until backward, and the gradients are the same bits."""
    from torch.utils.checkpoint import checkpoint

    class Mine(torch.Tensor):
        pass

    f, t, dy, size, saved = scan_for_memory(dev)
    y, bytes_ = kept(lambda: f(*t))
    assert bytes_ >= size + saved
    want = torch.autograd.grad(y, t, dy)

    def call():
        if how == "checkpoint":
            return checkpoint(f, *t, use_reentrant=False)
        with torch.autograd.graph.save_on_cpu():
            return f(*t) if how == "save_on_cpu" else f(t[0].as_subclass(Mine), *t[1:])

    y2, bytes_ = kept(call)
    assert bytes_ < size + saved // 4
    assert torch.equal(y2.as_subclass(torch.Tensor), y)
    for a, b in zip(torch.autograd.grad(y2, t, dy), want):
        assert torch.equal(a.as_subclass(torch.Tensor), b)


@pytest.mark.parametrize("subclass", [False, True])
def test_the_scans_checkpoints_can_be_done_without(dev, monkeypatch, subclass):
    """HDLA_RECOMPUTE=1, as for the chunked operator: nothing of them is kept, and the gradients are the same bits, twice."""
    class Mine(torch.Tensor):
        pass

    f, t, dy, size, saved = scan_for_memory(dev)
    want = torch.autograd.grad(f(*t), t, dy)
    monkeypatch.setenv("HDLA_RECOMPUTE", "1")
    y, bytes_ = kept(lambda: f(t[0].as_subclass(Mine) if subclass else t[0], *t[1:]))
    assert bytes_ < size + saved // 4
    for again in (True, False):
        for a, b in zip(torch.autograd.grad(y, t, dy, retain_graph=again), want):
            assert torch.equal(a.as_subclass(torch.Tensor), b)


def test_the_norms_factors_go_through_saved_tensor_hooks(dev):
    from hdla_impl_b200 import layer_ops
    g = gen(5)
    x, w, do = rn(g, 40, 64).to(dev).requires_grad_(True), rn(g, 64).to(dev).requires_grad_(True), rn(g, 40, 64).to(dev)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(tuple(t.shape)) or t.cpu(), lambda t: t.to(dev)):
        r, u = layer_ops.rms_norm_residual(x, post_weight=w, pre_weight=w)
    r2, u2 = layer_ops.rms_norm_residual(x, post_weight=w, pre_weight=w)
    assert (40, 2) in seen
    for a, b in zip(torch.autograd.grad([r, u], [x, w], [do, do]), torch.autograd.grad([r2, u2], [x, w], [do, do])):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------------------------- offsets
@pytest.mark.parametrize("given,taken", [([0, -3, 20, 50], [0, 0, 20, 50]), ([5, 20, 50, 50], [0, 20, 50, 50]), ([0, 20, 1000, 1 << 40], [0, 20, 50, 50]),
                                         ([-(1 << 40), -7, 0, 33], [0, 0, 0, 33])])
def test_offsets_on_the_gpu_are_cut_to_the_batch(dev, given, taken):
    """Offsets on the GPU are not looked at by the host: the first counts as 0, those outside 0..T are cut to that range.  Outputs,
    states and all gradients are those of the offsets that result."""
    from hdla_impl_b200 import ssm
    g = gen(50)
    T, D, N = 50, 16, 4
    t = {"x": rn(g, 1, T, D), "w": rn(g, D, 4), "h": rn(g, 3, 3, D), "dt": rn(g, 1, T, D), "A": -torch.exp(rn(g, D, N)), "B": rn(g, 1, T, N),
         "C": rn(g, 1, T, N), "z": rn(g, 1, T, D), "s": rn(g, 3, D, N)}
    dy, dh, ds = rn(g, 1, T, D).to(dev), rn(g, 3, 3, D).to(dev), rn(g, 3, D, N).to(dev)

    def f(cu):
        v = {k: a.to(dev).requires_grad_(True) for k, a in t.items()}
        c, h = ssm.short_convolution(v["x"], v["w"], initial_state=v["h"], output_final_state=True, cu_seqlens=cu)
        y, s = ssm.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], z=v["z"], initial_state=v["s"], output_final_state=True, cu_seqlens=cu)
        return [c, h, y, s, *torch.autograd.grad([c, h, y, s], list(v.values()), [dy, dh, dy, ds])]

    for a, b in zip(f(torch.tensor(given, device=dev)), f(torch.tensor(taken, device=dev))):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


# --------------------------------------------------------------------------------------------- gradients that are long sums
# Inputs without signs, so that no sum cancels and a lost or doubled token shows in every entry: errors are taken entry by entry,
# relative to the sum of the magnitudes of what it consists of.  u = 2^-24 is a rounding of fp32.
U = 2.0 ** -24


def entries_close(got, ref, size, tol, name):
    assert got.dtype == F32 and got.shape == ref.shape
    e = float(((got.cpu().double() - ref).abs() / size).max())
    assert e <= tol, f"{name}: {e:.3g} > {tol:.3g}"


def scan64(x, dt, dt2, A, B, C, D, z, bias, bias2, h0, cu):
    """The definition, with the time steps of the decays (dt2, bias2) apart from those of the inputs: their gradients have opposite signs."""
    T = x.shape[1]
    sp = lambda v: torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    d, d2 = sp(dt + bias), sp(dt2 + bias2)
    per = x.shape[2] // B.shape[2]
    ys, first, h = [], dict(zip(cu, range(len(cu) - 1))), None
    for t in range(T):
        if t in first:
            h = h0[first[t]][None]
        h = torch.exp(d2[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t].repeat_interleave(per, 1)
        ys.append(((C[:, t].repeat_interleave(per, 1) * h).sum(-1) + D * x[:, t]) * z[:, t] / (1 + torch.exp(-z[:, t])))
    return torch.stack(ys, 1)


@pytest.mark.parametrize("T,D,N,G,dtype,slow,cu", [(1300, 8, 16, 1, F32, 64, None), (1300, 8, 16, 2, BF, 64, [0, 1, 640, 1300]), (200, 24, 5, 1, F32, 1e6, None),
                                                   (700, 8, 128, 2, BF, 64, None), (900, 12, 8, 1, F32, 16, [0, 899, 900])])
def test_every_token_is_in_the_weights_gradients_once(dev, T, D, N, G, dtype, slow, cu):
    """Decays of 1 / slow a token and more: a state remembers min(T, slow) tokens.  Each of them costs a rounding, the exponential's
    4 u and what the rounding of its argument does, 5 u in all, for the state and for its gradient; 10 u each for the time step in
    the exponent; T u at most for a sum of T terms without signs; 64 u for the rest.  A token is 1 / T of such a sum."""
    from hdla_impl_b200 import ssm
    g = gen(T)
    pos = lambda *s, dtype=dtype: (0.5 + torch.rand(*s, generator=g)).to(dtype)  # noqa: E731
    seqs = [0, T] if cu is None else cu
    v = {"x": pos(1, T, D), "dt": torch.randn(1, T, D, generator=g).to(dtype), "A": -(1 + torch.rand(D, N, generator=g)) / slow * 4, "B": pos(1, T, G, N),
         "C": pos(1, T, G, N), "D": pos(D, dtype=F32), "z": pos(1, T, D), "bias": 0.5 + torch.rand(D, generator=g), "h0": pos(len(seqs) - 1, D, N, dtype=F32)}
    dy = pos(1, T, D)
    own = {k: a.to(dev).requires_grad_(k in ("A", "D", "bias", "h0")) for k, a in v.items()}
    y, _ = ssm.selective_scan(own["x"], own["dt"], own["A"], own["B"], own["C"], D=own["D"], z=own["z"], dt_bias=own["bias"], initial_state=own["h0"],
                              cu_seqlens=cu)
    names = ["A", "D", "bias", "h0"]
    got = dict(zip(names, torch.autograd.grad(y, [own[k] for k in names], dy.to(dev))))
    ref = {k: a.double().requires_grad_(k in names) for k, a in v.items()}
    bias2 = ref["bias"].detach().clone().requires_grad_(True)
    r = scan64(ref["x"], ref["dt"], ref["dt"], ref["A"], ref["B"], ref["C"], ref["D"], ref["z"], ref["bias"], bias2, ref["h0"], seqs)
    want = dict(zip([*names, "bias2"], torch.autograd.grad(r, [*(ref[k] for k in names), bias2], dy.double())))
    size = {k: w.abs() for k, w in want.items()}
    size["bias"] = size["bias"] + size["bias2"]
    want["bias"] = want["bias"] + want["bias2"]
    tol = (2 * (10 + 5 * min(T, slow)) + T + 64) * U
    assert tol < 0.5 / T
    for k in names:
        entries_close(got[k], want[k], size[k], tol, "d" + k)


@pytest.mark.parametrize("rows,D,dtype,rt", [(1300, 256, BF, BF), (1300, 256, BF, F32), (3001, 1001, F32, F32), (700, 2048, BF, F32), (900, 5000, BF, F32)])
def test_every_row_is_in_the_norms_weights_gradients_once(dev, rows, D, dtype, rt):
    """A factor of a row costs the roundings of a tree over D squares, 32 u, and its root's 4 u; the gate 16 u; a block's rows and
    the blocks one after another, at most rows / 100 + 64 u."""
    from hdla_impl_b200 import layer_ops
    g = gen(D)
    pos = lambda *s, dtype=dtype: (0.5 + torch.rand(*s, generator=g)).to(dtype)  # noqa: E731
    x, r, gate, do = pos(rows, D), pos(rows, D, dtype=rt), pos(rows, D), pos(rows, D)
    w = {k: pos(D, dtype=F32) for k in ("scale", "post_weight", "pre_weight")}
    tol = (32 + 4 + 16 + 64 + 64 + rows / 100) * U
    assert tol < 0.5 / rows
    # the scale's and the first norm's gradients where there is no second norm, whose own gradient is a difference
    for names in (("scale", "post_weight"), ("pre_weight", "scale", "post_weight")):
        own = {k: w[k].to(dev).requires_grad_(True) for k in names}
        out = layer_ops.rms_norm_residual(x.to(dev), r.to(dev), gate=gate.to(dev), **own)
        last, up = (out[0], do.to(rt)) if len(names) == 2 else (out[1], do)
        ref = {k: w[k].double().requires_grad_(True) for k in names}
        ro = orc.norm_residual(x.double(), r.double(), gate.double(), ref["scale"], ref["post_weight"], ref.get("pre_weight"))
        want = torch.autograd.grad(ro[0] if len(names) == 2 else ro[1], list(ref.values()), up.double())
        got = torch.autograd.grad(last, list(own.values()), up.to(dev))
        for k, a, b in list(zip(names, got, want))[:1 if len(names) == 3 else 2]:
            entries_close(a, b, b.abs(), tol, "d" + k)


@pytest.mark.parametrize("B,T,D,W,dtype,cu", [(2, 3001, 40, 4, BF, None), (1, 5000, 33, 7, F32, [0, 1, 2, 2400, 5000]), (3, 129, 64, 2, F32, None)])
def test_every_token_is_in_the_convolutions_weights_gradients_once(dev, B, T, D, W, dtype, cu):
    """W + 1 roundings and a sigmoid's 16 u a token; a strip of 128 tokens, eight strips and the blocks' sums one after another."""
    from hdla_impl_b200 import ssm
    g = gen(W)
    pos = lambda *s, dtype=dtype: (0.5 + torch.rand(*s, generator=g)).to(dtype)  # noqa: E731
    n = B if cu is None else len(cu) - 1
    x, w, b, h0, dy = pos(B, T, D), pos(D, W, dtype=F32), pos(D, dtype=F32), pos(n, W - 1, D), pos(B, T, D)
    own = [w.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)]
    got = torch.autograd.grad(ssm.short_convolution(x.to(dev), *own, initial_state=h0.to(dev), cu_seqlens=cu)[0], own, dy.to(dev))
    ref = [w.double().requires_grad_(True), b.double().requires_grad_(True)]
    want = torch.autograd.grad(orc.short_conv(x.double(), *ref, "silu", h0.double(), cu)[0], ref, dy.double())
    tol = (16 + W + 1 + 128 + 8 + 32 + B * T / 1024) * U
    assert tol < 0.5 / (B * T)
    for k, a, q in zip("wb", got, want):
        entries_close(a, q, q.abs(), tol, "d" + k)
