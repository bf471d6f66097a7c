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
