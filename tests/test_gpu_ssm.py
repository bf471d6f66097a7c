"""GPU: the short convolution, the selective scan and the norms round a block against their fp64 definitions.

Errors are taken relative to the largest value of the tensor.  What they may be: an output of type t is rounded once
(finfo(t).eps / 2); all else is fp32, whose rounding is 2^-24 an operation.  A recurrence of T steps adds about four roundings and an
exponential (2^-22) a step to what it carries, which decays no slower than the state itself: (T + 64) 2^-21 covers it, with the
softplus and the gate.  A sum of n terms of random signs is about sqrt(n) smaller than the terms' magnitudes, to which its error
belongs: sqrt(n) times that."""
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
    ref = ref.detach()
    got = got.detach().cpu().double()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all())
    top = float(ref.abs().max()) if ref.numel() else 0.0
    return float((got - ref).abs().max()) / top if top else (float(got.abs().max()) if got.numel() else 0.0)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, ref, steps, name, terms=1):
    tol = half_step(got.dtype) + (steps + 64) * 2.0 ** -21 * math.sqrt(terms)
    e = off(got, ref)
    assert e <= tol, f"{name}: {e:.3g} > {tol:.3g}"


def run(f, leaves, outs, dev):
    """(outputs, gradients of the leaves) of f(leaves) with the gradients `outs` of the outputs."""
    y = [t for t in f(leaves) if t is not None]
    need = [k for k, t in leaves.items() if t is not None and t.requires_grad]
    live = [(t, o.to(t.device, t.dtype)) for o, t in zip(outs, y) if t.requires_grad]       # (no tokens or no state rows: none)
    g = torch.autograd.grad([t for t, _ in live], [leaves[k] for k in need], [o for _, o in live], allow_unused=True) if live else ()
    return y, dict(zip(need, g))


def both(own, oracle, tensors, outs, dev):
    """The framework's results and the oracle's: outputs and gradients."""
    mine = {k: None if t is None else t.to(dev).requires_grad_(t.is_floating_point()) for k, t in tensors.items()}
    ref = {k: None if t is None else t.double().requires_grad_(t.is_floating_point()) for k, t in tensors.items()}
    return run(own, mine, outs, dev), run(oracle, ref, [o.double() for o in outs], dev)


# --------------------------------------------------------------------------------------------- short convolution
CONV = [
    # B, T, D, W, dtype, weights' type, activation, bias, state, offsets
    (2, 100, 64, 4, BF, BF, "silu", True, True, None),
    (2, 101, 264, 4, F32, F32, "silu", True, True, None),
    (1, 1, 64, 4, BF, BF, "silu", True, True, None),
    (3, 2, 5, 4, BF, F32, "silu", False, True, None),
    (2, 3, 33, 3, F32, F32, None, True, False, None),
    (1, 67, 40, 2, BF, BF, None, False, False, None),
    (2, 9, 24, 1, F32, F32, "silu", True, True, None),
    (2, 37, 12, 5, F32, F32, "silu", True, True, None),
    (1, 300, 100, 8, BF, F32, "silu", True, True, None),
    (1, 60, 64, 4, BF, BF, "silu", True, True, [0, 0, 1, 3, 3, 20, 60]),       # empty ones, shorter than the taps
    (1, 60, 33, 4, F32, F32, "silu", True, True, [0, 0, 4, 36, 36, 50, 50]),   # the last ten rows belong to none; empty at the back
    (1, 45, 20, 7, F32, F32, "silu", True, True, [0, 2, 4, 32, 45, 45]),
    (1, 33, 16, 3, BF, BF, "silu", True, False, [0, 16, 33]),
    (1, 8, 16, 4, F32, F32, "silu", True, True, [0, 0]),                       # nothing at all
]


def conv_own(cu, act, dev):
    from hdla_impl_b200 import ssm
    c = None if cu is None else torch.tensor(cu, device=dev)
    return lambda t: ssm.short_convolution(t["x"], t["w"], t["b"], activation=act, initial_state=t["h0"], output_final_state=True,
                                           cu_seqlens=c)


@pytest.mark.parametrize("B,T,D,W,dtype,wt,act,bias,state,cu", CONV)
def test_short_convolution(dev, B, T, D, W, dtype, wt, act, bias, state, cu):
    g = gen(T + D + W)
    n = B if cu is None else len(cu) - 1
    t = {"x": rn(g, B, T, D, dtype=dtype), "w": rn(g, D, W, dtype=wt, scale=0.5), "b": rn(g, D, dtype=wt) if bias else None,
         "h0": rn(g, n, W - 1, D, dtype=dtype) if state else None}
    outs = [rn(g, B, T, D, dtype=dtype), rn(g, n, W - 1, D, dtype=dtype)]
    (y, gy), (r, gr) = both(conv_own(cu, act, dev), lambda t: orc.short_conv(t["x"], t["w"], t["b"], act, t["h0"], cu), t, outs, dev)
    close(y[0], r[0], 0, "y")
    assert torch.equal(y[1].cpu().double(), r[1].detach()), "the final state is rows of the inputs"
    for k in gr:
        if gr[k] is not None:
            close(gy[k], gr[k], 0, "d" + k, B * T if k in "wb" else 1)


def test_short_convolution_of_slices(dev):
    """x as a slice of a wider projection, and not dense at all."""
    from hdla_impl_b200 import ssm
    g = gen(1)
    w = rn(g, 64, 4, dtype=BF).to(dev)
    for wide, cut in ((rn(g, 2, 50, 192, dtype=BF), slice(64, 128)), (rn(g, 2, 50, 193, dtype=BF), slice(65, 129)),
                      (rn(g, 2, 50, 128, dtype=BF), slice(0, 128, 2))):
        wide = wide.to(dev).requires_grad_(True)
        y, h = ssm.short_convolution(wide[..., cut], w, output_final_state=True)
        x = wide.detach()[..., cut].contiguous().requires_grad_(True)
        y2, h2 = ssm.short_convolution(x, w, output_final_state=True)
        assert torch.equal(y, y2) and torch.equal(h, h2)
        a, = torch.autograd.grad(y, wide, torch.ones_like(y))
        b, = torch.autograd.grad(y2, x, torch.ones_like(y))
        assert torch.equal(a[..., cut], b)


@pytest.mark.parametrize("D,W,dtype", [(64, 4, BF), (33, 4, F32), (5, 3, BF), (40, 8, F32), (8, 1, F32), (264, 2, BF)])
def test_short_convolution_steps_go_on_from_a_prompt(dev, D, W, dtype):
    from hdla_impl_b200 import ssm
    g = gen(D)
    x, w, b = rn(g, 3, 12, D, dtype=dtype).to(dev), rn(g, D, W, dtype=dtype).to(dev), rn(g, D, dtype=dtype).to(dev)
    y, last = ssm.short_convolution(x, w, b, output_final_state=True)
    _, state = ssm.short_convolution(x[:, :7], w, b, output_final_state=True)
    for t in range(7, 12):
        assert torch.equal(ssm.short_convolution_step(x[:, t], state, w, b), y[:, t])
    assert torch.equal(state, last)


def test_taps_that_do_not_exist_are_not_multiplied(dev):
    """Five of the eight taps a kernel has room for: an infinite input reaches five outputs and no more."""
    from hdla_impl_b200 import ssm
    x = torch.ones(1, 20, 4, device=dev)
    x[0, 3] = float("inf")
    y, _ = ssm.short_convolution(x, torch.ones(4, 5, device=dev), activation=None)
    assert bool(torch.isinf(y[0, 3:8]).all()) and bool((y[0, 8:] == 5).all()) and bool(torch.isfinite(y[0, :3]).all())


# --------------------------------------------------------------------------------------------- selective scan
SCAN = [
    # B, T, D, N, G, dtype, parts (z gate, s skip, b bias, p softplus, h state), offsets
    (2, 100, 64, 16, 1, BF, "zsbph", None),
    (2, 101, 72, 16, 1, F32, "zsbph", None),
    (1, 1, 64, 16, 1, BF, "zsbph", None),
    (2, 3, 5, 16, 1, F32, "zsbph", None),
    (1, 40, 48, 1, 1, F32, "zsp", None),
    (1, 40, 48, 5, 2, F32, "zsbph", None),
    (1, 70, 132, 8, 4, F32, "bp", None),
    (1, 70, 130, 20, 2, BF, "zbph", None),
    (1, 33, 33, 33, 3, F32, "zsbph", None),
    (2, 50, 40, 64, 1, BF, "zsbph", None),
    (1, 35, 20, 100, 2, F32, "zsbph", None),
    (1, 35, 24, 128, 1, BF, "zsbph", None),
    (1, 100, 16, 16, 1, F32, "h", None),                          # dt as it is
    (1, 1300, 8, 16, 1, F32, "zsbph", None),                      # a long row of few channels: segments
    (2, 700, 24, 4, 1, BF, "zsbp", None),
    (1, 90, 64, 16, 1, F32, "zsbph", [0, 0, 1, 9, 9, 24, 90]),
    (1, 90, 40, 12, 2, BF, "zsbph", [0, 16, 16, 32, 70, 70]),     # twenty rows of none, ends on tiles' edges, empty at the back
    (1, 1000, 8, 16, 1, F32, "zsbph", [0, 0, 300, 301, 301, 640, 900]),       # segments with several sequences in them
    (1, 1000, 8, 7, 1, F32, "zsbp", [0, 999, 1000, 1000]),
    (1, 40, 8, 16, 1, F32, "zsbph", [0, 0]),
]


def scan_tensors(g, B, T, D, N, G, dtype, parts, n, fast=1.0):
    t = {"x": rn(g, B, T, D, dtype=dtype), "dt": rn(g, B, T, D, dtype=dtype), "A": -torch.exp(rn(g, D, N)) * fast,
         "B": rn(g, B, T, G, N, dtype=dtype), "C": rn(g, B, T, G, N, dtype=dtype),
         "D": rn(g, D) if "s" in parts else None, "z": rn(g, B, T, D, dtype=dtype) if "z" in parts else None,
         "bias": rn(g, D) - 2 if "b" in parts else None, "h0": rn(g, n, D, N) if "h" in parts else None}
    if "p" not in parts:
        t["dt"] = t["dt"].abs() * 0.2
    return t


def scan_own(parts, cu, dev):
    from hdla_impl_b200 import ssm
    c = None if cu is None else torch.tensor(cu, device=dev)
    return lambda t: ssm.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["bias"],
                                        dt_softplus="p" in parts, initial_state=t["h0"], output_final_state=True, cu_seqlens=c)


def scan_ref(parts, cu):
    return lambda t: orc.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], "p" in parts, t["h0"], cu)


def scan_close(got, ref, T, rows, D):
    (y, gy), (r, gr) = got, ref
    close(y[0], r[0], T, "y")
    close(y[1], r[1], T, "final state")
    for k in gr:
        if gr[k] is not None:
            close(gy[k], gr[k], T, "d" + k, rows if k in ("A", "D", "bias") else D if k in "BC" else 1)


@pytest.mark.parametrize("B,T,D,N,G,dtype,parts,cu", SCAN)
def test_selective_scan(dev, B, T, D, N, G, dtype, parts, cu):
    g = gen(T + D + N)
    n = B if cu is None else len(cu) - 1
    t = scan_tensors(g, B, T, D, N, G, dtype, parts, n)
    outs = [rn(g, B, T, D, dtype=dtype), rn(g, n, D, N)]
    got, ref = both(scan_own(parts, cu, dev), scan_ref(parts, cu), t, outs, dev)
    scan_close(got, ref, T, B * T, D)


@pytest.mark.parametrize("fast", [1e-4, 300.0])
def test_selective_scan_of_slow_and_of_fast_decays(dev, fast):
    """Decays near one (the state is a long sum) and decays that underflow within a step."""
    g = gen(5)
    t = scan_tensors(g, 1, 200, 16, 16, 1, F32, "zsbph", 1, fast)
    outs = [rn(g, 1, 200, 16), rn(g, 1, 16, 16)]
    got, ref = both(scan_own("zsbph", None, dev), scan_ref("zsbph", None), t, outs, dev)
    scan_close(got, ref, 200, 200, 16)


def test_small_time_steps_keep_their_digits(dev):
    """softplus of large negative values is e^v: the steps and their gradients are right to fp32, not to fp32 of one."""
    from hdla_impl_b200 import ssm
    v = torch.linspace(-30, 30, 512).view(1, 1, 512)
    one = torch.ones(1, 1, 1, 1, device=dev)
    dt = v.to(dev).requires_grad_(True)
    y, _ = ssm.selective_scan(torch.ones(1, 1, 512, device=dev), dt, -torch.ones(512, 1, device=dev), one, one)
    g, = torch.autograd.grad(y, dt, torch.ones_like(y))
    d = v.double()
    want = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))
    # e^v in fp32: v log2 e rounded to 24 bits is off by 2^-25 43 = 1.3e-6 in the exponent at 30, times ln 2; with a few roundings 2e-6
    assert float(((y.cpu().double() - want) / want).abs().max()) < 2e-6
    slope = 1 / (1 + torch.exp(-d))
    assert float(((g.cpu().double() - slope) / slope).abs().max()) < 2e-6


def test_selective_scan_of_slices_and_shared_groups(dev):
    """x and z as halves of one projection, dt, B and C as slices of another, B and C with and without the group's dimension."""
    from hdla_impl_b200 import ssm
    for D, N in ((64, 16), (40, 6), (33, 5)):
        g = gen(D)
        xz = rn(g, 2, 60, 2 * D, dtype=BF).to(dev).requires_grad_(True)
        dbc = rn(g, 2, 60, D + 2 * N, dtype=BF).to(dev).requires_grad_(True)
        A = -torch.exp(rn(g, D, N)).to(dev)

        def f(xz, dbc, dense, groups):
            t = [xz[..., :D], dbc[..., :D], dbc[..., D:D + N], dbc[..., D + N:], xz[..., D:]]
            t = [v.contiguous() for v in t] if dense else t
            if groups:
                t[2], t[3] = t[2].unsqueeze(2), t[3].unsqueeze(2)
            y, h = ssm.selective_scan(*t[:2], A, *t[2:4], z=t[4], output_final_state=True)
            return [y, h, *torch.autograd.grad([y, h], [xz, dbc], [torch.ones_like(y), torch.ones_like(h)])]

        want = f(xz, dbc, True, True)
        for dense, groups in ((False, True), (False, False), (True, False)):
            for a, b in zip(f(xz, dbc, dense, groups), want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("B,D,N,G,dtype,parts", [(3, 64, 16, 1, BF, "zsbp"), (2, 33, 5, 3, F32, "zsbp"), (9, 4096, 16, 1, BF, "zsbp"),
                                                 (1, 20, 128, 2, F32, "p"), (5, 7, 1, 1, BF, "zb"), (70, 520, 64, 2, F32, "zsbp")])
def test_selective_scan_steps_go_on_from_a_prompt(dev, B, D, N, G, dtype, parts):
    from hdla_impl_b200 import ssm
    g = gen(D + N)
    t = {k: None if v is None else v.to(dev) for k, v in scan_tensors(g, B, 9, D, N, G, dtype, parts, B).items()}
    opt = dict(D=t["D"], dt_bias=t["bias"], dt_softplus="p" in parts)
    cut = lambda a, b: [None if t[k] is None else t[k][:, a:b] for k in ("x", "dt", "B", "C", "z")]  # noqa: E731
    x, dt, Bm, Cm, z = cut(0, 9)
    y, last = ssm.selective_scan(x, dt, t["A"], Bm, Cm, z=z, output_final_state=True, **opt)
    x, dt, Bm, Cm, z = cut(0, 6)
    _, state = ssm.selective_scan(x, dt, t["A"], Bm, Cm, z=z, output_final_state=True, **opt)
    for i in range(6, 9):
        x, dt, Bm, Cm, z = [None if v is None else v[:, 0] for v in cut(i, i + 1)]
        yt = ssm.selective_scan_step(x, dt, t["A"], Bm, Cm, state, z=z, **opt)
        close(yt, y[:, i].cpu().double(), 9, "y")
        if dtype == BF:           # both sides are rounded
            assert off(yt, y[:, i].cpu().double()) <= 2 * half_step(BF)
    close(state, last.cpu().double(), 9, "state")


def test_only_the_final_state_or_only_some_inputs_need_gradients(dev):
    from hdla_impl_b200 import ssm
    g = gen(3)
    t = {k: None if v is None else v.to(dev) for k, v in scan_tensors(g, 2, 30, 16, 8, 1, F32, "zsbph", 2).items()}
    t["A"].requires_grad_(True)
    y, h = scan_own("zsbph", None, dev)(t)
    dht = torch.ones_like(h)
    a, = torch.autograd.grad(h, t["A"], dht, retain_graph=True)
    b, = torch.autograd.grad([y, h], t["A"], [torch.zeros_like(y), dht], retain_graph=True)
    assert torch.equal(a, b)
    c, = torch.autograd.grad(y, t["A"], torch.ones_like(y))
    d, = torch.autograd.grad(scan_own("zsbph", None, dev)(t)[0], t["A"], torch.ones_like(y))
    assert torch.equal(c, d)
    w = rn(g, 16, 4).to(dev).requires_grad_(True)
    y, h = ssm.short_convolution(t["x"], w, output_final_state=True)
    assert h.requires_grad and float(torch.autograd.grad(h, w, torch.ones_like(h))[0].abs().max()) == 0


def test_gradients_against_differences(dev):
    """Directional central differences of the fp32 forward.  With a step of e the difference is off by e^2 times a third derivative
    of order one and by the outputs' rounding, about 2^-20 of their size over e: e = 2^-6 leaves 2^-12 + 2^-14; 1e-2 is asked for."""
    from hdla_impl_b200 import layer_ops, ssm
    g = gen(11)
    t = scan_tensors(g, 1, 40, 8, 4, 2, F32, "zsbph", 1)
    t = {k: v.to(dev) for k, v in t.items()}
    conv = {"x": rn(g, 1, 40, 8).to(dev), "w": rn(g, 8, 4).to(dev), "b": rn(g, 8).to(dev), "h0": rn(g, 1, 3, 8).to(dev)}
    norm = {k: rn(g, 1, 40, 8).to(dev) for k in ("x", "r", "g")} | {k: rn(g, 8).to(dev) for k in ("v", "p", "n")}
    fs = ((scan_own("zsbph", None, dev), t),
          (lambda c: ssm.short_convolution(c["x"], c["w"], c["b"], initial_state=c["h0"], output_final_state=True), conv),
          (lambda c: layer_ops.rms_norm_residual(c["x"], c["r"], gate=c["g"], scale=c["v"], post_weight=c["p"], pre_weight=c["n"]), norm))
    for f, x in fs:
        outs = [torch.randn(o.shape, generator=g).to(dev) for o in f(x)]
        leaves = {k: v.clone().requires_grad_(True) for k, v in x.items()}
        grads = torch.autograd.grad(f(leaves), list(leaves.values()), outs)
        for (k, v), d in zip(x.items(), grads):
            way = torch.randn(v.shape, generator=g).to(dev)
            e = 2.0 ** -6
            far = [sum(float((o.double() * c.double()).sum()) for o, c in zip(f({**x, k: v + s * e * way}), outs)) for s in (1, -1)]
            want, got = (far[0] - far[1]) / (2 * e), float((d.double() * way.double()).sum())
            size = float(d.double().norm() * way.double().norm()) / math.sqrt(d.numel()) + 1e-3
            assert abs(want - got) <= 1e-2 * max(size, abs(got)), (k, want, got)


# --------------------------------------------------------------------------------------------- norms
NORM = [
    # rows, D, type, residual's type, weights' type, parts (r residual, g gate, p norm after, n norm before, v scale vector), gate's activation
    ((3, 37), 2048, BF, BF, BF, "rgpnv", "sigmoid"),
    ((700,), 64, F32, F32, F32, "rgpnv", "silu"),
    ((5,), 4096, BF, F32, F32, "rgpn", "sigmoid"),
    ((3,), 8192, BF, BF, BF, "rgpnv", None),
    ((2,), 8192, F32, F32, F32, "rgpnv", "silu"),
    ((9,), 1000, F32, F32, F32, "rnv", None),
    ((11,), 1001, BF, F32, BF, "rgpnv", "sigmoid"),
    ((4, 3), 7, F32, F32, F32, "rgpnv", "sigmoid"),
    ((1,), 3, F32, F32, F32, "rpn", None),
    ((1,), 520, BF, BF, BF, "p", None),
    ((2, 2), 300, BF, BF, F32, "gn", "silu"),
    ((600,), 768, BF, BF, BF, "", None),
    ((1300,), 256, BF, BF, BF, "rgpnv", "sigmoid"),
    ((50,), 5000, F32, F32, BF, "rgpnv", "sigmoid"),
]


@pytest.mark.parametrize("rows,D,dtype,rt,wt,parts,act", NORM)
def test_rms_norm_residual(dev, rows, D, dtype, rt, wt, parts, act):
    from hdla_impl_b200 import layer_ops
    g = gen(D)
    has = lambda k, *s, **kw: rn(g, *s, **kw) if k in parts else None  # noqa: E731
    t = {"x": rn(g, *rows, D, dtype=dtype), "r": has("r", *rows, D, dtype=rt), "g": has("g", *rows, D, dtype=dtype),
         "v": has("v", D, dtype=wt), "p": has("p", D, dtype=wt), "n": has("n", D, dtype=wt)}
    outs = [rn(g, *rows, D, dtype=rt if "r" in parts else dtype), rn(g, *rows, D, dtype=dtype)]
    scale = lambda t: 0.5 if t["v"] is None else t["v"]  # noqa: E731
    own = lambda t: layer_ops.rms_norm_residual(t["x"], t["r"], gate=t["g"], scale=scale(t), post_weight=t["p"], pre_weight=t["n"],  # noqa: E731
                                                gate_act=act, eps=1e-5)
    ref = lambda t: orc.norm_residual(t["x"], t["r"], t["g"], scale(t), t["p"], t["n"], act, 1e-5)  # noqa: E731
    (y, gy), (r, gr) = both(own, ref, t, outs, dev)
    assert len(y) == len(r) == 1 + ("n" in parts)
    # a row's sums add D roundings of random sign to their terms: 64 + sqrt(D) steps cover them
    steps = math.sqrt(D)
    for k, (a, b) in enumerate(zip(y, r)):
        close(a, b, steps, "ru"[k])
    for k in gr:
        # a gradient through a norm is the difference of terms of like size, a few times larger than it: 8
        close(gy[k], gr[k], 8 * (steps + 64), "d" + k, math.prod(rows) if k in "vpn" else 1)


def test_norms_of_rows_of_zeros(dev):
    from hdla_impl_b200 import layer_ops
    for eps in (1e-5, 1e-12):
        x = torch.zeros(300, 64, device=dev, requires_grad=True)
        w = torch.ones(64, device=dev, requires_grad=True)
        r, u = layer_ops.rms_norm_residual(x, torch.zeros_like(x), post_weight=w, pre_weight=w, eps=eps)
        assert float(r.abs().max()) == 0 and float(u.abs().max()) == 0
        gx, gw = torch.autograd.grad([r, u], [x, w], [torch.zeros_like(r)] * 2)
        assert float(gx.abs().max()) == 0 and float(gw.abs().max()) == 0


# --------------------------------------------------------------------------------------------- together
def block_weights(g, D, N, R, W, dev, dtype):
    w = {"in": rn(g, 2 * D, D, scale=D ** -0.5), "conv": rn(g, D, W, scale=0.5), "cb": rn(g, D, scale=0.1),
         "bcd": rn(g, 2 * N + R, D, scale=D ** -0.5), "dtw": rn(g, D, R, scale=R ** -0.5), "out": rn(g, D, D, scale=D ** -0.5),
         "post": 1 + rn(g, D, scale=0.1), "pre": 1 + rn(g, D, scale=0.1), "first": 1 + rn(g, D, scale=0.1)}
    w = {k: v.to(dtype) for k, v in w.items()}
    w.update(A=-torch.exp(rn(g, D, N)), D=rn(g, D), bias=rn(g, D) - 2)
    return {k: v.to(dev) for k, v in w.items()}


def block(w, x, N, R, conv, scan, norm):
    """norm before -> projection -> convolution -> scan -> projection -> norm after, residual, next norm before."""
    D = x.shape[-1]
    u = norm(x, None, w["first"], None)
    xz = u @ w["in"].t()
    c = conv(xz[..., :D])
    bcd = c @ w["bcd"].t()
    y = scan(c, bcd[..., 2 * N:] @ w["dtw"].t(), bcd[..., :N], bcd[..., N:2 * N], xz[..., D:])
    return norm(y @ w["out"].t(), x, w["pre"], w["post"])


def test_a_block_trains_like_its_definition(dev):
    from hdla_impl_b200 import layer_ops, ssm
    D, N, R, T = 48, 8, 4, 70
    g = gen(21)
    w = block_weights(g, D, N, R, 4, dev, F32)
    x = rn(g, 2, T, D).to(dev)
    do = [rn(g, 2, T, D).to(dev) for _ in range(2)]

    def own_norm(x, res, pre, post):
        r, u = layer_ops.rms_norm_residual(x, res, post_weight=post, pre_weight=pre, scale=0.5 if res is not None else 1.0)
        return u if res is None else (r, u)

    def ref_norm(x, res, pre, post):
        r, u = orc.norm_residual(x, res, None, 0.5 if res is not None else 1.0, post, pre)
        return u if res is None else (r, u)

    lw = {k: v.clone().requires_grad_(True) for k, v in w.items()}
    lx = x.clone().requires_grad_(True)
    r, u = block(lw, lx, N, R, lambda c: ssm.short_convolution(c, lw["conv"], lw["cb"])[0],
                 lambda c, dt, b, cc, z: ssm.selective_scan(c, dt, lw["A"], b, cc, D=lw["D"], z=z, dt_bias=lw["bias"])[0], own_norm)
    got = [r, u, *torch.autograd.grad([r, u], [lx, *lw.values()], do)]
    dw = {k: v.cpu().double().requires_grad_(True) for k, v in w.items()}
    dx = x.cpu().double().requires_grad_(True)
    r, u = block(dw, dx, N, R, lambda c: orc.short_conv(c, dw["conv"], dw["cb"])[0],
                 lambda c, dt, b, cc, z: orc.selective_scan(c, dt, dw["A"], b[:, :, None], cc[:, :, None], dw["D"], z, dw["bias"])[0], ref_norm)
    want = [r, u, *torch.autograd.grad([r, u], [dx, *dw.values()], [d.cpu().double() for d in do])]
    for name, a, b in zip(["r", "u", "x", *w], got, want):
        # the chain's five stages each add what a recurrence of T steps does
        close(a, b, 5 * T, name, 2 * T if name in w else 1)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_block_decodes_what_it_prefills(dev, dtype):
    """Packed prompts of different lengths, then single tokens, against whole sequences one by one."""
    from hdla_impl_b200 import layer_ops, ssm
    D, N, R, W = 64, 16, 4, 4
    g = gen(31)
    w = block_weights(g, D, N, R, W, dev, dtype)
    lens, more = [5, 1, 33, 17], 4
    seqs = [rn(g, n + more, D, dtype=dtype).to(dev) for n in lens]

    def norm(x, res, pre, post):
        r, u = layer_ops.rms_norm_residual(x, res, post_weight=post, pre_weight=pre, scale=0.5 if res is not None else 1.0)
        return u if res is None else r

    kw = dict(D=w["D"], dt_bias=w["bias"])
    state = {}

    def conv_all(cu):
        def f(c):
            y, state["conv"] = ssm.short_convolution(c, w["conv"], w["cb"], output_final_state=True, cu_seqlens=cu)
            return y
        return f

    def scan_all(cu):
        def f(c, dt, b, cc, z):
            y, state["scan"] = ssm.selective_scan(c, dt, w["A"], b, cc, z=z, output_final_state=True, cu_seqlens=cu, **kw)
            return y
        return f

    with torch.no_grad():
        whole = [block(w, s[None], N, R, conv_all(None), scan_all(None), norm)[0] for s in seqs]
        ends = [sum(lens[:i]) for i in range(len(lens) + 1)]
        packed = block(w, torch.cat([s[:n] for s, n in zip(seqs, lens)])[None], N, R, conv_all(ends), scan_all(ends), norm)[0]
        tol = (4 if dtype == BF else 0) * half_step(dtype) + (40 * 5 + 64) * 2.0 ** -21     # four stages round to bf16 on each side
        for i, n in enumerate(lens):
            assert off(packed[ends[i]:ends[i + 1]], whole[i][:n].cpu().double()) <= 2 * tol
        for t in range(more):
            x = torch.stack([s[n + t] for s, n in zip(seqs, lens)])
            y = block(w, x, N, R, lambda c: ssm.short_convolution_step(c, state["conv"], w["conv"], w["cb"]),
                      lambda c, dt, b, cc, z: ssm.selective_scan_step(c, dt, w["A"], b, cc, state["scan"], z=z, **kw), norm)
            want = torch.stack([o[n + t] for o, n in zip(whole, lens)])
            assert off(y, want.cpu().double()) <= 2 * tol


def all_ops(dev, dtype=BF, T=300, D=64):
    """A training pass through the three operators: (tensors it reads, function)."""
    from hdla_impl_b200 import layer_ops, ssm
    g = gen(7)
    t = {k: v.to(dev) for k, v in scan_tensors(g, 1, T, D, 16, 1, dtype, "zsbph", 3).items()}
    t["w"], t["p"] = rn(g, D, 4, dtype=dtype).to(dev), rn(g, D, dtype=dtype).to(dev)
    cu = torch.tensor([0, 40, 40, T - 20], device=dev)
    do = rn(g, 1, T, D, dtype=dtype).to(dev)
    for v in t.values():
        v.requires_grad_(True)

    def f():
        c, hc = ssm.short_convolution(t["x"], t["w"], output_final_state=True, cu_seqlens=cu)
        y, hs = ssm.selective_scan(c, t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["bias"], initial_state=t["h0"],
                                   output_final_state=True, cu_seqlens=cu)
        r, u = layer_ops.rms_norm_residual(y, t["x"], gate=t["z"], scale=t["p"], post_weight=t["p"], pre_weight=t["p"])
        return [hc, hs, r, u, *torch.autograd.grad([r, u, hs], list(t.values()), [do, do, torch.ones_like(hs)])]

    return t, cu, f


def test_the_same_call_gives_the_same_bits_and_streams_do_not_mix(dev):
    _, _, f = all_ops(dev)
    want = f()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            got.append(f())
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_a_training_pass_is_captured_and_replayed_on_new_inputs(dev):
    t, cu, f = all_ops(dev)
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        for _ in range(2):
            f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = f()
    with torch.no_grad():
        t["x"].normal_()
        t["B"].normal_()
        cu.copy_(torch.tensor([0, 0, 190, 300], device=dev))
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in out]
    for a, b in zip(got, f()):
        assert torch.equal(a, b)


def test_single_tokens_are_captured_and_replayed(dev):
    """A decode step in a graph moves the states on at every replay, as the calls themselves do."""
    from hdla_impl_b200 import layer_ops, ssm
    g = gen(13)
    B, D, N = 5, 72, 16
    t = {k: v.to(dev) for k, v in scan_tensors(g, B, 1, D, N, 1, BF, "zsbp", B).items() if v is not None}
    w = rn(g, D, 4, dtype=BF).to(dev)
    x, dt, z, Bm, Cm = (t[k][:, 0].clone() for k in ("x", "dt", "z", "B", "C"))
    states = [[torch.zeros(B, 3, D, dtype=BF, device=dev), torch.zeros(B, D, N, device=dev)] for _ in range(2)]

    def f(conv, scan):
        c = ssm.short_convolution_step(x, conv, w)
        y = ssm.selective_scan_step(c, dt, t["A"], Bm, Cm, scan, D=t["D"], z=z, dt_bias=t["bias"])
        return layer_ops.rms_norm_residual(y, x, pre_weight=w[:, 0])[1]

    side = torch.cuda.Stream(dev)
    with torch.no_grad(), torch.cuda.stream(side):
        f(*[s.clone() for s in states[0]])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=side):
        out = f(*states[0])
    for i in range(4):
        x.copy_(rn(g, B, D, dtype=BF))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(f(*states[1]), out)
    for a, b in zip(*states):
        assert torch.equal(a, b)


def test_an_eager_graph_that_lives_on_does_not_disturb_a_captured_backward(dev):
    """The leaves' eager graph (made on the capturing stream, as a training loop makes it) is kept while a backward pass of the same
    leaves is captured, and used after that."""
    from hdla_impl_b200 import ssm
    t, cu, f = all_ops(dev)
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        f()
        kept, _ = ssm.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], z=t["z"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = f()
    graph.replay()
    with torch.cuda.stream(side):
        a, = torch.autograd.grad(kept, t["A"], torch.ones_like(kept))
        y, _ = ssm.selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], z=t["z"])
        b, = torch.autograd.grad(y, t["A"], torch.ones_like(y))
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for p, q in zip(out, f()):
        assert torch.equal(p, q)


def test_offsets_that_make_no_sense_stay_inside_the_tensors(dev):
    """A device tensor of offsets is not looked at by the host: those outside 0..T are cut, those that fall back end at once."""
    from hdla_impl_b200 import ssm
    x = torch.randn(1, 50, 16, device=dev)
    a = ssm.short_convolution(x, torch.ones(16, 4, device=dev), cu_seqlens=torch.tensor([0, 20, 1000], device=dev))[0]
    b = ssm.short_convolution(x, torch.ones(16, 4, device=dev), cu_seqlens=[0, 20, 50])[0]
    assert torch.equal(a, b)
    bc = torch.randn(1, 50, 4, device=dev)
    A = -torch.ones(16, 4, device=dev)
    a = ssm.selective_scan(x, x, A, bc, bc, cu_seqlens=torch.tensor([0, 20, 1000], device=dev))[0]
    b = ssm.selective_scan(x, x, A, bc, bc, cu_seqlens=[0, 20, 50])[0]
    assert torch.equal(a, b)


def test_rows_of_no_sequence_may_hold_anything(dev):
    """NaN and infinities behind the last offset, as memory that was never written holds them, reach nothing."""
    from hdla_impl_b200 import ssm
    g = gen(9)
    for T, end in ((61, 40), (700, 330)):                          # within a tile of tokens; in segments of their own
        cu = torch.tensor([0, 13, end], device=dev)
        t = {k: v.to(dev) for k, v in scan_tensors(g, 1, T, 24, 16, 2, F32, "zsbph", 2).items()}
        t["w"] = rn(g, 24, 4).to(dev)
        dy = rn(g, 1, T, 24).to(dev)

        def f(t, dy):
            leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
            c, hc = ssm.short_convolution(leaves["x"], leaves["w"], output_final_state=True, cu_seqlens=cu)
            y, hs = ssm.selective_scan(leaves["x"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], D=leaves["D"], z=leaves["z"],
                                       dt_bias=leaves["bias"], initial_state=leaves["h0"], output_final_state=True, cu_seqlens=cu)
            return [c, hc, y, hs, *torch.autograd.grad([c, hc, y, hs], list(leaves.values()), [dy, hc, dy, hs])]

        clean = {k: v.clone() for k, v in t.items()}
        for k in ("x", "dt", "z", "B", "C"):
            clean[k][:, end:] = 0
            t[k][:, end:] = float("nan")
            t[k][:, end + 1] = float("inf")
        cleandy = dy.clone()
        cleandy[:, end:] = 0
        dy[:, end:] = float("nan")
        for a, b in zip(f(t, dy), f(clean, cleandy)):
            assert torch.equal(a, b)


def test_a_sequences_nan_stays_in_it(dev):
    """A NaN in one packed sequence leaves the others' outputs, states and row gradients alone."""
    from hdla_impl_b200 import ssm
    g = gen(10)
    ends = [0, 30, 75, 75, 300]
    cu = torch.tensor(ends, device=dev)
    t = {k: v.to(dev) for k, v in scan_tensors(g, 1, 300, 16, 5, 1, F32, "zsbph", 4).items()}
    t["w"] = rn(g, 16, 4).to(dev)

    def f(t):
        leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
        c, hc = ssm.short_convolution(leaves["x"], leaves["w"], output_final_state=True, cu_seqlens=cu)
        y, hs = ssm.selective_scan(leaves["x"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], D=leaves["D"], z=leaves["z"],
                                   dt_bias=leaves["bias"], initial_state=leaves["h0"], output_final_state=True, cu_seqlens=cu)
        rows = ["x", "dt", "B", "C", "z", "h0"]
        return [c, y, hc, hs], torch.autograd.grad([c, y, hs], [leaves[k] for k in rows], [torch.ones_like(c), torch.ones_like(y), torch.ones_like(hs)])

    want = f(t)
    bad = {k: v.clone() for k, v in t.items()}
    bad["x"][0, 40] = float("nan")
    got = f(bad)
    keep = torch.ones(300, dtype=torch.bool, device=dev)
    keep[30:75] = False
    for a, b in zip(got[0][:2] + list(got[1][:5]), want[0][:2] + list(want[1][:5])):
        assert torch.equal(a[0, keep], b[0, keep])
    for a, b in zip([*got[0][2:], got[1][5]], [*want[0][2:], want[1][5]]):
        assert torch.equal(a[[0, 2, 3]], b[[0, 2, 3]])
    assert bool(torch.isnan(got[0][3][1]).all())


def test_shares_of_many_states_take_turns(dev):
    """128 states and 512 channels: the tiles of four channels share the 1 GiB for their shares of dB and dC, in several launches."""
    from hdla_impl_b200 import ssm
    g = gen(12)
    T, D, N = 4500, 512, 128
    t = {k: None if v is None else v.to(dev) for k, v in scan_tensors(g, 2, T, D, N, 1, BF, "p", 2).items()}
    dy = rn(g, 2, T, D, dtype=BF).to(dev)

    def f(rows):
        leaves = {k: (v if k == "A" else v[rows]).clone().requires_grad_(True) for k, v in t.items() if v is not None}
        y, _ = ssm.selective_scan(leaves["x"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"])
        return torch.autograd.grad(y, list(leaves.values()), dy[rows])

    whole, parts = f(slice(0, 2)), [f(slice(i, i + 1)) for i in range(2)]
    for name, a, b, c in zip(("x", "dt", "A", "B", "C"), whole, *parts):
        if name == "A":
            close(a, (b.double() + c.double()).cpu(), T, name, 2 * T)
        else:
            # the same sums in fp32 in another order, then rounded on both sides: two half steps more
            e = off(a, torch.cat([b, c]).cpu().double())
            assert e <= 2 * half_step(BF) + T * 2.0 ** -21, (name, e)


def test_checkpointing_and_subclasses(dev):
    """Recomputation gives the same bits; a tensor subclass takes the Python route and gives them too."""
    from torch.utils.checkpoint import checkpoint
    from hdla_impl_b200 import layer_ops, ssm

    class Mine(torch.Tensor):
        pass

    g = gen(2)
    t = {k: v.to(dev).requires_grad_(True) for k, v in scan_tensors(g, 2, 40, 16, 8, 1, BF, "zsbph", 2).items()}
    w = rn(g, 16, 4, dtype=BF).to(dev).requires_grad_(True)

    def f(x):
        c, _ = ssm.short_convolution(x, w)
        y, _ = ssm.selective_scan(c, t["dt"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], dt_bias=t["bias"], initial_state=t["h0"])
        return layer_ops.rms_norm_residual(y, x, gate=t["z"], pre_weight=w[:, 0], post_weight=w[:, 1])[1]

    need = [t["x"], t["A"], t["B"], t["h0"], w]
    plain = f(t["x"])
    want = torch.autograd.grad(plain, need, torch.ones_like(plain))
    again = checkpoint(f, t["x"], use_reentrant=False)
    for a, b in zip(torch.autograd.grad(again, need, torch.ones_like(plain)), want):
        assert torch.equal(a, b)
    sub = f(t["x"].as_subclass(Mine))
    for a, b in zip(torch.autograd.grad(sub, need, torch.ones_like(plain)), want):
        assert torch.equal(a.as_subclass(torch.Tensor), b)


def test_a_saved_input_that_was_changed_is_an_error(dev):
    from hdla_impl_b200 import ssm
    x = torch.randn(1, 8, 16, device=dev)
    w = torch.randn(16, 4, device=dev, requires_grad=True)
    y, _ = ssm.short_convolution(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, torch.ones_like(y))
    state = torch.zeros(1, 3, 16, device=dev)
    y, _ = ssm.short_convolution(x, w, initial_state=state)
    ssm.short_convolution_step(x[:, 0], state, w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, torch.ones_like(y))


def test_refusals(dev):
    from hdla_impl_b200 import layer_ops, ssm
    z = lambda *s, t=F32: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    x, w = z(2, 5, 8), z(8, 4)
    conv, scan, norm = ssm.short_convolution, ssm.selective_scan, layer_ops.rms_norm_residual
    bc, A = z(2, 5, 1, 4), z(8, 4)
    bad = [
        (ValueError, lambda: conv(x[0], w)), (ValueError, lambda: conv(x, z(7, 4))), (ValueError, lambda: conv(x, z(8, 9))),
        (ValueError, lambda: conv(x, z(8, 0))), (ValueError, lambda: conv(z(2, 0, 8), w)), (ValueError, lambda: conv(x, w, z(7))),
        (ValueError, lambda: conv(x, w, activation="relu")), (ValueError, lambda: conv(x, w, initial_state=z(2, 4, 8))),
        (TypeError, lambda: conv(x, w, initial_state=z(2, 3, 8, t=BF))), (TypeError, lambda: conv(x.half(), w)),
        (ValueError, lambda: conv(x, w, cu_seqlens=[0, 5])), (ValueError, lambda: conv(x[:1], w, cu_seqlens=[0, 6])),
        (ValueError, lambda: conv(x[:1], w, cu_seqlens=[1, 5])), (ValueError, lambda: conv(x[:1], w, cu_seqlens=[0, 4, 3])),
        (ValueError, lambda: conv(x[:1], w, cu_seqlens=[0])), (ValueError, lambda: conv(x[:1], w, cu_seqlens=z(2))),
        (RuntimeError, lambda: conv(x.cpu(), w)), (RuntimeError, lambda: conv(x, w.cpu())),
        (ValueError, lambda: ssm.short_convolution_step(x[:, 0], z(2, 8, 3).transpose(1, 2), w)),
        (RuntimeError, lambda: ssm.short_convolution_step(x[:, 0], z(2, 3, 8), w.clone().requires_grad_(True))),
        (ValueError, lambda: ssm.short_convolution_step(x, z(2, 3, 8), w)),
        (ValueError, lambda: scan(x, x[:, :4], A, bc, bc)), (ValueError, lambda: scan(x, x, z(7, 4), bc, bc)),
        (ValueError, lambda: scan(x, x, z(8, 129), z(2, 5, 129), z(2, 5, 129))), (ValueError, lambda: scan(x, x, A, z(2, 5, 3, 4), z(2, 5, 3, 4))),
        (ValueError, lambda: scan(x, x, A, bc, z(2, 5, 2, 4))), (ValueError, lambda: scan(x, x, A, bc, bc, D=z(7))),
        (ValueError, lambda: scan(x, x, A, bc, bc, initial_state=z(1, 8, 4))), (TypeError, lambda: scan(x, x.bfloat16(), A, bc, bc)),
        (TypeError, lambda: scan(x, x, A.int(), bc, bc)), (ValueError, lambda: scan(x, x, A, bc, bc, z=x[:1])),
        (ValueError, lambda: scan(x, x, A, bc, bc, cu_seqlens=[0, 5])), (RuntimeError, lambda: scan(x, x, A.cpu(), bc, bc)),
        (ValueError, lambda: ssm.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], z(2, 8, 4, t=BF))),
        (RuntimeError, lambda: ssm.selective_scan_step(x[:, 0], x[:, 0], A.clone().requires_grad_(True), bc[:, 0], bc[:, 0], z(2, 8, 4))),
        (ValueError, lambda: norm(x, x[:1])), (ValueError, lambda: norm(z(2, 8193))), (ValueError, lambda: norm(x, gate=x[:1])),
        (ValueError, lambda: norm(x, pre_weight=z(7))), (TypeError, lambda: norm(x.bfloat16(), gate=x)), (TypeError, lambda: norm(x, x.bfloat16())),
        (ValueError, lambda: norm(x, gate=x, gate_act="relu")), (ValueError, lambda: norm(z(0, 8))), (RuntimeError, lambda: norm(x, x.cpu())),
        (TypeError, lambda: norm(x, scale=None)),
    ]
    for kind, f in bad:
        with pytest.raises(kind):
            f()
    torch.cuda.synchronize()


def test_offsets_beyond_32_bits(dev):
    """More than 2^31 elements: the last rows are where they should be."""
    from hdla_impl_b200 import layer_ops, ssm
    T, D = (1 << 31) // 4096 + 5, 4096
    x = torch.zeros(1, T, D, dtype=BF, device=dev)
    x[0, -3:] = torch.randn(3, D, generator=gen(1)).to(BF).to(dev)
    w = torch.randn(D, 4, generator=gen(2)).to(BF).to(dev)
    with torch.no_grad():
        y, _ = ssm.short_convolution(x, w)
        assert torch.equal(y[:, -3:], ssm.short_convolution(x[:, -6:], w)[0][:, -3:])
        r, u = layer_ops.rms_norm_residual(x, y, pre_weight=w[:, 0], post_weight=w[:, 1])
        r2, u2 = layer_ops.rms_norm_residual(x[:, -3:], y[:, -3:], pre_weight=w[:, 0], post_weight=w[:, 1])
        assert torch.equal(r[:, -3:], r2) and torch.equal(u[:, -3:], u2)
        del r, u
        bc = torch.ones(1, T, 4, dtype=BF, device=dev)
        A = -torch.ones(D, 4, device=dev)
        y, h = ssm.selective_scan(x, x, A, bc, bc, dt_softplus=False, output_final_state=True)
        y2, h2 = ssm.selective_scan(x[:, -3:], x[:, -3:], A, bc[:, -3:], bc[:, -3:], dt_softplus=False, output_final_state=True)
        assert torch.equal(y[:, -3:], y2) and torch.equal(h, h2)
