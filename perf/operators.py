"""Performance cases of the selective state space mixer and of the norms round a block.

What a training or serving program calls for one token-mixing block next to the delta rule: the short causal convolution
(``ssm.short_convolution`` and its single-token step), the selective scan (``ssm.selective_scan`` and its step), and the RMS
norms after and before a block fused with gate, residual scale and residual sum (``layer_ops.rms_norm_residual``).

Keys of a case
    op       "conv" / "scan" / "norm"
    mode     "step"   one token for each of B running sequences, the state updated in place
             "infer"  forward without gradients; from an initial state to a final state where ``h0``
             "train"  forward and backward, all gradients
    B,T,D    sequences, tokens, channels (``seqs`` > 0: B = 1 and T packed tokens of that many sequences)
    N,G      states of a channel, groups of channels that share B and C (scan)
    W        taps (conv)
    dtype    "bf16" / "fp32" of the activations.  A, D, dt_bias and the recurrent state are fp32; other weights are like x
    parts    which of the optional inputs a case has: conv "b" bias; scan "z" gate, "s" skip D;
             norm "r" residual, "p" norm after the block, "g" gate, "n" norm before the next block, "v" scale per channel
"""
import math
import random

import torch

own = False
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def _case(op, mode, B, T, D, dtype="bf16", *, N=0, G=0, W=0, seqs=0, h0=False, parts="", name=None):
    c = dict(op=op, mode=mode, B=B, T=T, D=D, N=N, G=G, W=W, dtype=dtype, seqs=seqs, h0=h0, parts=parts)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one token of a full serving batch through the convolution: 32 heads of 128 channels, as the decode configuration
        _case("conv", "step", 256, 1, 4096, W=4, parts="b", name="conv_step_b256"),
        # a server's batch of prompts of different lengths, packed, with carried states
        _case("conv", "infer", 1, 16411, 2048, W=4, seqs=24, h0=True, parts="b", name="conv_packed"),
        # the headline training batch: 16 heads of 128 channels
        _case("conv", "train", 8, 4096, 2048, W=4, parts="b", name="conv_train_b8_t4096"),
        # one token for each of a handful of running conversations: what an interactive server does per token and layer
        _case("scan", "step", 4, 1, 2048, N=16, G=1, parts="zs", name="scan_step_b4"),
        # one token of a full serving batch
        _case("scan", "step", 256, 1, 4096, N=16, G=1, parts="zs", name="scan_step_b256"),
        # the prompts of a server's batch, packed, of odd lengths
        _case("scan", "infer", 1, 16411, 2048, N=16, G=1, seqs=24, h0=True, parts="zs", name="scan_packed"),
        # one long document: few channels, so the time axis has to be split
        _case("scan", "infer", 1, 65536, 2048, N=16, G=1, parts="zs", name="scan_t65536"),
        # a full precision run of a small model, odd lengths, several groups
        _case("scan", "train", 2, 1000, 768, "fp32", N=16, G=4, h0=True, parts="zs", name="scan_train_fp32"),
        # the headline training batch
        _case("scan", "train", 8, 4096, 2048, N=16, G=1, parts="zs", name="scan_train_b8_t4096"),
        # the rows of a decode step
        _case("norm", "infer", 16, 1, 2048, parts="rpgn", name="norm_decode_b16"),
        # odd width, no gate: a pre-norm block in full precision
        _case("norm", "train", 3, 1001, 1000, "fp32", parts="rnv", name="norm_train_fp32"),
        # the headline training batch
        _case("norm", "train", 8, 4096, 2048, parts="rpgnv", name="norm_train_b8_t4096"),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _some(rng, letters):
    return "".join(x for x in letters if rng.random() < 0.7)


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    mode = rng.choice(["step", "infer", "train"]) if op != "norm" else rng.choice(["infer", "train"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    h0 = rng.random() < 0.5
    if op == "norm":
        D = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)])
        return _case("norm", mode, _log(rng, 1, 8), _log(rng, 1, 2 ** 25 // D // 8), D, dtype, parts=_some(rng, "rpgnv"))
    D = rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 1, 64), 128 * _log(rng, 1, 32)])
    N = rng.choice([16, 16, 16, 8, 32, _log(rng, 1, 64)]) if op == "scan" else 0
    G = rng.choice([1, 1, 2, 4]) if op == "scan" else 0
    D = max(G, D - D % G) if G else D
    W = rng.choice([4, 4, 3, 2]) if op == "conv" else 0
    parts = _some(rng, "zs" if op == "scan" else "b")
    if mode == "step":
        return _case(op, "step", _log(rng, 1, 256), 1, D, dtype, N=N, G=G, W=W, parts=parts)
    most = 2 ** 25 // D if op == "conv" else 2 ** 28 // (D * max(N, 8))       # tokens
    if rng.random() < 0.4:
        n = _log(rng, 2, 32)
        return _case(op, mode, 1, max(4 * n, min(65536, _log(rng, 64, most))), D, dtype, N=N, G=G, W=W, seqs=n, h0=h0, parts=parts)
    B = _log(rng, 1, 8)
    return _case(op, mode, B, min(65536, _log(rng, 2, most // B)), D, dtype, N=N, G=G, W=W, h0=h0, parts=parts)


def _offsets(case):
    """Offsets of a packed batch: lengths from a quarter of the mean to about twice it.  They belong to the case."""
    n, T = case["seqs"], case["T"]
    rng = random.Random(1000 * n + T)
    w = [rng.uniform(0.25, 1.75) for _ in range(n)]
    return [int(T * sum(w[:i]) / sum(w)) for i in range(n)] + [T]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt, B, T, D = _DT[case["dtype"]], case["B"], case["T"], case["D"]
    rn = lambda *s, t=dt: torch.randn(*s, generator=g, device=dev).to(t)  # noqa: E731
    ru = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    op, mode, has = case["op"], case["mode"], case["parts"]
    s = {"case": case, "cu": None}
    rows = (B,) if mode == "step" else (B, T)
    n = case["seqs"] or B
    if case["seqs"]:
        s["cu"] = torch.tensor(_offsets(case), device=dev)
    if op == "conv":
        W = case["W"]
        s["x"], s["w"] = rn(*rows, D), (ru(D, W) * 2 - 1).mul_(W ** -0.5).to(dt)
        s["b"] = (ru(D) * 2 - 1).mul_(W ** -0.5).to(dt) if "b" in has else None
        s["h0"] = rn(n, W - 1, D) if case["h0"] or mode == "step" else None
        leaves, dht = ("x", "w", "b", "h0"), lambda: rn(n, W - 1, D)
    elif op == "scan":
        N, G = case["N"], case["G"]
        s["x"], s["B"], s["C"] = rn(*rows, D), rn(*rows, G, N), rn(*rows, G, N)
        s["dt"] = rn(*rows, D, t=torch.float32).mul_(0.5).to(dt)
        # time steps from 1e-3 to 1e-1, decay rates 1 .. N with a learned spread: the layers' usual initialisation
        step = torch.exp(ru(D) * math.log(100.0) + math.log(1e-3))
        s["bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -torch.arange(1, N + 1, device=dev, dtype=torch.float32) * torch.exp(0.2 * rn(D, N, t=torch.float32))
        s["skip"] = 1 + 0.1 * rn(D, t=torch.float32) if "s" in has else None
        s["z"] = rn(*rows, D) if "z" in has else None
        s["h0"] = rn(n, D, N, t=torch.float32) if case["h0"] or mode == "step" else None
        leaves, dht = ("x", "dt", "A", "B", "C", "skip", "z", "bias", "h0"), lambda: rn(n, D, N, t=torch.float32)
    else:
        s["x"] = rn(B, T, D)
        s["r"], s["g"] = (rn(B, T, D) if k in has else None for k in "rg")
        s["p"], s["n"] = ((1 + 0.1 * rn(D, t=torch.float32)).to(dt) if k in has else None for k in "pn")
        s["v"] = (0.5 + 0.1 * rn(D, t=torch.float32)).to(dt) if "v" in has else 0.5
        leaves, dht = ("x", "r", "g", "v", "p", "n"), lambda: rn(B, T, D) if "n" in has else None
    if mode == "train":
        s["dy"] = rn(*s["x"].shape)
        s["dht"] = dht() if case["h0"] or op == "norm" else None
        s["leaves"] = [k for k in leaves if isinstance(s[k], torch.Tensor)]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# --------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from hdla_impl_b200 import layer_ops, ssm
    c = s["case"]
    op, mode = c["op"], c["mode"]
    if op == "conv":
        if mode == "step":
            return [ssm.short_convolution_step(s["x"], s["h0"], s["w"], s["b"], activation="silu"), s["h0"]]
        y, ht = ssm.short_convolution(s["x"], s["w"], s["b"], activation="silu", initial_state=s["h0"],
                                      output_final_state=c["h0"], cu_seqlens=s["cu"])
    elif op == "scan":
        opt = dict(D=s["skip"], z=s["z"], dt_bias=s["bias"], dt_softplus=True)
        if mode == "step":
            return [ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["h0"], **opt), s["h0"]]
        y, ht = ssm.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], **opt, initial_state=s["h0"],
                                   output_final_state=c["h0"], cu_seqlens=s["cu"])
    else:
        y, ht = layer_ops.rms_norm_residual(s["x"], s["r"], gate=s["g"], scale=s["v"], post_weight=s["p"], pre_weight=s["n"],
                                            gate_act="sigmoid", eps=EPS)
    out = [y] if ht is None else [y, ht]
    if mode == "train":
        out = [t.detach() for t in out] + list(torch.autograd.grad(out, [s[k] for k in s["leaves"]],
                                                                   [s["dy"]] if ht is None else [s["dy"], s["dht"]]))
    return out


# --------------------------------------------------------------------------------------------- the plain forms
def _silu_grad(p):
    s = torch.sigmoid(p)
    return s * (1 + p * (1 - s))


def _sequence_of(s, T):
    """(number of the sequence of each of the T tokens, first tokens, ends); lengths of zero are possible."""
    cu = s["cu"]
    seq = torch.searchsorted(cu, torch.arange(T, device=cu.device), right=True) - 1
    return seq, cu[:-1], cu[1:]


def _extended(s, x, h0):
    """The input with W - 1 rows of history before each sequence, packed, and where the tokens stand in it."""
    B, T, D = x.shape
    W = s["case"]["W"]
    n = s["case"]["seqs"] or B
    hist = x.new_zeros(n, W - 1, D) if h0 is None else h0.float()
    if s["cu"] is None:
        return torch.cat([hist, x], 1).reshape(-1, D), (torch.arange(T, device=x.device) + (W - 1)
                                                        + (torch.arange(B, device=x.device) * (T + W - 1))[:, None]).reshape(-1)
    seq, first, end = _sequence_of(s, T)
    at = torch.arange(T, device=x.device) + (W - 1) * (seq + 1)
    ext = x.new_empty(T + n * (W - 1), D)
    ext[at] = x[0]
    rows = first + (W - 1) * torch.arange(n, device=x.device)
    ext[(rows[:, None] + torch.arange(W - 1, device=x.device)).reshape(-1)] = hist.reshape(-1, D)
    return ext, at


def _plain_conv(s):
    c = s["case"]
    W, dt = c["W"], _DT[c["dtype"]]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    b = None if s["b"] is None else s["b"].detach().float()
    h0 = None if s["h0"] is None else s["h0"].detach()
    if c["mode"] == "step":
        ext = torch.cat([h0.float(), x[:, None]], 1)
        p = (ext * w.t()).sum(1)
        p = p if b is None else p + b
        h0.copy_(ext[:, 1:])
        return [(p * torch.sigmoid(p)).to(dt), h0]
    ext, at = _extended(s, x, h0)
    lag = torch.arange(W, device=x.device) - (W - 1)                       # tap j multiplies the input of `lag` rows later
    end = (torch.arange(1, c["B"] + 1, device=x.device) * (c["T"] + W - 1) if s["cu"] is None
           else s["cu"][1:] + (W - 1) * torch.arange(1, c["seqs"] + 1, device=x.device))
    last = (end[:, None] + torch.arange(1 - W, 0, device=x.device)).reshape(-1)
    p = sum(ext[at + lag[j]] * w[:, j] for j in range(W))
    p = p if b is None else p + b
    y = p * torch.sigmoid(p)
    out = [y.reshape(s["x"].shape).to(dt)]
    if c["h0"]:
        out.append(ext[last].reshape(-1, W - 1, c["D"]).to(dt))
    if c["mode"] != "train":
        return out
    dp = s["dy"].float().reshape(p.shape) * _silu_grad(p)
    dext, dw = torch.zeros_like(ext), []
    for j in range(W):
        dext.index_add_(0, at + lag[j], dp * w[:, j])
        dw.append((dp * ext[at + lag[j]]).sum(0))
    if c["h0"]:
        dext.index_add_(0, last, s["dht"].float().reshape(-1, c["D"]))
    g = {"x": dext[at].reshape(s["x"].shape), "w": torch.stack(dw, 1), "b": dp.sum(0)}
    if h0 is not None:
        keep = torch.ones(ext.shape[0], dtype=torch.bool, device=x.device)
        keep[at] = False
        g["h0"] = dext[keep].reshape(h0.shape)
    return out + [g[k].to(dt) for k in s["leaves"]]


def _running(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, by doubling: after k rounds every h_t holds its last 2^k terms (a recurrence has no
    product form whose factors all stay in range, so log2(T) rounds over the whole axis stand in its place)."""
    k = 1
    while k < a.shape[1]:
        u2 = u.clone()
        u2[:, k:] += a[:, k:] * u[:, :-k]
        a2 = a.clone()
        a2[:, k:] *= a[:, :-k]
        a, u, k = a2, u2, 2 * k
    return u


def _plain_scan(s):
    c = s["case"]
    dt, N, G, D = _DT[c["dtype"]], c["N"], c["G"], c["D"]
    f = lambda k: None if s[k] is None else s[k].detach().float()  # noqa: E731
    step = c["mode"] == "step"
    x, dtr, A, Bv, Cv, skip, z, h0 = (f(k) for k in ("x", "dt", "A", "B", "C", "skip", "z", "h0"))
    if step:
        x, dtr, Bv, Cv, z = (None if t is None else t[:, None] for t in (x, dtr, Bv, Cv, z))
    B, T = x.shape[:2]
    v = dtr + f("bias")
    d = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
    Be, Ce = (t.repeat_interleave(D // G, 2) for t in (Bv, Cv))             # [B, T, D, N]
    a = torch.exp(d[..., None] * A)
    u = (d * x)[..., None] * Be
    if s["cu"] is not None:
        seq, first, end = _sequence_of(s, T)
        start = torch.arange(T, device=x.device) == first[seq]
    ahead = a                                                               # what reaches back over a sequence's start
    if h0 is not None or s["cu"] is not None:
        a = a.clone()
        if s["cu"] is None:
            u[:, 0] += a[:, 0] * h0
            a[:, 0] = 0
        else:
            if h0 is not None:
                u[0] += torch.where(start[:, None, None], a[0] * h0[seq], torch.zeros_like(u[0]))
            a[:, start] = 0
    h = _running(a, u)
    del u
    p = (h * Ce).sum(-1)
    p = p if skip is None else p + skip * x
    y = p if z is None else p * z * torch.sigmoid(z)
    out = [(y[:, 0] if step else y).to(dt)]
    if step:
        s["h0"].copy_(h[:, 0])
        return out + [s["h0"]]
    if c["h0"]:
        ht = h[:, -1].clone() if s["cu"] is None else torch.where((end > first)[:, None, None], h[0, (end - 1).clamp(min=0)], h0)
        out.append(ht)
    if c["mode"] != "train":
        return out
    dy = s["dy"].float()
    g = dy if z is None else dy * z * torch.sigmoid(z)
    du = g[..., None] * Ce
    an = torch.zeros_like(a)                                                # the decay of the token to the right
    an[:, :-1] = a[:, 1:]
    dht = None if s["dht"] is None else s["dht"]
    if dht is not None:
        if s["cu"] is None:
            du[:, -1] += dht
        else:
            some = end > first
            du[0].index_add_(0, (end - 1)[some], dht[some])
    dh = _running(an.flip(1), du.flip(1)).flip(1)
    del du, an
    grad = {}
    if h0 is not None:
        first_rows = ahead[:, 0] * dh[:, 0] if s["cu"] is None else (ahead[0] * dh[0])[first.clamp(max=T - 1)]
        grad["h0"] = first_rows if s["cu"] is None else torch.where(some[:, None, None], first_rows, dht)
    before = torch.zeros_like(h)                                            # the state that a token's decay multiplies
    before[:, 1:] = h[:, :-1]
    if s["cu"] is None:
        before[:, 0] = 0 if h0 is None else h0
    else:
        before[0] = torch.where(start[:, None, None], torch.zeros_like(before[0]) if h0 is None else h0[seq], before[0])
    q = before.mul_(ahead).mul_(dh)                                         # dh e^{dA} h_{t-1}
    dot = (dh * Be).sum(-1)
    dd = x * dot + (q * A).sum(-1)
    grad["x"] = d * dot if skip is None else d * dot + skip * g
    grad["dt"] = dd * torch.sigmoid(v)
    grad["bias"] = grad["dt"].sum((0, 1))
    grad["A"] = torch.einsum("btdn,btd->dn", q, d)
    grad["B"] = (dh * (d * x)[..., None]).reshape(B, T, G, D // G, N).sum(3)
    grad["C"] = (h * g[..., None]).reshape(B, T, G, D // G, N).sum(3)
    if skip is not None:
        grad["skip"] = (g * x).sum((0, 1))
    if z is not None:
        grad["z"] = dy * p * _silu_grad(z)
    return out + [grad[k].to(s[k].dtype) for k in s["leaves"]]


def _rms(a):
    return a.shape[-1] ** 0.5 * torch.rsqrt((a * a).sum(-1, keepdim=True) + EPS)


def _rms_grad(a, r, w, dn):
    """(gradient of a, of w) of n = a r w, r = sqrt(D) / sqrt(sum a^2 + eps)."""
    t = dn * w
    return r * t - a * r ** 3 / a.shape[-1] * (t * a).sum(-1, keepdim=True), (dn * a * r).sum((0, 1))


def _plain_norm(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    f = lambda k: s[k].detach().float() if isinstance(s[k], torch.Tensor) else s[k]  # noqa: E731
    x, res, gate, scale, pw, nw = (f(k) for k in ("x", "r", "g", "v", "p", "n"))
    rx = _rms(x) if pw is not None else None
    n = x if pw is None else x * rx * pw
    sg = None if gate is None else torch.sigmoid(gate)
    v = n if gate is None else n * sg
    r = scale * v if res is None else res + scale * v
    out = [r.to(dt)]
    rr = _rms(r) if nw is not None else None
    if nw is not None:
        out.append((r * rr * nw).to(dt))
    if c["mode"] != "train":
        return out
    grad = {}
    dr = s["dy"].float()
    if nw is not None:
        more, grad["n"] = _rms_grad(r, rr, nw, s["dht"].float())
        dr = dr + more
    grad["r"] = dr
    grad["v"] = (dr * v).sum((0, 1))
    dv = scale * dr
    if gate is not None:
        grad["g"] = dv * n * sg * (1 - sg)
        dv = dv * sg
    if pw is None:
        grad["x"] = dv
    else:
        grad["x"], grad["p"] = _rms_grad(x, rx, pw, dv)
    return out + [grad[k].to(dt) for k in s["leaves"]]


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, mode, has = case["op"], case["mode"], case["parts"]
    e = 2 if case["dtype"] == "bf16" else 4
    train = mode == "train"
    rows, D, n = case["B"] * case["T"], case["D"], case["seqs"] or case["B"]
    if op == "conv":
        W = case["W"]
        big = rows * D
        state = 2 * n * (W - 1) * D * e if case["h0"] or mode == "step" else 0
        small = D * (W + ("b" in has)) * e
        return {"bytes": (4 if train else 2) * big * e + (2 if train else 1) * (state + small),
                "flops": big * ((6 * W + 14) if train else (2 * W + 4))}
    if op == "scan":
        N, G = case["N"], case["G"]
        big, bc = rows * D * e, rows * 2 * G * N * e
        z = "z" in has
        state = 2 * n * D * N * 4 if case["h0"] or mode == "step" else 0
        small = D * (N + 1 + ("s" in has)) * 4
        fwd, bwd = (3 + z) * big + bc, (3 + z) * big + bc                  # x, dt, z, y and then dy, dx, ddt, dz
        return {"bytes": fwd + (bwd if train else 0) + (2 if train else 1) * (state + small),
                "flops": rows * D * ((24 if train else 7) * N + 10)}
    tensors = 2 + ("r" in has) + ("g" in has) + ("n" in has)                # x, r out, residual, gate, u; and their gradients
    return {"bytes": (2 if train else 1) * (tensors * rows * D * e + 3 * D * e), "flops": rows * D * (40 if train else 12)}


# --------------------------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](case, s)


def _spans(case, s):
    """(batch row, first token, end, number of the state) of every sequence."""
    if case["seqs"]:
        cu = _offsets(case)
        return [(0, cu[i], cu[i + 1], i) for i in range(case["seqs"])]
    return [(b, 0, case["T"], b) for b in range(case["B"])]


def _exact_conv(case, s):
    W, D = case["W"], case["D"]
    w = s["w"].double()
    if case["mode"] == "step":
        win = torch.cat([s["h0"].double(), s["x"].double()[:, None]], 1)
        p = torch.einsum("bwd,dw->bd", win, w) + (0 if s["b"] is None else s["b"].double())
        return [p / (1 + torch.exp(-p)), win[:, 1:]]
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device=w.device)
    dx, dw, db, finals, dh0 = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(w[:, 0]), [], []
    for b, t0, t1, i in _spans(case, s):
        hist = torch.zeros(W - 1, D, dtype=torch.float64, device=w.device) if s["h0"] is None else s["h0"][i].double()
        win = torch.cat([hist, s["x"][b, t0:t1].double()])
        finals.append(win[win.shape[0] - (W - 1):])
        if t1 == t0:
            dh0.append(torch.zeros_like(hist) if s.get("dht") is None else s["dht"][i].double())
            continue
        p = win.unfold(0, W, 1).mul(w).sum(-1) + (0 if s["b"] is None else s["b"].double())
        y[b, t0:t1] = p / (1 + torch.exp(-p))
        if case["mode"] == "train":
            sg = 1 / (1 + torch.exp(-p))
            dp = s["dy"][b, t0:t1].double() * (sg + p * sg * (1 - sg))
            dwin = torch.zeros_like(win)
            for j in range(W):
                dwin[j:j + t1 - t0] += dp * w[:, j]
                dw[:, j] += (dp * win[j:j + t1 - t0]).sum(0)
            if s["dht"] is not None:
                dwin[win.shape[0] - (W - 1):] += s["dht"][i].double()
            db += dp.sum(0)
            dx[b, t0:t1] = dwin[W - 1:]
            dh0.append(dwin[:W - 1])
    out = [y] + ([torch.stack(finals)] if case["h0"] else [])
    if case["mode"] == "train":
        g = {"x": dx, "w": dw, "b": db, "h0": torch.stack(dh0)}
        out += [g[k] for k in s["leaves"]]
    return out


def _exact_scan(case, s):
    """Token by token, all batch rows at once; a packed batch restarts at each sequence's first token."""
    D, N, G, step = case["D"], case["N"], case["G"], case["mode"] == "step"
    dbl = lambda k: None if s[k] is None else (s[k].double()[:, None] if step and k in ("x", "dt", "B", "C", "z") else s[k].double())  # noqa: E731
    x, dtr, A, Bv, Cv, skip, z, bias, h0 = (dbl(k) for k in ("x", "dt", "A", "B", "C", "skip", "z", "bias", "h0"))
    nb, T = x.shape[:2]
    dev = x.device
    v = dtr + bias
    d = torch.nn.functional.softplus(v, threshold=60.0)
    per = D // G
    wide = lambda m, t: m[:, t].repeat_interleave(per, 1) if G > 1 else m[:, t].expand(nb, D, N)  # noqa: E731
    spans = _spans(case, s)
    first = {t0: i for b, t0, t1, i in spans if t1 > t0} if case["seqs"] else {0: None}
    last = {t1 - 1: i for b, t0, t1, i in spans if t1 > t0} if case["seqs"] else {T - 1: None}
    zero = torch.zeros(nb, D, N, dtype=torch.float64, device=dev)
    state = lambda m, i: zero.clone() if m is None else (m.clone() if i is None else m[i][None].clone())  # noqa: E731
    train = case["mode"] == "train"
    hs = torch.empty(T, nb, D, N, dtype=torch.float64, device=dev) if train else None
    p = torch.empty(nb, T, D, dtype=torch.float64, device=dev)
    ht = None if h0 is None else h0.clone()
    h = None
    for t in range(T):
        if t in first:
            h = state(h0, first[t])
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * wide(Bv, t)
        if train:
            hs[t] = h
        p[:, t] = (h * wide(Cv, t)).sum(-1)
        if t in last and ht is not None:
            if last[t] is None:
                ht = h.clone()
            else:
                ht[last[t]] = h[0]
    if skip is not None:
        p += skip * x
    gate = None if z is None else z / (1 + torch.exp(-z))
    y = p if gate is None else p * gate
    if step:
        return [y[:, 0], ht]
    out = [y] + ([ht] if case["h0"] else [])
    if not train:
        return out
    dy = s["dy"].double()
    g = dy if gate is None else dy * gate
    dht = None if s["dht"] is None else s["dht"].double()
    dB, dC, dA = torch.zeros_like(Bv), torch.zeros_like(Cv), torch.zeros_like(A)
    dot, from_decay = torch.empty_like(x), torch.empty_like(x)
    dh0 = None if dht is None else dht.clone()
    carry = None
    for t in range(T - 1, -1, -1):
        if t in last:
            carry = state(dht, last[t])
        dh = carry + g[:, t, :, None] * wide(Cv, t)
        prev = state(h0, first[t]) if t in first else hs[t - 1]
        e = torch.exp(d[:, t, :, None] * A)
        q = dh * e * prev
        dA += (q * d[:, t, :, None]).sum(0)
        from_decay[:, t] = (q * A).sum(-1)
        dot[:, t] = (dh * wide(Bv, t)).sum(-1)
        dB[:, t] = (dh * (d[:, t] * x[:, t])[..., None]).view(nb, G, per, N).sum(2)
        dC[:, t] = (hs[t] * g[:, t, :, None]).view(nb, G, per, N).sum(2)
        carry = dh * e
        if t in first and dh0 is not None:
            if first[t] is None:
                dh0 = carry.clone()
            else:
                dh0[first[t]] = carry[0]
    ddt = (x * dot + from_decay) / (1 + torch.exp(-v))
    grads = {"x": d * dot + (0 if skip is None else skip * g), "dt": ddt, "A": dA, "B": dB, "C": dC, "bias": ddt.sum((0, 1)),
             "skip": (g * x).sum((0, 1)), "h0": dh0}
    if z is not None:
        sg = 1 / (1 + torch.exp(-z))
        grads["z"] = dy * p * (sg + z * sg * (1 - sg))
    return out + [grads[k] for k in s["leaves"]]


def _exact_norm(case, s):
    """Forward from the definition; gradients by the same expressions under 64-bit differentiation."""
    names = ("x", "r", "g", "v", "p", "n")
    with torch.enable_grad():
        t = {k: s[k].detach().double().requires_grad_(case["mode"] == "train") if isinstance(s[k], torch.Tensor) else s[k] for k in names}
        rms = lambda a, w: w * a * math.sqrt(case["D"]) / torch.sqrt(torch.sum(a ** 2, -1, keepdim=True) + EPS)  # noqa: E731
        v = t["x"] if t["p"] is None else rms(t["x"], t["p"])
        if t["g"] is not None:
            v = v / (1 + torch.exp(-t["g"]))
        r = t["v"] * v
        if t["r"] is not None:
            r = r + t["r"]
        out = [r] if t["n"] is None else [r, rms(r, t["n"])]
        if case["mode"] != "train":
            return out
        up = [s["dy"].double()] if t["n"] is None else [s["dy"].double(), s["dht"].double()]
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [t[k] for k in s["leaves"]], up))
