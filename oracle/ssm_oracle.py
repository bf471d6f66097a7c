"""fp64 torch-on-CPU restatement of the selective state space mixer and the norms round a block, token by token and sequence by
sequence; gradients by autograd through these definitions."""
from __future__ import annotations

import torch


def _act(v, name):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return 1 / (1 + torch.exp(-v)) if name == "sigmoid" else v


def spans(B, T, cu=None):
    """(batch row, first token, end, number of the state) of every sequence."""
    return [(b, 0, T, b) for b in range(B)] if cu is None else [(0, cu[i], cu[i + 1], i) for i in range(len(cu) - 1)]


def short_conv(x, w, bias=None, act="silu", h0=None, cu=None):
    """(y, final states); tokens of no sequence give zeros."""
    B, T, D = x.shape
    W = w.shape[1]
    y, finals = [[x.new_zeros(D)] * T for _ in range(B)], []
    for b, t0, t1, i in spans(B, T, cu):
        win = list(x.new_zeros(W - 1, D) if h0 is None else h0[i])
        for t in range(t0, t1):
            win.append(x[b, t])
            p = sum(w[:, j] * win[len(win) - W + j] for j in range(W))
            y[b][t] = _act(p if bias is None else p + bias, act)
        finals.append(torch.stack(win[len(win) - W + 1:]) if W > 1 else x.new_zeros(0, D))
    return torch.stack([torch.stack(r) for r in y]), torch.stack(finals)


def selective_scan(x, dt, A, Bm, Cm, D=None, z=None, bias=None, softplus=True, h0=None, cu=None):
    """(y, final states); Bm, Cm are [B, T, G, N]."""
    B, T, ch = x.shape
    per = ch // Bm.shape[2]
    d = dt if bias is None else dt + bias
    if softplus:
        d = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))
    y, finals = [[x.new_zeros(ch)] * T for _ in range(B)], []
    for b, t0, t1, i in spans(B, T, cu):
        h = x.new_zeros(A.shape) if h0 is None else h0[i]
        for t in range(t0, t1):
            h = torch.exp(d[b, t][:, None] * A) * h + (d[b, t] * x[b, t])[:, None] * Bm[b, t].repeat_interleave(per, 0)
            p = (Cm[b, t].repeat_interleave(per, 0) * h).sum(-1)
            p = p if D is None else p + D * x[b, t]
            y[b][t] = p if z is None else p * _act(z[b, t], "silu")
        finals.append(h)
    return torch.stack([torch.stack(r) for r in y]), torch.stack(finals)


def norm_residual(x, residual=None, gate=None, scale=1.0, post=None, pre=None, act="sigmoid", eps=1e-5):
    """(r, u or None)."""
    rms = lambda a, w: a.shape[-1] ** 0.5 * a / torch.sqrt((a * a).sum(-1, keepdim=True) + eps) * w  # noqa: E731
    v = x if post is None else rms(x, post)
    v = v if gate is None else v * _act(gate, act)
    r = scale * v if residual is None else residual + scale * v
    return r, None if pre is None else rms(r, pre)
