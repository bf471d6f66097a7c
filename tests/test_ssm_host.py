"""CPU: refusals of the state space mixer's C entry points, the oracle's gradients against differences, no CPU path."""
import ctypes as C
import os
import re

import pytest
import torch

from hdla_impl_b200 import _lib, layer_ops, ssm
from oracle import ssm_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def struct_of(name):
    """The argument struct as the header declares it."""
    text = open(os.path.join(ROOT, "include", "hdla.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S)[1], flags=re.S)
    kinds = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
    fields = []
    for line in body.split(";"):
        m = re.match(r"\s*(?:const\s+)?(\w+)\s*(.*)", line.strip(), re.S)
        if m:
            for f in m[2].split(","):
                f = f.strip()
                fields.append((f.lstrip("* "), C.c_void_p if "*" in m[2] else kinds[m[1]]))
    return type(name, (C.Structure,), {"_fields_": fields})


Conv, Scan, Norm = (struct_of(n) for n in ("HdlaConvArgs", "HdlaScanArgs", "HdlaNormResidualArgs"))
SOME = 256                 # stands for a pointer in calls that are refused before anything is read


def answer(name, args, *more):
    f = getattr(_lib.load(), name)
    f.restype = C.c_int
    return f(C.byref(args) if args is not None else None, *more, None), _lib.last_error()


def conv(**kw):
    return Conv(**{**dict(B=1, T=1, D=8, W=4, x=SOME, weight=SOME, y=SOME, h0=SOME, ht=SOME, dx=SOME, dweight=SOME), **kw})


def scan(**kw):
    return Scan(**{**dict(B=1, T=1, D=8, N=4, G=1, x=SOME, dt=SOME, Bm=SOME, Cm=SOME, A=SOME, y=SOME, h0=SOME, ht=SOME, checkpoints=SOME,
                          dx=SOME, ddt=SOME, dB=SOME, dC=SOME, dA=SOME), **kw})


def norm(**kw):
    return Norm(**{**dict(rows=1, D=8, x=SOME, r=SOME, dx=SOME, eps=1e-5), **kw})


WS = (C.c_void_p(SOME), C.c_size_t(0))
NO_WS = (None, C.c_size_t(1 << 30))


@pytest.mark.parametrize("name,args,more,code,text", [
    ("hdla_short_conv_fwd", None, (), -1, "null"),
    ("hdla_short_conv_fwd", conv(D=0), (), -1, "non-positive"),
    ("hdla_short_conv_fwd", conv(T=(1 << 30) + 1), (), -2, "at most"),
    ("hdla_short_conv_fwd", conv(W=9), (), -2, "taps"),
    ("hdla_short_conv_fwd", conv(W=0), (), -2, "taps"),
    ("hdla_short_conv_fwd", conv(dtype=2), (), -2, "dtype"),
    ("hdla_short_conv_fwd", conv(w_dtype=7), (), -2, "dtype"),
    ("hdla_short_conv_fwd", conv(activation=2), (), -2, "activation"),
    ("hdla_short_conv_fwd", conv(n_seqs=2), (), -1, "n_seqs"),
    ("hdla_short_conv_fwd", conv(B=2, n_seqs=2, cu_seqlens=SOME), (), -1, "n_seqs"),
    ("hdla_short_conv_fwd", conv(y=None), (), -1, "null"),
    ("hdla_short_conv_bwd", conv(dx=None), WS, -1, "null"),
    ("hdla_short_conv_bwd", conv(), WS, -3, "too small"),
    ("hdla_short_conv_bwd", conv(), NO_WS, -3, "aligned"),
    ("hdla_short_conv_step", conv(T=2), (), -1, "one token"),
    ("hdla_short_conv_step", conv(ht=2 * SOME), (), -1, "not h0"),
    ("hdla_selective_scan_fwd", None, WS, -1, "null"),
    ("hdla_selective_scan_fwd", scan(N=129), WS, -2, "states"),
    ("hdla_selective_scan_fwd", scan(N=0), WS, -2, "states"),
    ("hdla_selective_scan_fwd", scan(G=3), WS, -1, "groups"),
    ("hdla_selective_scan_fwd", scan(B=-1), WS, -1, "non-positive"),
    ("hdla_selective_scan_fwd", scan(A=None), WS, -1, "null"),
    ("hdla_selective_scan_fwd", scan(T=100000), WS, -3, "too small"),
    ("hdla_selective_scan_bwd", scan(checkpoints=None), WS, -1, "null"),
    ("hdla_selective_scan_bwd", scan(z=SOME), WS, -1, "null"),
    ("hdla_selective_scan_bwd", scan(), WS, -3, "too small"),
    ("hdla_selective_scan_step", scan(h0=None), (), -1, "null"),
    ("hdla_selective_scan_step", scan(n_seqs=1, cu_seqlens=SOME), (), -1, "one token"),
    ("hdla_norm_residual_fwd", None, (), -1, "null"),
    ("hdla_norm_residual_fwd", norm(rows=0), (), -1, "bad size"),
    ("hdla_norm_residual_fwd", norm(D=8193), (), -2, "at most"),
    ("hdla_norm_residual_fwd", norm(dtype=0, r_dtype=1), (), -2, "dtype"),
    ("hdla_norm_residual_fwd", norm(activation=3), (), -2, "activation"),
    ("hdla_norm_residual_fwd", norm(pre_weight=SOME), (), -1, "null"),
    ("hdla_norm_residual_bwd", norm(), WS, -3, "too small"),
    ("hdla_norm_residual_bwd", norm(post_weight=SOME), WS, -1, "null"),
])
def test_refusals_of_the_c_entry_points(name, args, more, code, text):
    rc, said = answer(name, args, *more)
    assert rc == code and text in said, (rc, said)


def test_a_size_is_zero_where_the_call_would_be_refused():
    lib = _lib.load()
    for name, bad, good, more in (("hdla_short_conv_bwd_workspace_bytes", conv(W=9), conv(), ()),
                                  ("hdla_selective_scan_checkpoint_bytes", scan(N=0), scan(), ()),
                                  ("hdla_selective_scan_workspace_bytes", scan(G=3), scan(), (1,)),
                                  ("hdla_norm_residual_bwd_workspace_bytes", norm(D=-1), norm(), ())):
        f = getattr(lib, name)
        f.restype = C.c_size_t
        assert f(C.byref(bad), *more) == 0 and f(C.byref(good), *more) > 0


def test_no_cpu_path():
    x, w, A, bc = torch.zeros(1, 4, 8), torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(1, 4, 2)
    for f in (lambda: ssm.short_convolution(x, w), lambda: ssm.short_convolution_step(x[:, 0], torch.zeros(1, 3, 8), w),
              lambda: ssm.selective_scan(x, x, A, bc, bc), lambda: layer_ops.rms_norm_residual(x, x),
              lambda: ssm.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], torch.zeros(1, 8, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


@pytest.mark.parametrize("cu", [None, [0, 0, 2, 5, 5]])
def test_the_oracles_gradients_against_differences(cu):
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    n = 1 if cu is None else 4
    conv_in = (rn(1, 6, 4), rn(4, 3), rn(4), rn(n, 2, 4))
    assert torch.autograd.gradcheck(lambda x, w, b, h: orc.short_conv(x, w, b, "silu", h, cu), conv_in)
    scan_in = (rn(1, 6, 4), rn(1, 6, 4), rn(4, 3), rn(1, 6, 2, 3), rn(1, 6, 2, 3), rn(4), rn(1, 6, 4), rn(4), rn(n, 4, 3))
    assert torch.autograd.gradcheck(lambda x, dt, A, B, C, D, z, b, h: orc.selective_scan(x, dt, A, B, C, D, z, b, True, h, cu), scan_in)
    assert torch.autograd.gradcheck(lambda x, r, g, v, p, q: orc.norm_residual(x, r, g, v, p, q),
                                    (rn(2, 5), rn(2, 5), rn(2, 5), rn(5), rn(5), rn(5)))
