"""CPU checks of the sequence operators: the 64-bit restatement's gradients against differences, the structs against the header,
and what the entry points refuse before they touch a device."""
import ctypes
import os
import re

import numpy as np
import pytest

from oracle import sequence as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _directional(f, arrays, grads, rng):
    """d/de f(arrays + e v) by central differences against sum(grads * v), for a random direction per array."""
    for name, a in arrays.items():
        v = rng.standard_normal(a.shape)
        e = 1e-6
        up, down = (f(**(arrays | {name: a + k * e * v})) for k in (1, -1))
        want = float((grads[name] * v).sum())
        # central differences in 64 bits: e^2 from the third derivative, 2^-53 |f| / e from rounding
        assert abs((up - down) / (2 * e) - want) < 1e-6 * (1 + abs(want)), name


@pytest.mark.parametrize("reverse", (False, True))
@pytest.mark.parametrize("softplus", (False, True))
def test_restated_scan_gradient_against_differences(reverse, softplus):
    rng = np.random.default_rng(3)
    nb, n, d, ns, g = 2, 6, 4, 3, 2
    a = dict(x=rng.standard_normal((nb, n, d)), dt=rng.uniform(0.1, 0.6, (nb, n, d)), A=-rng.uniform(0.2, 2, (d, ns)),
             B=rng.standard_normal((nb, n, g, ns)), C=rng.standard_normal((nb, n, g, ns)), D=rng.standard_normal(d),
             z=rng.standard_normal((nb, n, d)), dt_bias=0.1 * rng.standard_normal(d), state=rng.standard_normal((nb, d, ns)))
    frames = np.array([6, 3])
    dy, dl = rng.standard_normal((nb, n, d)), rng.standard_normal((nb, d, ns))
    kw = dict(use_softplus=softplus, frames=frames, reverse=reverse)

    def f(**v):
        o = S.scan(**v, **kw)
        return float((o["y"][0] * dy).sum() + (o["last"][0] * dl).sum())

    o = S.scan(**a, **kw, dy=dy, dlast=dl)
    grads = {k: o["d" + {"dt_bias": "bias"}.get(k, k)][0] for k in a}
    _directional(f, a, grads, rng)
    assert np.all(o["y"][0][1, 3:] == 0) and np.all(o["dx"][0][1, 3:] == 0)


@pytest.mark.parametrize("own", (0, 1, 2, 7))
@pytest.mark.parametrize("reverse", (False, True))
def test_restated_conv_gradient_against_differences(reverse, own):
    rng = np.random.default_rng(4)
    nb, n, d, W = 2, 7, 3, 4
    a = dict(x=rng.standard_normal((nb, n, d)), weight=rng.standard_normal((d, W)), bias=rng.standard_normal(d),
             state=rng.standard_normal((nb, W - 1, d)))
    dy, dl = rng.standard_normal((nb, n, d)), rng.standard_normal((nb, W - 1, d))
    kw = dict(silu=True, frames=np.array([own, 5]), reverse=reverse)

    def f(**v):
        o = S.conv(**v, **kw)
        return float((o["y"][0] * dy).sum() + (o["last"][0] * dl).sum())

    o = S.conv(**a, **kw, dy=dy, dlast=dl)
    _directional(f, a, {k: o[{"weight": "dw", "bias": "db"}.get(k, "d" + k)][0] for k in a}, rng)


@pytest.mark.parametrize("act", (None, "silu", "gelu"))
def test_restated_norm_gradient_against_differences(act):
    rng = np.random.default_rng(5)
    a = dict(x=rng.standard_normal((2, 5, 2, 6)), weight=rng.standard_normal(6), bias=rng.standard_normal(6))
    dy = rng.standard_normal((2, 5, 2, 6))
    kw = dict(groups=2, act=act, frames=np.array([5, 2]))
    o, _ = S.group_norm(**a, **kw, dy=dy)
    _directional(lambda **v: float((S.group_norm(**v, **kw)[0]["y"][0] * dy).sum()), a,
                 {"x": o["dx"][0], "weight": o["dw"][0], "bias": o["db"][0]}, rng)


@pytest.mark.parametrize("name,cls", (("sed_scan_args", "ScanArgs"), ("sed_conv_args", "ConvArgs"), ("sed_norm_args", "NormArgs")))
def test_structs_match_the_header(name, cls):
    from sed_amd import _lib
    text = open(os.path.join(ROOT, "include", "sed_hip.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    want = []
    for decl in (d.strip() for d in body.split(";")):
        if not decl:
            continue
        decl = decl.replace("const ", "")
        base, rest = decl.split(None, 1) if not decl.split(None, 1)[0].endswith("*") else (decl.split(None, 1)[0], decl.split(None, 1)[1])
        pointer = base.endswith("*")
        for n in rest.split(","):
            n = n.strip()
            kind = ctypes.c_void_p if pointer or n.startswith("*") else {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}[base]
            want.append((n.lstrip("* "), kind))
    assert list(getattr(_lib, cls)._fields_) == want


def test_c_entry_points_refuse():
    from sed_amd import _lib as L
    byref = ctypes.byref
    assert L.lib.sed_gated_scan_workspace(None, 0) == L.SED_ERR_BAD_ARG
    assert L.lib.sed_gated_scan_workspace(byref(L.ScanArgs(B=1, L=8, D=4, N=33, G=1)), 0) == L.SED_ERR_BAD_ARG
    assert L.lib.sed_gated_scan_workspace(byref(L.ScanArgs(B=1, L=8, D=4, N=4, G=3)), 0) == L.SED_ERR_BAD_ARG
    assert L.lib.sed_gated_scan_saved_floats(1, 8, 0, 4) == L.SED_ERR_BAD_ARG
    assert L.lib.sed_causal_conv_workspace(1, 8, 4, 9) == L.SED_ERR_BAD_ARG
    assert L.lib.sed_group_norm_workspace(1, 8, 1, 6, 4) == L.SED_ERR_BAD_ARG
    for fn in (L.lib.sed_gated_scan_forward, L.lib.sed_gated_scan_backward, L.lib.sed_gated_scan_step):
        assert fn(None, None) == L.SED_ERR_BAD_ARG
        a = L.ScanArgs(B=1, L=1, D=4, N=4, G=1)
        assert fn(byref(a), None) == L.SED_ERR_BAD_ARG      # no pointers
        a = L.ScanArgs(B=1, L=1, D=4, N=33, G=1, x=16, dt=16, A=16, Bm=16, Cm=16, y=16)
        assert fn(byref(a), None) == L.SED_ERR_BAD_ARG      # too many states
        a = L.ScanArgs(B=1, L=1, D=4, N=4, G=1, dtype=7, x=16, dt=16, A=16, Bm=16, Cm=16, y=16)
        assert fn(byref(a), None) == L.SED_ERR_BAD_ARG
        a = L.ScanArgs(B=0, L=1, D=4, N=4, G=1)
        assert fn(byref(a), None) == L.SED_OK               # nothing to do
    many = dict(B=1, L=512, D=64, N=16, G=1, x=16, dt=16, A=16, Bm=16, Cm=16, y=16)
    assert L.lib.sed_gated_scan_workspace(byref(L.ScanArgs(B=1, L=512, D=64, N=16, G=1)), 0) > 0
    far = many | {"x_t": (1 << 26) + 1}
    assert L.lib.sed_gated_scan_forward(byref(L.ScanArgs(**far)), None) == L.SED_ERR_CAPACITY
    assert L.lib.sed_gated_scan_forward(byref(L.ScanArgs(**many)), None) == L.SED_ERR_CAPACITY  # no workspace
    assert L.lib.sed_gated_scan_step(byref(L.ScanArgs(**(many | {"h_last": 16}))), None) == L.SED_ERR_BAD_ARG  # 512 frames
    for fn in (L.lib.sed_causal_conv_forward, L.lib.sed_causal_conv_backward, L.lib.sed_causal_conv_step):
        assert fn(None, None) == L.SED_ERR_BAD_ARG
        assert fn(byref(L.ConvArgs(B=1, L=1, D=4, W=9, x=16, weight=16, y=16)), None) == L.SED_ERR_BAD_ARG
        assert fn(byref(L.ConvArgs(B=1, L=1, D=4, W=4, act=L.ACT_GELU, x=16, weight=16, y=16)), None) == L.SED_ERR_BAD_ARG
        assert fn(byref(L.ConvArgs(B=1, L=0, D=4, W=4)), None) == L.SED_OK
    a = L.ConvArgs(B=1, L=4, D=4, W=4, x=16, weight=16, dy=16, dx=16, dw=16)
    assert L.lib.sed_causal_conv_backward(byref(a), None) == L.SED_ERR_CAPACITY
    for fn in (L.lib.sed_group_norm_forward, L.lib.sed_group_norm_backward):
        assert fn(None, None) == L.SED_ERR_BAD_ARG
        ok = dict(B=1, T=2, F=1, C=4, G=2, eps=1e-5, x=16, mean=16, rstd=16, y=16, dy=16, dx=16)
        assert fn(byref(L.NormArgs(**ok)), None) == L.SED_ERR_CAPACITY  # no workspace
        for bad in (dict(G=3), dict(act=9), dict(eps=-1.0), dict(F=0), dict(x=None), dict(dtype=3)):
            assert fn(byref(L.NormArgs(**(ok | bad))), None) == L.SED_ERR_BAD_ARG
        assert fn(byref(L.NormArgs(**(ok | dict(B=65536)))), None) == L.SED_ERR_CAPACITY


def test_python_entry_points_refuse_cpu_tensors():
    import torch
    import sed_amd
    x = torch.zeros(1, 4, 8)
    bc = torch.zeros(1, 4, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sed_amd.gated_scan(x, x, torch.zeros(8, 2), bc, bc)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sed_amd.gated_scan_step(torch.zeros(1, 8, 2), x[:, 0], x[:, 0], torch.zeros(8, 2), bc[:, 0], bc[:, 0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        sed_amd.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        sed_amd.causal_conv_step(torch.zeros(1, 3, 8), x[:, 0], torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        sed_amd.group_norm_act(x, 2)


def test_workspaces_of_empty_and_of_large_calls():
    """Host arithmetic only: no clip, no frame, one wave and more waves than the card holds; never negative, never less for a gradient."""
    from ctypes import byref
    from sed_amd import _lib as L
    for B in (0, 1, 2, 63, 5000):
        for n in (0, 1, 9, 700, 100000):
            for N in (1, 4, 8, 16, 17):
                for dtype in (L.F32, L.BF16):
                    for ragged in (None, 16):
                        a = L.ScanArgs(B=B, L=n, D=96, N=N, G=1, dtype=dtype, frames=ragged)
                        forward, back = L.lib.sed_gated_scan_workspace(byref(a), 0), L.lib.sed_gated_scan_workspace(byref(a), 1)
                        assert forward >= 0 and back >= 4 * B * n * 2 * N
            assert L.lib.sed_causal_conv_workspace(B, n, 96, 4) >= 0
            assert L.lib.sed_group_norm_workspace(B, n, 3, 96, 8) >= 0
