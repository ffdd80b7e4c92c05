"""GPU tests of the sequence operators against the 64-bit restatement (oracle/sequence.py).

Tolerances.  u = 2^-24.  A value of the recurrence is a sum of products of at most L decays; every step of it rounds the decay
(2u), the product and the sum (2u), so a term is off by 4 L u of itself, twice that where a gradient joins two walks; the
exponents delta A are off by 8u of themselves, which moves a term decayed by e^-S by 8u S e^-S <= 3u of what it was before it
decayed (6u for two walks).  delta, the gate and the skip add under 100u.  Sums over channels, clips and chunks add one u per
addition in a row.  Outputs are rounded once: half a step of their type."""
import numpy as np
import pytest
import torch

from oracle import sequence as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _dev():
    import sed_amd  # noqa: F401
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def _rounded(a, dtype):
    """The values a tensor of this type holds, as a tensor on the device and in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(a)).to(dtype)
    return t.to(_dev()), t.double().numpy()


def _close(got, want, bound, name):
    t = got.dtype
    half = torch.finfo(t).eps / 2 * np.abs(want) + (2.0 ** -25 if t == torch.float16 else 2.0 ** -126)  # fp16: half a subnormal step
    # a value off by `bound` can round the other way: half a step of what it then is
    tol = bound * (1 + torch.finfo(t).eps) + half
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.shape, name
    assert np.isfinite(g).all(), name
    off = np.abs(g - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape) if off.size else None
    assert (off <= tol).all(), (name, worst, g[worst], want[worst], off[worst], tol[worst])


def _scan_inputs(nb, n, d, g, ns, dtype, seed, softplus=True, gate=True, bias=True, skip=True, state=False, frames=None):
    rng = np.random.default_rng(seed)
    v = {"x": rng.standard_normal((nb, n, d)), "B": rng.standard_normal((nb, n, g, ns)), "C": rng.standard_normal((nb, n, g, ns)),
         "dt": rng.standard_normal((nb, n, d)) - 2 if softplus else rng.uniform(0.001, 0.3, (nb, n, d))}
    if gate:
        v["z"] = rng.standard_normal((nb, n, d))
    p = {"A": -np.arange(1, ns + 1) * np.exp(0.3 * rng.standard_normal((d, ns)))}
    if skip:
        p["D"] = rng.standard_normal(d)
    if bias:
        p["dt_bias"] = 0.3 * rng.standard_normal(d) if softplus else rng.uniform(0, 0.05, d)
    if state:
        p["state"] = rng.standard_normal((nb, d, ns))
    dev, ref = {}, {}
    for k, a in v.items():
        dev[k], ref[k] = _rounded(a, dtype)
    for k, a in p.items():
        dev[k], ref[k] = _rounded(a, torch.float32)
    if frames is not None:
        ref["frames"] = np.asarray(frames)
        dev["frames"] = torch.tensor(frames, dtype=torch.int32, device=_dev())
    return dev, ref, rng


NAMES = {"x": "dx", "dt": "ddt", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "dt_bias": "dbias", "state": "dstate"}


def _scan_bound(o, name, nb, n, d):
    rows = nb * n / 8 + 16 if name in ("dA", "dD", "dbias") else 0  # clips x chunks (a chunk is two tiles of 8 frames at least)
    lanes = d / 4 if name in ("dB", "dC") else 0
    return U * ((8 * n + 200 + rows + lanes) * o[name][1] + 8 * o[name][2])


def _scan_case(nb, n, d, g, ns, dtype, seed=0, softplus=True, reverse=False, grad=True, last=True, **kw):
    import sed_amd
    dev, ref, rng = _scan_inputs(nb, n, d, g, ns, dtype, seed, softplus=softplus, **kw)
    dy, rdy = _rounded(rng.standard_normal((nb, n, d)), dtype)
    dl, rdl = _rounded(rng.standard_normal((nb, d, ns)), torch.float32)
    leaves = {k: t.requires_grad_(grad) for k, t in dev.items() if k != "frames"}
    args = {k: dev[k] for k in dev}
    out = sed_amd.gated_scan(args.pop("x"), args.pop("dt"), args.pop("A"), args.pop("B"), args.pop("C"), **args, softplus=softplus,
                             reverse=reverse, return_state=last)
    y, hl = out if last else (out, None)
    with np.errstate(over="ignore"):
        o = S.scan(**ref, use_softplus=softplus, reverse=reverse, dy=rdy, dlast=rdl if last else None)
    _close(y, o["y"][0], _scan_bound(o, "y", nb, n, d), "y")
    if last:
        _close(hl, o["last"][0], _scan_bound(o, "last", nb, n, d), "last")
    if grad:
        grads = torch.autograd.grad([y, hl] if last else [y], list(leaves.values()), [dy, dl] if last else [dy])
        for (k, t), got in zip(leaves.items(), grads):
            assert got.dtype == t.dtype
            _close(got, o[NAMES[k]][0], _scan_bound(o, NAMES[k], nb, n, d), NAMES[k])


@pytest.mark.parametrize("dtype", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("nb,n,d,g,ns", ((1, 1, 1, 1, 1), (2, 7, 3, 1, 16), (1, 8, 4, 2, 16), (2, 9, 64, 1, 16), (1, 33, 65, 1, 16),
                                         (2, 65, 96, 3, 16), (1, 130, 260, 1, 16), (2, 40, 6, 3, 8), (1, 70, 130, 1, 8), (1, 37, 12, 1, 5),
                                         (2, 66, 33, 1, 4), (1, 20, 300, 1, 4), (1, 50, 7, 1, 3), (1, 90, 257, 1, 1), (3, 17, 36, 2, 1),
                                         (1, 66, 68, 1, 32), (2, 19, 5, 1, 17), (1, 35, 8, 2, 11), (1, 64, 64, 1, 2)))
def test_scan_sizes(nb, n, d, g, ns, dtype):
    _scan_case(nb, n, d, g, ns, DTYPES[dtype], seed=n * d + ns)


@pytest.mark.parametrize("reverse", (False, True))
@pytest.mark.parametrize("ns,d", ((16, 68), (16, 7), (8, 20), (4, 12), (1, 9), (32, 16)))
def test_scan_own_lengths(ns, d, reverse):
    """Clips of no, one, some and all frames, an initial state, and lengths that end inside a tile and on its edge."""
    _scan_case(6, 70, d, 1, ns, torch.float32, seed=ns, reverse=reverse, state=True, frames=[70, 0, 1, 8, 33, 64])
    _scan_case(3, 70, d, 1, ns, torch.bfloat16, seed=ns + 1, reverse=reverse, state=True, frames=[69, 16, 1])


@pytest.mark.parametrize("softplus,gate,bias,skip,state,last", ((False, True, True, True, True, True), (True, False, True, False, False, False),
                                                                (True, True, False, True, False, True), (False, False, False, False, True, False)))
def test_scan_optional_inputs(softplus, gate, bias, skip, state, last):
    for nb, n in ((2, 50), (1, 5)):
        _scan_case(nb, n, 36, 2, 16, torch.float32, softplus=softplus, gate=gate, bias=bias, skip=skip, state=state, last=last, reverse=n == 5)


def test_scan_many_waves_stay_whole():
    """1024 waves and more: no chunks, several tiles of frames in one walk."""
    _scan_case(1030, 21, 4, 1, 4, torch.float32, seed=2, state=True)
    _scan_case(260, 20, 256, 1, 16, torch.bfloat16, seed=3, frames=[(7 * i) % 21 for i in range(260)], reverse=True)


def test_parameter_gradients_of_many_clips():
    """More clips than one pass over their sums takes, a last part of other size among them."""
    _scan_case(2053, 3, 4, 1, 4, torch.float32, seed=11)
    _scan_case(4999, 1, 6, 2, 3, torch.bfloat16, seed=12)
    _conv_case(2050, 2, 5, 4, torch.float32, seed=13)
    _conv_case(5001, 1, 72, 2, torch.bfloat16, seed=14)
    _norm_case((2051, 2, 8), 2, torch.float32, seed=15)
    _norm_case((4500, 3, 40), 5, torch.bfloat16, seed=16)


@pytest.mark.parametrize("nb", (2, 63, 64, 65, 130))
def test_scan_orders_of_clips(nb):
    """Every clip is walked once whatever the order of lengths: equal ones, none, rising and falling, past the ends, more than 64 clips."""
    for k, frames in enumerate(([9] * nb, [0] * nb, list(range(nb)), list(range(nb, 0, -1)), [(29 * i) % 47 - 3 for i in range(nb)])):
        _scan_case(nb, 41, 4, 1, (1, 4, 8, 16, 17)[k], torch.float32, seed=k, frames=frames, reverse=k % 2 == 0, state=True)


@pytest.mark.parametrize("nb,n,d,ns,frames", ((1, 70, 5, 3, None), (3, 1200, 5, 3, (1200, 2, 700)), (260, 9, 257, 3, None), (3, 1200, 5, 8, (3, 1200, 41)),
                                              (260, 9, 512, 8, None), (100, 9, 511, 16, None), (3, 1200, 12, 16, (1200, 0, 99)), (2, 2000, 130, 16, (1999, 1)),
                                              (3, 1200, 6, 32, (5, 640, 1200)), (520, 20, 31, 32, None), (2, 1500, 9, 1, (1500, 17))))
def test_scan_instances_and_chunks(nb, n, d, ns, frames):
    """Few waves and many, so that every instance runs, and long clips in more chunks than a short clip beside them has tiles."""
    _scan_case(nb, n, d, 1, ns, torch.float32, seed=n + ns, frames=frames, state=True, reverse=n % 100 == 0)


@pytest.mark.parametrize("nb,n,d,ns,frames", ((32, 600, 255, 16, None), (2, 2000, 768, 16, (1201, 2000)), (40, 300, 260, 8, None), (32, 300, 255, 32, None)))
def test_scan_large_batches_clip_by_clip(nb, n, d, ns, frames):
    """Batches in which every wave is full and clips are cut: two of the clips against the restatement of those alone."""
    import sed_amd
    dev, ref, rng = _scan_inputs(nb, n, d, 1, ns, torch.bfloat16, ns, state=True, frames=frames)
    dy, rdy = _rounded(rng.standard_normal((nb, n, d)), torch.bfloat16)
    leaves = {k: t.requires_grad_(True) for k, t in dev.items() if k != "frames"}
    args = dict(dev)
    base = [args.pop(k) for k in ("x", "dt", "A", "B", "C")]
    y, last = sed_amd.gated_scan(*base, **args, softplus=True, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    per_clip = ("x", "dt", "B", "C", "z", "state", "frames")
    for b in (0, nb - 1):
        o = S.scan(**{k: (v[b:b + 1] if k in per_clip else v) for k, v in ref.items()}, use_softplus=True, dy=rdy[b:b + 1])
        _close(y[b:b + 1], o["y"][0], _scan_bound(o, "y", nb, n, d), "y")
        _close(last[b:b + 1], o["last"][0], _scan_bound(o, "last", nb, n, d), "last")
        for k in per_clip[:-1]:
            _close(grads[k][b:b + 1], o[NAMES[k]][0], _scan_bound(o, NAMES[k], nb, n, d), NAMES[k])


def test_scan_rows_behind_are_neither_read_nor_kept():
    import sed_amd
    dev, _, rng = _scan_inputs(3, 40, 64, 1, 16, torch.bfloat16, 7, frames=[40, 13, 0])
    dirty = {k: t.clone() for k, t in dev.items()}
    for k in ("x", "dt", "z", "B", "C"):
        dirty[k][1, 13:] = float("nan")
        dirty[k][2] = float("inf")
    dy = torch.randn(3, 40, 64, device=_dev(), dtype=torch.bfloat16)
    bad = dy.clone()
    bad[1, 13:] = float("nan")
    got = []
    for v, g in ((dev, dy), (dirty, bad)):
        leaves = {k: t.clone().requires_grad_(True) for k, t in v.items() if k != "frames"}
        args = dict(leaves)
        y, last = sed_amd.gated_scan(args.pop("x"), args.pop("dt"), args.pop("A"), args.pop("B"), args.pop("C"), **args, softplus=True,
                                     frames=v["frames"], return_state=True)
        got.append([y, last, *torch.autograd.grad(y, list(leaves.values()), g)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    y, dx = got[1][0], got[1][2]
    assert (y[1, 13:] == 0).all() and (y[2] == 0).all() and (dx[1, 13:] == 0).all() and (dx[2] == 0).all()


def test_scan_reads_views_in_place():
    """Halves of a joint projection, rows with odd offsets, a time-major batch and an expanded clip, as they are and copied."""
    import sed_amd
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    A, D = -torch.rand(20, 16, generator=g, device=dev) * 4, r(20)
    for dtype in (torch.bfloat16, torch.float32):
        xz, bc = r(3, 50, 40).to(dtype), r(3, 50, 37).to(dtype)
        time_major = r(50, 3, 20).to(dtype)
        views = (
            (xz[..., :20], time_major.transpose(0, 1), bc[..., 3:19], bc[..., 19:35], xz[..., 20:]),
            (xz[..., 1:21], xz[..., 20:], bc[..., :16], bc[..., 21:], xz[..., 3:23]),
            (xz[:1, :, :20].expand(3, 50, 20), xz[..., 20:], bc[:, :1, :16].expand(3, 50, 16), bc[..., 17:33], None),
            (r(3, 20, 50).to(dtype).transpose(1, 2), xz[..., 20:], bc[..., :16], bc[..., 16:32], None),
        )
        for x, dt, B, C, z in views:
            a = sed_amd.gated_scan(x, dt, A, B, C, D=D, z=z, softplus=True)
            b = sed_amd.gated_scan(x.contiguous(), dt.contiguous(), A, B.contiguous(), C.contiguous(), D=D, z=None if z is None else z.contiguous(), softplus=True)
            assert torch.equal(a, b)
        x = xz[:1, :, :20].detach().clone().requires_grad_(True)
        y = sed_amd.gated_scan(x.expand(3, 50, 20), xz[..., 20:], A, bc[..., :16], bc[..., 16:32], softplus=True)
        (got,) = torch.autograd.grad(y, x, torch.ones_like(y).transpose(0, 1).contiguous().transpose(0, 1))
        full = x.detach().expand(3, 50, 20).contiguous().requires_grad_(True)
        y = sed_amd.gated_scan(full, xz[..., 20:], A, bc[..., :16], bc[..., 16:32], softplus=True)
        (want,) = torch.autograd.grad(y, full, torch.ones_like(y))
        assert torch.equal(got, want.sum(0, keepdim=True))


def test_scan_continues_from_its_state():
    """A sequence in pieces, and frame by frame through the one-frame form, against the whole (bounds as for any output)."""
    import sed_amd
    for dtype in (torch.float32, torch.bfloat16):
        dev, ref, _ = _scan_inputs(3, 45, 24, 2, 16, dtype, 11, state=True)
        o = S.scan(**ref, use_softplus=True)
        cut = lambda t, a, b: t[:, a:b]  # noqa: E731
        state, ys = dev["state"].clone(), []
        for a, b in ((0, 1), (1, 20), (20, 45)):
            y, state = sed_amd.gated_scan(cut(dev["x"], a, b), cut(dev["dt"], a, b), dev["A"], cut(dev["B"], a, b), cut(dev["C"], a, b),
                                          D=dev["D"], z=cut(dev["z"], a, b), dt_bias=dev["dt_bias"], softplus=True, state=state, return_state=True)
            ys.append(y)
        _close(torch.cat(ys, 1), o["y"][0], _scan_bound(o, "y", 3, 45, 24), "pieces")
        _close(state, o["last"][0], _scan_bound(o, "last", 3, 45, 24), "state")
        state, ys = dev["state"].clone(), []
        for t in range(45):
            ys.append(sed_amd.gated_scan_step(state, dev["x"][:, t], dev["dt"][:, t], dev["A"], dev["B"][:, t], dev["C"][:, t], D=dev["D"],
                                              z=dev["z"][:, t], dt_bias=dev["dt_bias"], softplus=True))
        _close(torch.stack(ys, 1), o["y"][0], _scan_bound(o, "y", 3, 45, 24), "frames")
        _close(state, o["last"][0], _scan_bound(o, "last", 3, 45, 24), "state")


@pytest.mark.parametrize("nb,d,g,ns", ((1, 1, 1, 1), (5, 33, 1, 16), (3, 64, 2, 16), (2, 7, 1, 32), (4, 10, 1, 8), (2, 6, 3, 4), (3, 5, 1, 7), (2, 9, 1, 17), (2, 12, 1, 12), (1, 40, 1, 28)))
def test_scan_step_sizes(nb, d, g, ns):
    import sed_amd
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        dev, ref, _ = _scan_inputs(nb, 1, d, g, ns, dtype, ns + d, state=True)
        o = S.scan(**ref, use_softplus=True)
        state = dev["state"].clone()
        y = sed_amd.gated_scan_step(state, dev["x"][:, 0], dev["dt"][:, 0], dev["A"], dev["B"][:, 0], dev["C"][:, 0], D=dev["D"], z=dev["z"][:, 0],
                                    dt_bias=dev["dt_bias"], softplus=True)
        _close(y[:, None], o["y"][0], _scan_bound(o, "y", nb, 1, d), "y")
        _close(state, o["last"][0], _scan_bound(o, "last", nb, 1, d), "state")


def test_scan_gradient_against_differences():
    """A step along the gradient of every input moves the output as the gradient says.  fp32.  Along the gradient a step of
    2^-7 of the input's norm falls on few entries, which it moves by far more than 2^-7 of themselves, so one central difference
    is off by its e^2 term (9 % for A).  Differences of steps e, e/2 and e/4, joined so that the e^2 and e^4 terms cancel, leave
    e^6 (0.09^3 of the slope) and the rounding of f, under 200 u |f|_1 / e: 2 % of the slope covers both."""
    import sed_amd
    dev, _, rng = _scan_inputs(2, 60, 16, 1, 8, torch.float32, 5, state=True)
    dy = torch.from_numpy(rng.standard_normal((2, 60, 16)).astype(np.float32)).to(_dev())
    names = list(dev)

    def f(v):
        y = sed_amd.gated_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], D=v["D"], z=v["z"], dt_bias=v["dt_bias"], softplus=True, state=v["state"])
        return (y.double() * dy).sum()

    leaves = {k: dev[k].clone().requires_grad_(True) for k in names}
    grads = dict(zip(names, torch.autograd.grad(f(leaves), list(leaves.values()))))
    for k in names:
        v = grads[k] / grads[k].norm() * dev[k].norm()
        with torch.no_grad():
            s0, s1, s2 = ((f(dev | {k: dev[k] + e * v}) - f(dev | {k: dev[k] - e * v})) / (2 * e) for e in (2.0 ** -7, 2.0 ** -8, 2.0 ** -9))
        r0, r1 = (4 * s1 - s0) / 3, (4 * s2 - s1) / 3
        slope = (16 * r1 - r0) / 15
        want = (grads[k].double() * v).sum()
        assert abs(slope - want) <= 0.02 * abs(want), (k, float(slope), float(want))


def test_scan_refusals():
    import sed_amd
    dev = _dev()
    x, A = torch.zeros(2, 5, 8, device=dev), torch.zeros(8, 4, device=dev)
    bc = torch.zeros(2, 5, 4, device=dev)
    ok = dict(x=x, dt=x, A=A, B=bc, C=bc)
    for err, bad in ((TypeError, dict(x=x.double())), (TypeError, dict(dt=x.half())), (TypeError, dict(C=bc.bfloat16())), (ValueError, dict(dt=x[:, :4])),
                     (ValueError, dict(A=A[:7])), (ValueError, dict(A=torch.zeros(8, 33, device=dev))), (ValueError, dict(B=bc[..., :3])),
                     (ValueError, dict(B=bc.unsqueeze(2))), (ValueError, dict(x=x[0])), (TypeError, dict(A=A.int())),
                     (ValueError, dict(B=torch.zeros(2, 5, 3, 4, device=dev), C=torch.zeros(2, 5, 3, 4, device=dev))),
                     (ValueError, dict(D=torch.zeros(7, device=dev))), (TypeError, dict(z=x.half())), (RuntimeError, dict(dt_bias=torch.zeros(8))),
                     (TypeError, dict(frames=torch.zeros(2, device=dev))), (TypeError, dict(frames=torch.zeros(3, device=dev, dtype=torch.int32))),
                     (TypeError, dict(frames=torch.zeros(2, dtype=torch.int32))), (ValueError, dict(state=torch.zeros(2, 8, 3, device=dev))),
                     (TypeError, dict(state=torch.zeros(2, 8, 4, device=dev).half()))):
        with pytest.raises(err):
            sed_amd.gated_scan(**(ok | bad))
    st = torch.zeros(2, 8, 4, device=dev)
    step = dict(state=st, x=x[:, 0], dt=x[:, 0], A=A, B=bc[:, 0], C=bc[:, 0])
    for err, bad in ((ValueError, dict(state=st.transpose(0, 1).contiguous().transpose(0, 1))), (TypeError, dict(state=st.half())), (ValueError, dict(x=x)),
                     (RuntimeError, dict(A=A.clone().requires_grad_(True)))):
        with pytest.raises(err):
            sed_amd.gated_scan_step(**(step | bad))
    with pytest.raises(RuntimeError):  # one gradient only
        v = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(sed_amd.gated_scan(v, x, A, bc, bc).sum(), v, create_graph=True)
        g.sum().backward()


def test_empty_calls():
    import sed_amd
    dev = _dev()
    A = torch.zeros(8, 4, device=dev)
    for nb, n in ((0, 5), (2, 0)):
        x = torch.zeros(nb, n, 8, device=dev, requires_grad=True)
        bc, st = torch.zeros(nb, n, 4, device=dev), torch.ones(nb, 8, 4, device=dev, requires_grad=True)
        y, last = sed_amd.gated_scan(x, x, A, bc, bc, state=st, return_state=True)
        assert y.shape == x.shape and torch.equal(last, st)
        gx, gs = torch.autograd.grad([y, last], [x, st], [torch.zeros_like(y), 2 * torch.ones_like(last)])
        assert gx.shape == x.shape and torch.equal(gs, 2 * torch.ones_like(last))
        cs = torch.ones(nb, 3, 8, device=dev)
        y, last = sed_amd.causal_conv(x, torch.ones(8, 4, device=dev), state=cs, return_state=True)
        assert y.shape == x.shape and torch.equal(last, cs)
        assert sed_amd.group_norm_act(x, 2).shape == x.shape
    none = torch.zeros(0, 8, device=dev)
    assert sed_amd.gated_scan_step(torch.zeros(0, 8, 4, device=dev), none, none, A, none[:, :4], none[:, :4]).shape == (0, 8)
    assert sed_amd.causal_conv_step(torch.zeros(0, 3, 8, device=dev), none, A).shape == (0, 8)


# ---- causal convolution -------------------------------------------------------------------------------------------------


def _conv_case(nb, n, d, W, dtype, seed=0, silu=True, bias=True, reverse=False, state=False, frames=None, last=True):
    import sed_amd
    rng = np.random.default_rng(seed)
    x, rx = _rounded(rng.standard_normal((nb, n, d)), dtype)
    w, rw = _rounded(rng.standard_normal((d, W)), torch.float32)
    b, rb = _rounded(rng.standard_normal(d), torch.float32) if bias else (None, None)
    st, rst = _rounded(rng.standard_normal((nb, W - 1, d)), dtype) if state else (None, None)
    dy, rdy = _rounded(rng.standard_normal((nb, n, d)), dtype)
    dl, rdl = _rounded(rng.standard_normal((nb, W - 1, d)), dtype)
    fr = None if frames is None else torch.tensor(frames, dtype=torch.int32, device=_dev())
    leaves = [t.requires_grad_(True) for t in (x, w, b, st) if t is not None]
    out = sed_amd.causal_conv(x, w, b, activation="silu" if silu else None, frames=fr, reverse=reverse, state=st, return_state=last)
    y, hl = out if last else (out, None)
    o = S.conv(rx, rw, rb, silu, frames, reverse, rst, rdy, rdl if last else None)
    # W + 1 additions, the activation (its argument's rounding, 16u), the sums over a run of 64 rows, then over the runs
    few, many = U * (2 * W + 32), U * (2 * W + 150 + nb * n / 8)
    _close(y, o["y"][0], few * o["y"][1], "y")
    if last:
        assert np.array_equal(hl.detach().double().cpu().numpy(), o["last"][0])
    grads = torch.autograd.grad([y, hl] if last and hl.requires_grad else [y], leaves, [dy, dl] if last and hl.requires_grad else [dy])
    names = ["dx", "dw"] + (["db"] if bias else []) + (["dstate"] if state else [])
    for k, got in zip(names, grads):
        _close(got, o[k][0], (many if k in ("dw", "db") else 2 * few) * o[k][1], k)


@pytest.mark.parametrize("dtype", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("nb,n,d,W", ((1, 1, 1, 4), (2, 3, 5, 4), (1, 8, 8, 4), (2, 17, 24, 4), (1, 65, 16, 3), (3, 130, 40, 2), (1, 200, 7, 4),
                                      (2, 31, 64, 1), (1, 40, 12, 8), (1, 2, 8, 8), (2, 9, 33, 5)))
def test_conv_sizes(nb, n, d, W, dtype):
    _conv_case(nb, n, d, W, DTYPES[dtype], seed=n + d, state=n % 2 == 0)


@pytest.mark.parametrize("dtype", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("nb,n,d,W", ((2, 97, 256, 4), (1, 200, 260, 3), (1, 65, 516, 2), (2, 130, 260, 8), (1, 70, 256, 5), (1, 9, 256, 1), (3, 1, 768, 7)))
def test_conv_rows_of_whole_vectors(nb, n, d, W, dtype):
    _conv_case(nb, n, d, W, DTYPES[dtype], seed=n + d, state=n % 2 == 0)
    _conv_case(nb, n, d, W, DTYPES[dtype], seed=n + d + 1, state=True, reverse=True, silu=False, frames=[n - n // 3, 0, n][:nb])


@pytest.mark.parametrize("d,W,dtype", ((1, 4, torch.float32), (1, 6, torch.bfloat16), (256, 4, torch.bfloat16), (256, 8, torch.bfloat16), (256, 8, torch.float32)))
def test_conv_batches_that_fill_the_card(d, W, dtype):
    """Runs of the longest kind (2100 clips of two): all clips but two are zeros, so that those two are the weights' gradient."""
    import sed_amd
    nb, n, pick = 2100, 70, [3, 2099]
    rng = np.random.default_rng(d + W)
    x, rx = _rounded(rng.standard_normal((2, n, d)), dtype)
    dy, rdy = _rounded(rng.standard_normal((2, n, d)), dtype)
    w, rw = _rounded(rng.standard_normal((d, W)), torch.float32)
    b, rb = _rounded(rng.standard_normal(d), torch.float32)
    bx, bdy = (torch.zeros(nb, n, d, dtype=dtype, device=_dev()) for _ in range(2))
    bx[pick], bdy[pick] = x, dy
    fr = torch.full((nb,), n, dtype=torch.int32, device=_dev())
    fr[3] = 67
    leaves = [t.requires_grad_(True) for t in (bx, w, b)]
    y = sed_amd.causal_conv(bx, w, b, activation="silu", frames=fr)
    o = S.conv(rx, rw, rb, True, [67, n], False, None, rdy, None)
    few, many = U * (2 * W + 32), U * (2 * W + 150 + 2 * n / 8)  # as in every case: a zero clip adds nothing to a sum
    _close(y[pick], o["y"][0], few * o["y"][1], "y")
    dx, dw, db = torch.autograd.grad(y, leaves, bdy)
    _close(dx[pick], o["dx"][0], 2 * few * o["dx"][1], "dx")
    _close(dw, o["dw"][0], many * o["dw"][1], "dw")
    _close(db, o["db"][0], many * o["db"][1], "db")
    rest = torch.ones(nb, dtype=torch.bool)
    rest[pick] = False
    assert (dx[rest.to(dx.device)] == 0).all()


@pytest.mark.parametrize("reverse", (False, True))
def test_conv_own_lengths(reverse):
    for dtype in (torch.float32, torch.bfloat16):
        _conv_case(6, 70, 16, 4, dtype, reverse=reverse, state=True, frames=[70, 0, 1, 2, 33, 64])
        _conv_case(3, 20, 5, 8, dtype, reverse=reverse, state=False, frames=[0, 3, 20], silu=False, bias=False)
    _conv_case(2, 20, 16, 4, torch.float32, reverse=reverse, last=False)


@pytest.mark.parametrize("W", range(1, 9))
@pytest.mark.parametrize("d", (3, 256))
def test_conv_infinities_reach_their_window_only(W, d):
    import sed_amd
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(W)
    x, dy = (torch.randn(2, 90, d, generator=g, device=dev) for _ in range(2))
    w = torch.randn(d, W, generator=g, device=dev)
    got = []
    for bad in (False, True):
        v, e = x.clone(), dy.clone()
        if bad:
            v[0, 40], e[1, 30] = float("inf"), float("nan")
        v.requires_grad_(True)
        y = sed_amd.causal_conv(v, w, activation=None)
        got.append([y, *torch.autograd.grad(y, [v], e)])
    clean, dirty = got
    away = torch.ones(90, dtype=torch.bool, device=dev)
    away[40:40 + W] = False
    assert torch.equal(clean[0][0][away], dirty[0][0][away]) and torch.equal(clean[0][1], dirty[0][1])
    assert not dirty[0][0][~away].isfinite().any()
    away = torch.ones(90, dtype=torch.bool, device=dev)
    away[30 - W + 1:31] = False
    assert torch.equal(clean[1][0], dirty[1][0]) and torch.equal(clean[1][1][away], dirty[1][1][away])
    st = torch.randn(3, W - 1, d, generator=g, device=dev)
    rows = torch.randn(12, 3, d, generator=g, device=dev)
    rows[0, 1] = float("inf")
    ys = [sed_amd.causal_conv_step(st, t, w) for t in rows]
    assert all(t.isfinite().all() for t in ys[W:]) and st.isfinite().all()


def test_conv_rows_behind_are_neither_read_nor_kept():
    import sed_amd
    dev = _dev()
    x = torch.randn(2, 40, 16, device=dev, dtype=torch.bfloat16)
    fr = torch.tensor([13, 0], dtype=torch.int32, device=dev)
    w, dy = torch.randn(16, 4, device=dev), torch.randn(2, 40, 16, device=dev, dtype=torch.bfloat16)
    got = []
    for fill in (0.0, float("nan")):
        v, g = x.clone(), dy.clone()
        v[0, 13:], v[1], g[0, 13:], g[1] = fill, fill, fill, fill
        v.requires_grad_(True)
        wl = w.clone().requires_grad_(True)
        y, last = sed_amd.causal_conv(v, wl, activation="silu", frames=fr, return_state=True)
        got.append([y, last, *torch.autograd.grad(y, [v, wl], g)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[1][0][0, 13:] == 0).all() and (got[1][2][1] == 0).all()


@pytest.mark.parametrize("nb,d,W", ((1, 1, 4), (5, 33, 4), (3, 64, 3), (2, 8, 2), (2, 16, 1), (2, 24, 8)))
def test_conv_step_follows_the_whole(nb, d, W):
    """Frame by frame, the state in place: the same bits as the whole sequence (each output is formed by the same additions)."""
    import sed_amd
    dev = _dev()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, st = torch.randn(nb, 9, d, device=dev).to(dtype), torch.randn(nb, W - 1, d, device=dev).to(dtype)
        w, b = torch.randn(d, 1, W, device=dev), torch.randn(d, device=dev)
        y, last = sed_amd.causal_conv(x, w, b, activation="silu", state=st, return_state=True)
        ys = [sed_amd.causal_conv_step(st, x[:, t], w, b, activation="silu") for t in range(9)]
        assert torch.equal(torch.stack(ys, 1), y) and torch.equal(st, last)


def test_conv_views_and_refusals():
    import sed_amd
    dev = _dev()
    base = torch.randn(2, 30, 41, device=dev)
    w = torch.randn(16, 4, device=dev)
    for v in (base[..., :16], base[..., 1:17], base.transpose(1, 2)[:, :16], base[:1, :, :16].expand(2, 30, 16)):
        assert torch.equal(sed_amd.causal_conv(v, w[:v.shape[2]] if v.shape[2] < 16 else torch.cat([w] * 3)[:v.shape[2]], activation="silu"),
                           sed_amd.causal_conv(v.contiguous(), w[:v.shape[2]] if v.shape[2] < 16 else torch.cat([w] * 3)[:v.shape[2]], activation="silu"))
    x = base[..., :16].contiguous()
    for err, kw in ((ValueError, dict(weight=w[:15])), (ValueError, dict(weight=torch.zeros(16, 9, device=dev))), (ValueError, dict(weight=torch.zeros(16, 0, device=dev))),
                    (ValueError, dict(weight=w, activation="gelu")), (TypeError, dict(weight=w.int())), (ValueError, dict(weight=w, bias=w[:, 0][:8])),
                    (ValueError, dict(weight=w, state=torch.zeros(2, 4, 16, device=dev))), (TypeError, dict(weight=w, state=torch.zeros(2, 3, 16, device=dev).half())),
                    (TypeError, dict(weight=w, frames=torch.zeros(2, dtype=torch.int64, device=dev)))):
        with pytest.raises(err):
            sed_amd.causal_conv(x, **kw)
    with pytest.raises(ValueError):
        sed_amd.causal_conv_step(torch.zeros(3, 2, 16, device=dev).transpose(0, 1), x[:, 0], w)
    with pytest.raises(RuntimeError):
        sed_amd.causal_conv_step(torch.zeros(2, 3, 16, device=dev), x[:, 0], w.clone().requires_grad_(True))


# ---- group norm ---------------------------------------------------------------------------------------------------------


def _norm_case(shape, groups, dtype, act="silu", seed=0, affine=True, frames=None, mean=0.0, spread=1.0, grad=True):
    import sed_amd
    rng = np.random.default_rng(seed)
    c = shape[-1]
    x, rx = _rounded(mean + spread * rng.standard_normal(shape) * rng.uniform(0.5, 2, c), dtype)
    w, rw = _rounded(1 + 0.3 * rng.standard_normal(c), torch.float32) if affine else (None, None)
    b, rb = _rounded(0.3 * rng.standard_normal(c), torch.float32) if affine else (None, None)
    dy, rdy = _rounded(rng.standard_normal(shape), dtype)
    fr = None if frames is None else torch.tensor(frames, dtype=torch.int32, device=_dev())
    leaves = [t.requires_grad_(grad) for t in (x, w, b) if t is not None]
    four = (shape[0], shape[1], int(np.prod(shape[2:-1])), c)
    o, clear = S.group_norm(rx.reshape(four), groups, rw, rb, 1e-5, act, frames, rdy.reshape(four))
    assert act != "relu" or clear > 1  # no value sits where its own error could move it over relu's corner
    y = sed_amd.group_norm_act(x, groups, w, b, activation=act, frames=fr)
    _close(y, o["y"][0].reshape(shape), o["y"][1].reshape(shape), "y")
    if grad:
        grads = torch.autograd.grad(y, leaves, dy)
        for k, got in zip(("dx", "dw", "db"), grads):
            s = shape if k == "dx" else (c,)
            _close(got, o[k][0].reshape(s), o[k][1].reshape(s), k)


@pytest.mark.parametrize("dtype", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("shape,groups", (((1, 1, 1), 1), ((2, 1, 8), 2), ((1, 3, 5, 12), 3), ((2, 40, 16), 4), ((1, 101, 7, 32), 8), ((3, 65, 24), 1),
                                          ((1, 33, 40), 40), ((2, 9, 3, 2, 6), 2), ((1, 70, 2064), 3), ((1, 5, 4104), 2), ((1, 400, 257), 1), ((2, 130, 64), 32)))
def test_norm_sizes(shape, groups, dtype):
    _norm_case(shape, groups, DTYPES[dtype], act=(None, "silu", "gelu")[sum(shape) % 3], seed=sum(shape))


@pytest.mark.parametrize("act", (None, "silu", "gelu"))
@pytest.mark.parametrize("shape,groups", (((1, 700, 1, 256), 8), ((2, 433, 3, 64), 8), ((1, 1501, 2064), 3), ((1, 901, 33), 3)))
def test_norm_long_walks(shape, groups, act):
    """Blocks whose lanes meet many rows: whole batches of rows, a rest behind them, and blocks of uneven parts."""
    for dtype in (torch.float32, torch.bfloat16):
        _norm_case(shape, groups, dtype, act=act, seed=7, frames=[shape[1] - 5, 2][:shape[0]] if shape[3:] else None)


@pytest.mark.parametrize("dtype", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("shape,groups", (((1, 1, 8), 1), ((2, 1, 1, 4), 1), ((3, 7, 24), 1), ((1, 101, 3, 32), 8), ((2, 33, 96), 2), ((600, 3, 16), 2),
                                          ((1, 4, 4096), 1), ((1, 9, 6156), 3), ((1, 8, 4104), 2), ((130, 40, 16), 4), ((5, 257, 48), 1), ((1, 2049, 4), 1)))
def test_norm_groups_held_whole(shape, groups, dtype):
    """Groups that one workgroup holds, at the ends of what it holds, with lengths of their own and without."""
    n = shape[1]
    _norm_case(shape, groups, DTYPES[dtype], act="silu", seed=sum(shape), frames=[(n, 0, 1, n - 1, n + 3, -1)[i % 6] for i in range(shape[0])])
    _norm_case(shape, groups, DTYPES[dtype], act=None, seed=n, mean=100.0 if dtype == "fp32" else 3.0, affine=n % 2 == 0)


@pytest.mark.parametrize("act", (None, "silu", "gelu"))
@pytest.mark.parametrize("shape,groups,frames", (((3, 9000, 32), 4, (9000, 5, 4501)), ((1, 8300, 16), 2, None), ((2, 900, 3, 30), 6, (1, 900)), ((20, 1100, 128), 4, None)))
def test_norm_groups_walked_twice(shape, groups, frames, act):
    """Groups beyond one workgroup, whole vectors and single channels, with blocks that have no place and blocks of many rows."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _norm_case(shape, groups, dtype, act=act, seed=17, frames=frames)


@pytest.mark.parametrize("shape,groups", (((1, 2000, 64), 1), ((1, 300, 1200), 1), ((2, 700, 520), 1), ((1, 150, 3, 2052), 1), ((1, 6000, 40), 2)))
def test_norm_groups_of_many_blocks(shape, groups):
    """Blocks and channels a group that are joined by a launch of their own; clips that leave blocks without a place."""
    for dtype in (torch.float32, torch.bfloat16):
        _norm_case(shape, groups, dtype, act="silu", seed=sum(shape))
        _norm_case(shape, groups, dtype, act=None, seed=3, frames=[5, shape[1]][:shape[0]], mean=10.0)


@pytest.mark.parametrize("act", (None, "silu", "relu", "gelu"))
@pytest.mark.parametrize("affine", (True, False))
def test_norm_activations(act, affine):
    _norm_case((2, 21, 3, 16), 4, torch.float32, act=act, seed=1, affine=affine)
    _norm_case((2, 21, 3, 16), 4, torch.bfloat16, act=act, seed=2, affine=affine)


def test_norm_own_lengths_and_far_means():
    for dtype in (torch.float32, torch.bfloat16):
        _norm_case((5, 70, 2, 16), 4, dtype, seed=3, frames=[70, 0, 1, 33, 64])
    # a mean a thousand spreads away: the bound follows the mean (its rounding moves every value), the variance keeps its digits
    _norm_case((2, 300, 16), 2, torch.float32, act=None, seed=4, mean=1000.0)
    _norm_case((2, 300, 16), 2, torch.float32, act="silu", seed=5, spread=1e-4)


def test_norm_rows_behind_are_neither_read_nor_kept():
    import sed_amd
    dev = _dev()
    x, dy = torch.randn(3, 40, 2, 16, device=dev), torch.randn(3, 40, 2, 16, device=dev)
    fr = torch.tensor([13, 0, 40], dtype=torch.int32, device=dev)
    got = []
    for fill in (0.0, float("nan")):
        v, g = x.clone(), dy.clone()
        v[0, 13:], v[1], g[0, 13:], g[1] = fill, fill, fill, fill
        v.requires_grad_(True)
        w = torch.ones(16, device=dev, requires_grad=True)
        y = sed_amd.group_norm_act(v, 4, w, activation="gelu", frames=fr)
        got.append([y, *torch.autograd.grad(y, [v, w], g)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[1][0][0, 13:] == 0).all() and (got[1][0][1] == 0).all()


def test_norm_refusals():
    import sed_amd
    dev = _dev()
    x = torch.zeros(2, 4, 8, device=dev)
    for err, kw in ((ValueError, dict(groups=3)), (ValueError, dict(groups=0)), (ValueError, dict(groups=2, activation="tanh")), (ValueError, dict(groups=2, eps=-1.0)),
                    (ValueError, dict(groups=2, weight=torch.zeros(7, device=dev))), (TypeError, dict(groups=2, bias=torch.zeros(8, device=dev, dtype=torch.int32))),
                    (TypeError, dict(groups=2, frames=torch.zeros(2, device=dev)))):
        with pytest.raises(err):
            sed_amd.group_norm_act(x, **kw)
    with pytest.raises(ValueError):
        sed_amd.group_norm_act(x[0], 2)
    with pytest.raises(TypeError):
        sed_amd.group_norm_act(x.double(), 2)
    with pytest.raises(ValueError):
        sed_amd.group_norm_act(torch.zeros(65536, 1, 2, device=dev), 1)


# ---- as they are used ---------------------------------------------------------------------------------------------------


def _block(sed, p, img, frames, reverse=False):
    """Feature map -> group norm -> rows -> convolution -> recurrence -> class probabilities, with plain products in between."""
    h = sed.group_norm_act(img, 4, p["gw"], p["gb"], activation="silu", frames=frames)
    h = h.flatten(2) @ p["w_in"]
    x, z = h.chunk(2, -1)
    x = sed.causal_conv(x, p["cw"], p["cb"], activation="silu", frames=frames, reverse=reverse)
    dbc = x @ p["w_x"]
    dt, B, C = dbc[..., :48], dbc[..., 48:64], dbc[..., 64:]
    y = sed.gated_scan(x, dt, p["A"], B, C, D=p["D"], z=z, dt_bias=p["bias"], softplus=True, frames=frames, reverse=reverse)
    return torch.sigmoid(y @ p["w_out"])


def _block_params(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    return {"gw": 1 + 0.1 * r(8), "gb": 0.1 * r(8), "w_in": r(32, 96) / 6, "cw": r(48, 4) / 2, "cb": 0.1 * r(48), "w_x": r(48, 80) / 7,
            "A": -torch.rand(48, 16, generator=g, device=dev) * 4, "D": r(48), "bias": 0.1 * r(48) - 2, "w_out": r(48, 5) / 7}


def test_block_trains_and_feeds_the_decoder():
    import sed_amd
    dev = _dev()
    p = {k: v.requires_grad_(True) for k, v in _block_params(dev).items()}
    img = torch.randn(3, 60, 4, 8, device=dev)
    frames = torch.tensor([60, 31, 7], dtype=torch.int32, device=dev)
    probs = _block(sed_amd, p, img, frames)
    assert probs.shape == (3, 60, 5)
    grads = torch.autograd.grad((probs * torch.linspace(0, 1, 5, device=dev)).sum(), list(p.values()))
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    # each clip alone, without padding, gives its rows of the batch: same arithmetic up to the order of sums
    for b, n in enumerate((60, 31, 7)):
        with torch.no_grad():
            alone = _block(sed_amd, p, img[b:b + 1, :n].contiguous(), None)
        assert torch.allclose(alone[0], probs[b, :n].detach(), rtol=0, atol=2e-5)
    # the probabilities go to the decoders as any detector's do
    runs, counts = sed_amd.decode.threshold_runs(probs.detach().contiguous(), 0.5, None)
    p_host = probs.detach().cpu().numpy()
    for b in range(3):
        for c in range(5):
            act = np.concatenate([[0], (p_host[b, :, c] > 0.5).astype(int), [0]])
            want = np.stack([np.flatnonzero(np.diff(act) == k) for k in (1, -1)], 1)
            assert int(counts[b, c]) == len(want) and np.array_equal(runs[b, c, :len(want)].cpu().numpy(), want)


@pytest.mark.parametrize("op", ("scan", "conv", "norm"))
def test_replayed_graphs_follow_eager_calls(op):
    """Forward and gradient captured into a graph, replayed on new data with eager work in between."""
    import sed_amd
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    static = {"x": r(2, 70, 32), "dy": r(2, 70, 32)}
    fixed = {"dt": r(2, 70, 32) - 2, "A": -torch.rand(32, 16, device=dev) * 3, "B": r(2, 70, 16), "C": r(2, 70, 16), "w": r(32, 4)}

    def call(x, dy):
        x = x.detach().requires_grad_(True)
        if op == "scan":
            y = sed_amd.gated_scan(x, fixed["dt"], fixed["A"], fixed["B"], fixed["C"], softplus=True)
        elif op == "conv":
            y = sed_amd.causal_conv(x, fixed["w"], activation="silu")
        else:
            y = sed_amd.group_norm_act(x, 4, activation="gelu")
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(**static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(**static)
        graphs.append((graph, out))
    for k in range(3):
        new = {n: r(*t.shape) for n, t in static.items()}
        for n, t in static.items():
            t.copy_(new[n])
        want = call(**new)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_replayed_steps_follow_eager_steps():
    """One frame of both one-frame forms in a graph: every replay moves the states on by a frame, as eager calls do."""
    import sed_amd
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    A, w = -torch.rand(24, 16, generator=g, device=dev) * 3, r(24, 4)
    frame = {"x": r(5, 24).bfloat16(), "dt": (r(5, 24) - 2).bfloat16(), "B": r(5, 16).bfloat16(), "C": r(5, 16).bfloat16()}
    states = [[r(5, 3, 24).bfloat16(), r(5, 24, 16)] for _ in range(2)]
    states[1] = [t.clone() for t in states[0]]

    def call(v, s):
        x = sed_amd.causal_conv_step(s[0], v["x"], w, activation="silu")
        return sed_amd.gated_scan_step(s[1], x, v["dt"], A, v["B"], v["C"], softplus=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(frame, [t.clone() for t in states[0]])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(frame, states[0])
    for _ in range(4):
        for t in frame.values():
            t.copy_(r(*t.shape))
        want = call(frame, states[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(*states))


def test_lengths_out_of_range_are_clamped():
    import sed_amd
    dev = _dev()
    x, A, bc, w = torch.randn(3, 20, 8, device=dev), -torch.rand(8, 4, device=dev), torch.randn(3, 20, 4, device=dev), torch.randn(8, 4, device=dev)
    odd, even = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([-7, 2 ** 31 - 1, 5], [0, 20, 5]))
    for call in (lambda f: sed_amd.gated_scan(x, x, A, bc, bc, softplus=True, frames=f), lambda f: sed_amd.causal_conv(x, w, frames=f),
                 lambda f: sed_amd.group_norm_act(x, 2, frames=f)):
        assert torch.equal(call(odd), call(even))


def test_parameters_of_another_type():
    """bf16 parameters are read as the fp32 values they hold; their gradients are the fp32 ones, rounded to bf16."""
    import sed_amd
    dev = _dev()
    x, bc = torch.randn(2, 40, 16, device=dev), torch.randn(2, 40, 8, device=dev)
    small = {"A": -torch.rand(16, 8, device=dev), "D": torch.randn(16, device=dev), "dt_bias": torch.randn(16, device=dev) - 2,
             "w": torch.randn(16, 4, device=dev), "b": torch.randn(16, device=dev)}
    got = []
    for t in (torch.bfloat16, torch.float32):
        p = {k: v.bfloat16().to(t).requires_grad_(True) for k, v in small.items()}
        y = sed_amd.gated_scan(x, x, p["A"], bc, bc, D=p["D"], dt_bias=p["dt_bias"], softplus=True)
        y = y + sed_amd.causal_conv(x, p["w"], p["b"], activation="silu") + sed_amd.group_norm_act(x, 4, p["D"], p["b"], activation="silu")
        got.append([y.detach(), *torch.autograd.grad(y.sum(), list(p.values()))])
    assert torch.equal(got[0][0], got[1][0])
    for k, (a, b) in zip(small, zip(got[0][1:], got[1][1:])):
        assert a.dtype == torch.bfloat16
        if k in ("A", "dt_bias", "w"):  # D and b add two gradients, each rounded
            assert torch.equal(a, b.bfloat16()), k


def test_two_streams_and_repeated_calls_agree():
    import sed_amd
    dev = _dev()
    dev_in, _, _ = _scan_inputs(2, 200, 64, 1, 16, torch.bfloat16, 9)
    args = dict(dev_in)
    base = [args.pop(k) for k in ("x", "dt", "A", "B", "C")]
    leaves = [t.requires_grad_(True) for t in base]
    dy = torch.randn(2, 200, 64, device=dev, dtype=torch.bfloat16)

    def call():
        y = sed_amd.gated_scan(*leaves, **args, softplus=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_past_32_bits():
    """Clips more than 2^31 elements apart, and outputs longer than that: as the same clips alone."""
    import sed_amd
    dev = _dev()
    far = (1 << 31) + 64
    store = torch.zeros(far + 64 * 8, dtype=torch.bfloat16, device=dev)
    x = store.as_strided((2, 64, 8), (far, 8, 1))
    x.copy_(torch.randn(2, 64, 8, device=dev))
    A, bc, w = -torch.rand(8, 4, device=dev), torch.randn(2, 64, 4, device=dev).bfloat16(), torch.randn(8, 4, device=dev)
    for b in range(2):
        assert torch.equal(sed_amd.gated_scan(x, x, A, bc, bc, softplus=True)[b], sed_amd.gated_scan(x.contiguous(), x.contiguous(), A, bc, bc, softplus=True)[b])
    assert torch.equal(sed_amd.causal_conv(x, w, activation="silu"), sed_amd.causal_conv(x.contiguous(), w, activation="silu"))
    del store, x
    n = (1 << 31) // (64 * 512) + 2
    x = torch.randn(64, 64, 512, device=dev).bfloat16().repeat((n + 63) // 64, 1, 1)[:n]
    assert x.numel() > 1 << 31
    w, A = torch.randn(512, 4, device=dev), -torch.rand(512, 1, device=dev)
    assert torch.equal(sed_amd.causal_conv(x, w, activation="silu")[-2:], sed_amd.causal_conv(x[-2:].contiguous(), w, activation="silu"))
    bc = torch.randn(n, 64, 1, device=dev).bfloat16()
    y = sed_amd.gated_scan(x, x, A, bc, bc, softplus=True)
    last = slice(n - 1024, n)  # enough clips that neither call cuts them
    assert torch.equal(y[last], sed_amd.gated_scan(x[last].contiguous(), x[last].contiguous(), A, bc[last].contiguous(), bc[last].contiguous(), softplus=True))
    del y
    x = x.view(n // 2, 128, 512)
    y = sed_amd.group_norm_act(x, 2, activation="silu")[-2:]
    alone = sed_amd.group_norm_act(x[-2:].contiguous(), 2, activation="silu")
    # sums cut differently: equal before the rounding to 2^-15 of the values, so at most one step of bf16 apart
    assert ((y.float() - alone.float()).abs() <= 2.0 ** -7 * alone.float().abs() + 1e-4).all()
