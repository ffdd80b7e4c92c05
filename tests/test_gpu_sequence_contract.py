"""GPU tests of what the sequence operators promise beside their values on ordinary data: derivatives that would be wrong are refused,
limits and strides are those the documentation names, extreme parameters and recordings keep their digits."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import sequence as S
from test_gpu_sequence import NAMES, U, _close, _dev, _rounded, _scan_bound, _scan_inputs

pytestmark = pytest.mark.gpu


def _step_inputs(nb=2, d=16, ns=4, W=4):
    g = torch.Generator(device=_dev()).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=_dev())  # noqa: E731
    return {"x": r(nb, 9, d), "A": -torch.rand(d, ns, generator=g, device=_dev()), "bc": r(nb, 9, ns), "w": r(d, W), "conv": r(nb, W - 1, d), "scan": r(nb, d, ns)}


def test_a_step_on_a_saved_state_is_noticed():
    """causal_conv's gradient reads the state it was given: a step that moves it on in between is an error, as for torch's own operators."""
    import sed_amd
    v = _step_inputs()
    w = v["w"].clone().requires_grad_(True)
    for activation in (None, "silu"):
        state = v["conv"].clone()
        y = sed_amd.causal_conv(v["x"], w, activation=activation, state=state)
        with torch.no_grad():
            sed_amd.causal_conv_step(state, v["x"][:, 0], w, activation=activation)
        with pytest.raises(RuntimeError, match="inplace operation"):
            torch.autograd.grad(y.sum(), w)
    # any other operator that keeps the state is told as well
    for start, step in ((v["conv"], lambda s: sed_amd.causal_conv_step(s, v["x"][:, 0], v["w"])),
                        (v["scan"], lambda s: sed_amd.gated_scan_step(s, v["x"][:, 0], v["x"][:, 0], v["A"], v["bc"][:, 0], v["bc"][:, 0]))):
        state, scale = start.clone(), torch.ones((), device=_dev(), requires_grad=True)
        y = (scale * state).sum()
        with torch.no_grad():
            step(state)
        with pytest.raises(RuntimeError, match="inplace operation"):
            torch.autograd.grad(y, scale)


def test_a_step_behind_gated_scan_leaves_its_gradient():
    """gated_scan's gradient does not read the state in front: the stream may go on before it is taken."""
    import sed_amd
    v = _step_inputs()
    got = []
    for go_on in (False, True):
        x, state = v["x"].clone().requires_grad_(True), v["scan"].clone()
        y = sed_amd.gated_scan(x, v["x"], v["A"], v["bc"], v["bc"], softplus=True, state=state)
        if go_on:
            with torch.no_grad():
                sed_amd.gated_scan_step(state, v["x"][:, 0], v["x"][:, 0], v["A"], v["bc"][:, 0], v["bc"][:, 0], softplus=True)
        got.append(torch.autograd.grad(y.sum(), x)[0])
    assert torch.equal(*got)


def test_steps_in_inference_mode():
    import sed_amd
    v = _step_inputs()
    want = [v["conv"].clone(), v["scan"].clone()]
    step = lambda s: [sed_amd.causal_conv_step(s[0], v["x"][:, 0], v["w"]),  # noqa: E731
                      sed_amd.gated_scan_step(s[1], v["x"][:, 0], v["x"][:, 0], v["A"], v["bc"][:, 0], v["bc"][:, 0], softplus=True)]
    ys = step(want)
    with torch.inference_mode():
        states = [v["conv"].clone(), v["scan"].clone()]
        got = step(states)
    assert all(torch.equal(a, b) for a, b in zip(ys + want, got + states))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require grad; its tangent must not get lost without a word."""
    import sed_amd
    v = _step_inputs()
    calls = {
        "gated_scan": (sed_amd.gated_scan, dict(x=v["x"], dt=v["x"], A=v["A"], B=v["bc"], C=v["bc"], D=v["w"][:, 0], z=v["x"], dt_bias=v["w"][:, 1], state=v["scan"])),
        "gated_scan_step": (sed_amd.gated_scan_step, dict(state=v["scan"], x=v["x"][:, 0], dt=v["x"][:, 0], A=v["A"], B=v["bc"][:, 0], C=v["bc"][:, 0],
                                                          D=v["w"][:, 0], z=v["x"][:, 0], dt_bias=v["w"][:, 1])),
        "causal_conv": (sed_amd.causal_conv, dict(x=v["x"], weight=v["w"], bias=v["w"][:, 0], state=v["conv"])),
        "causal_conv_step": (sed_amd.causal_conv_step, dict(state=v["conv"], x=v["x"][:, 0], weight=v["w"], bias=v["w"][:, 0])),
        "group_norm_act": (sed_amd.group_norm_act, dict(x=v["x"], weight=v["w"][:, 0], bias=v["w"][:, 1], groups=4)),
    }
    for name, (call, kw) in calls.items():
        for k in (k for k, t in kw.items() if torch.is_tensor(t)):
            for grad in (False, True):
                if grad and "step" in name:
                    continue
                before = kw[k].clone()
                with forward_ad.dual_level():
                    dual = forward_ad.make_dual(kw[k].clone().requires_grad_(grad), torch.ones_like(kw[k]))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(**(kw | {k: dual}))
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                        call(**(kw | {k: dual}))
                    assert torch.equal(forward_ad.unpack_dual(dual).primal, before), (name, k)
        with forward_ad.dual_level():  # without a tangent the call is an ordinary one
            call(**{k: t.clone() if torch.is_tensor(t) else t for k, t in kw.items()})


def test_forward_over_reverse_is_refused():
    import sed_amd
    v = _step_inputs()
    for call in (lambda x: sed_amd.gated_scan(x, v["x"], v["A"], v["bc"], v["bc"], softplus=True), lambda x: sed_amd.causal_conv(x, v["w"]),
                 lambda x: sed_amd.group_norm_act(x, 4)):
        x = v["x"].clone().requires_grad_(True)
        y = call(x)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    for state, call in ((v["scan"], lambda s: sed_amd.gated_scan(v["x"], v["x"], v["A"], v["bc"], v["bc"], softplus=True, state=s, return_state=True)),
                        (v["conv"], lambda s: sed_amd.causal_conv(v["x"], v["w"], state=s, return_state=True))):
        state = state.clone().requires_grad_(True)
        last = call(state)[1]
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(last, state, forward_ad.make_dual(torch.ones_like(last), torch.ones_like(last)))


@pytest.mark.parametrize("ns", (1, 3, 8, 16, 32))
@pytest.mark.parametrize("nb,n,d,g,frames", ((2, 21, 5, 1, (21, 10)), (3, 70, 6, 3, None), (2, 900, 12, 1, (3, 900)), (1, 5000, 4, 1, None)))
def test_scan_forgets_at_once_with_the_lowest_decay(nb, n, d, g, frames, ns):
    """A of the type's lowest value: every frame starts from zero.  exp(delta A) is exactly zero for A = -10^6 as well (delta >= 0.01), so
    both give the same bits, in lanes without a channel, in frames behind a clip's own that share its tile, and over chunks without frames."""
    import sed_amd
    dev, _, rng = _scan_inputs(nb, n, d, g, ns, torch.float32, ns, softplus=False, frames=frames, state=True)
    dev["dt"] = dev["dt"].clamp(min=0.01)
    dy = torch.from_numpy(rng.standard_normal((nb, n, d)).astype(np.float32)).to(_dev())
    dl = torch.from_numpy(rng.standard_normal((nb, d, ns)).astype(np.float32)).to(_dev())
    for reverse in (False, True):
        got = []
        for low in (-1e6, torch.finfo(torch.float32).min):
            A = dev["A"].clone()
            A[1::2] = low
            A[:, -1] = low
            leaves = {k: t.detach().clone().requires_grad_(True) for k, t in (dev | {"A": A}).items() if k != "frames"}
            args = dict(leaves)
            y, last = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, frames=dev.get("frames"), reverse=reverse, return_state=True)
            got.append([y, last, *torch.autograd.grad([y, last], list(leaves.values()), [dy, dl])])
        for name, a, b in zip(["y", "last"] + list(leaves), *got):
            assert a.isfinite().all() and torch.equal(a, b), (name, reverse)


@pytest.mark.parametrize("ns", (1, 4, 8, 16, 32))
@pytest.mark.parametrize("n,d", ((900, 8), (900, 7), (9000, 4)))
def test_scan_growth_over_a_chunk_meets_a_zero_state(n, d, ns):
    """exp(delta A) > 1 in every frame, x only in the last one and dy only in the first: nothing is there that could grow, so every
    output is finite although the product of the growths is not."""
    import sed_amd
    dev, ref, rng = _scan_inputs(2, n, d, 1, ns, torch.float32, n + ns, softplus=False, bias=False)
    dy = np.zeros((2, n, d))
    dy[:, 0] = rng.standard_normal((2, d))
    ref["x"][:, :-1] = 0
    ref["A"] = np.full((d, ns), 8.0)
    ref["dt"] = np.full((2, n, d), 1.0)  # e^8 a frame: 16 frames pass the range of fp32
    dev = {k: torch.from_numpy(a.astype(np.float32)).to(_dev()).requires_grad_(True) for k, a in ref.items()}
    dy, rdy = _rounded(dy, torch.float32)
    args = dict(dev)
    y, last = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, return_state=True)
    grads = dict(zip(dev, torch.autograd.grad(y, list(dev.values()), dy)))
    # By the definition: only the last frame has a state, delta B x, and only the first one a gradient behind it, C gy.
    x, B, C, D, z = (ref[k] for k in ("x", "B", "C", "D", "z"))
    gate = z * S.sigmoid(z)
    h = x[:, -1, :, None] * B[:, -1, 0][:, None]
    want = {k: np.zeros_like(ref[k]) for k in ref}
    wy = np.zeros((2, n, d))
    pre = (h * C[:, -1, 0][:, None]).sum(-1) + D * x[:, -1]
    wy[:, -1] = pre * gate[:, -1]
    gy = (rdy * gate)[:, 0]
    want["x"][:, 0] = D * gy + (gy[..., None] * C[:, 0, 0][:, None] * B[:, 0, 0][:, None]).sum(-1)
    size = {k: np.zeros_like(ref[k]) for k in ref}
    size["x"][:, 0] = np.abs(D * gy) + np.abs(gy[..., None] * C[:, 0, 0][:, None] * B[:, 0, 0][:, None]).sum(-1)
    sy = np.zeros((2, n, d))
    sy[:, -1] = ((np.abs(h * C[:, -1, 0][:, None])).sum(-1) + np.abs(D * x[:, -1])) * np.abs(gate[:, -1])
    # sums of at most 34 terms, the gate's 100 u as in every case
    _close(y, wy, 200 * U * sy, "y")
    _close(last, h, 8 * U * np.abs(h), "last")
    for k in ref:  # h is zero where g is not and the other way round, but for the products above
        _close(grads[k], want[k], 200 * U * size[k], NAMES[k])


def test_scan_growth_over_a_chunk_meets_a_small_state():
    """A state of 1e-36 that grows by e^160 within 16 frames ends at 3e33: the growth alone, e^160, is beyond fp32."""
    import sed_amd
    nb, n, d, ns = 48, 96, 4, 4
    dev = _dev()
    dt = torch.zeros(nb, n, d, device=dev)
    for b in range(nb):  # wherever the chunks' borders are, some clips have the growth inside one
        dt[b, b:b + 16] = 10.0
    x, bc = torch.zeros(nb, n, d, device=dev), torch.ones(nb, n, ns, device=dev)
    state = torch.full((nb, d, ns), 1e-36, device=dev, requires_grad=True)
    few = lambda t: t.repeat(1, 40, 1)[:, :n * 40]  # noqa: E731
    for dt_, x_, bc_ in ((dt, x, bc), (torch.cat([dt, few(torch.zeros_like(dt))], 1), torch.cat([x, few(x)], 1), torch.cat([bc, few(bc)], 1))):
        y, last = sed_amd.gated_scan(x_, dt_, torch.ones(d, ns, device=dev), bc_, bc_, state=state, return_state=True)
        want = np.full((nb, d, ns), state.detach().flatten()[0].item() * np.exp(160.0))
        # 16 exponents of 10 (or one of 160), each off by 8 u of itself, and the decays' own rounding
        _close(last, want, U * (8 * 160 + 8 * 32) * want, "last")
        (g,) = torch.autograd.grad(last, state, torch.full_like(last, 1e-36))
        _close(g, want, U * (8 * 160 + 8 * 32) * want, "dstate")


@pytest.mark.parametrize("c,groups", ((129, 129), (129, 3)))
def test_norm_of_clips_that_begin_with_a_spike(c, groups):
    """A first frame a hundred spreads away in clips of which one lane walks 600 rows: the variance keeps its digits (100 u, the bound of
    every other case).  All clips but two are zeros."""
    import sed_amd
    nb, n, pick = 2048, 600, [5, 2047]
    rng = np.random.default_rng(c + groups)
    v = rng.standard_normal((2, n, c))
    v[:, 0] += 100.0
    x, rx = _rounded(v, torch.float32)
    dy, rdy = _rounded(rng.standard_normal((2, n, c)), torch.float32)
    bx, bdy = (torch.zeros(nb, n, c, device=_dev()) for _ in range(2))
    bx[pick], bdy[pick] = x, dy
    bx.requires_grad_(True)
    o, _ = S.group_norm(rx.reshape(2, n, 1, c), groups, None, None, 1e-5, None, None, rdy.reshape(2, n, 1, c))
    y = sed_amd.group_norm_act(bx, groups)
    _close(y[pick], o["y"][0].reshape(2, n, c), o["y"][1].reshape(2, n, c), "y")
    (dx,) = torch.autograd.grad(y, bx, bdy)
    _close(dx[pick], o["dx"][0].reshape(2, n, c), o["dx"][1].reshape(2, n, c), "dx")


def test_scan_batches_of_many_states():
    """Clips x states x channels past 2^26 in one call: all clips but two are zeros, so that those two are the parameters' gradient."""
    import sed_amd
    nb, n, d, ns, pick = 2100, 1, 1024, 32, [7, 2099]
    small, ref, rng = _scan_inputs(2, n, d, 1, ns, torch.bfloat16, 21)
    dy, rdy = _rounded(rng.standard_normal((2, n, d)), torch.bfloat16)
    big = {}
    for k, t in small.items():
        if t.shape[0] == 2 and t.dim() >= 3:
            big[k] = torch.zeros(nb, *t.shape[1:], dtype=t.dtype, device=_dev())
            big[k][pick] = t
        else:
            big[k] = t
    bdy = torch.zeros(nb, n, d, dtype=torch.bfloat16, device=_dev())
    bdy[pick] = dy
    leaves = {k: t.requires_grad_(True) for k, t in big.items()}
    args = dict(leaves)
    y, last = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, softplus=True, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), bdy)))
    o = S.scan(**ref, use_softplus=True, dy=rdy)
    _close(y[pick], o["y"][0], _scan_bound(o, "y", nb, n, d), "y")
    _close(last[pick], o["last"][0], _scan_bound(o, "last", nb, n, d), "last")
    for k, got in grads.items():
        _close(got[pick] if big[k].shape[0] == nb else got, o[NAMES[k]][0], _scan_bound(o, NAMES[k], nb, n, d), NAMES[k])
    with torch.no_grad():
        y20 = sed_amd.gated_scan(*(t.expand(-1, 3, *t.shape[2:]) if t.dim() >= 3 else t for t in (leaves[k] for k in ("x", "dt", "A", "B", "C"))), softplus=True)
        alone = sed_amd.gated_scan(*(t[pick].expand(-1, 3, *t.shape[2:]) if t.dim() >= 3 else t for t in (leaves[k] for k in ("x", "dt", "A", "B", "C"))), softplus=True)
    assert torch.allclose(y20[pick].float(), alone.float(), rtol=2.0 ** -7, atol=1e-5)


@pytest.mark.parametrize("reverse", (False, True))
@pytest.mark.parametrize("d", (6, 8))
def test_scan_of_one_frame_has_no_row_distance(d, reverse):
    """One frame whose frame axis has a stride past 2^26 (a time-major sequence's first frame): never used, so never refused."""
    import sed_amd
    dev, _, rng = _scan_inputs(3, 1, d, 1, 4, torch.float32, d, state=True)
    dy = torch.from_numpy(rng.standard_normal((3, 1, d)).astype(np.float32)).to(_dev())
    far = lambda t: t.as_strided(t.shape, (t.stride(0), (1 << 26) + 4, *t.stride()[2:]))  # noqa: E731
    got = []
    for wide in (lambda t: t, far):
        leaves = {k: t.detach().clone().requires_grad_(True) for k, t in dev.items()}
        args = {k: wide(t) if k in ("x", "dt", "B", "C", "z") else t for k, t in leaves.items()}
        y, last = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, softplus=True, reverse=reverse, return_state=True)
        got.append([y, last, *torch.autograd.grad(y, list(leaves.values()), wide(dy))])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    x = dev["x"]
    w = torch.from_numpy(rng.standard_normal((d, 4)).astype(np.float32)).to(_dev())
    assert torch.equal(sed_amd.causal_conv(far(x), w, reverse=reverse), sed_amd.causal_conv(x, w, reverse=reverse))


@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
@pytest.mark.parametrize("d,start", ((64, 0), (64, 1), (20, 0), (21, 3)))
@pytest.mark.parametrize("n,reverse", ((50, False), (300, True)))
def test_scan_gradients_of_views(n, reverse, d, start, dtype):
    """x, dt, z, B and C as slices of joint projections, dy with strides of its own: every gradient has the bits of the same call on copies."""
    import sed_amd
    t = {"fp32": torch.float32, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device=_dev()).manual_seed(n + d)
    r = lambda *s: torch.randn(s, generator=g, device=_dev())  # noqa: E731
    nb, ns = 3, 16
    rest = 4 * ((start + 3 * d + 2 * ns + 7) // 4)
    xzt, bc, bc4 = r(nb, n, rest).to(t), r(nb, n, 2 * ns + start).to(t), r(nb, n, 2, 3 * ns).to(t)
    A, D, bias = -4 * torch.rand(d, ns, generator=g, device=_dev()), r(d), 0.3 * r(d) - 2
    frames = torch.tensor([n, n // 3, 1], dtype=torch.int32, device=_dev())
    gaps = r(nb, n, 2 * d + 4 * start).to(t)
    time_major, wide = r(n, nb, d).to(t), r(nb, n + 5, d + 4).to(t)
    cases = ((xzt[..., start:start + d], xzt[..., start + d:start + 2 * d], xzt[..., start + 2 * d:start + 3 * d], bc[..., start:start + ns], bc[..., start + ns:], gaps[..., start:start + d]),
             (time_major.transpose(0, 1), wide[:, 5:, :d], wide[:, :n, 4:], bc[..., :ns], bc[..., ns:2 * ns], r(n, nb, d).to(t).transpose(0, 1)))
    if d % 2 == 0:
        cases += ((xzt[..., :d], wide[:, :n, :d], None, bc4[..., :ns], bc4[..., 2 * ns:], wide[:, 5:, 4:]),)
    for x, dt, z, B, C, dy in cases:
        got = []
        for keep in (lambda v: v, lambda v: v.contiguous()):
            # leaves are the views themselves, so that the call meets their strides
            data = [None if v is None else keep(v).detach().requires_grad_(True) for v in (x, dt, z, B, C)]
            lx, ldt, lz, lB, lC = data
            p = [v.clone().requires_grad_(True) for v in (A, D, bias)]
            y, last = sed_amd.gated_scan(lx, ldt, p[0], lB, lC, D=p[1], z=lz, dt_bias=p[2], softplus=True, frames=frames, reverse=reverse, return_state=True)
            leaves = [v for v in data if v is not None] + p
            got.append([y, last, *torch.autograd.grad(y, leaves, keep(dy))])
        for k, (a, b) in enumerate(zip(*got)):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
@pytest.mark.parametrize("d,start", ((256, 0), (256, 1), (40, 0), (33, 3)))
@pytest.mark.parametrize("W", (3, 4, 8))
def test_conv_gradients_of_views(W, d, start, dtype):
    import sed_amd
    t = {"fp32": torch.float32, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device=_dev()).manual_seed(W + d)
    r = lambda *s: torch.randn(s, generator=g, device=_dev())  # noqa: E731
    nb, n = 3, 130
    joint, gaps = r(nb, n, 2 * d + 4 * start).to(t), r(nb, n + 3, d + 4).to(t)
    w, b = r(d, W), r(d)
    frames = torch.tensor([n, n // 3, 1], dtype=torch.int32, device=_dev())
    for x, dy in ((joint[..., start:start + d], gaps[:, 3:, start:start + d]), (r(n, nb, d).to(t).transpose(0, 1), r(n, nb, d).to(t).transpose(0, 1)),
                  (joint[..., d:2 * d], joint[..., :d]), (r(nb, d, n).to(t).transpose(1, 2), r(nb, d, n).to(t).transpose(1, 2))):
        for reverse in (False, True):
            got = []
            for keep in (lambda v: v, lambda v: v.contiguous()):
                leaves = [v.detach().requires_grad_(True) for v in (keep(x), w.clone(), b.clone())]
                y, last = sed_amd.causal_conv(*leaves, activation="silu", frames=frames, reverse=reverse, return_state=True)
                got.append([y, last, *torch.autograd.grad(y, leaves, keep(dy))])
            assert all(torch.equal(p, q) for p, q in zip(*got))


def test_norm_gradients_of_views():
    import sed_amd
    g = torch.Generator(device=_dev()).manual_seed(8)
    r = lambda *s: torch.randn(s, generator=g, device=_dev())  # noqa: E731
    for x, dy in ((r(3, 16, 40, 2).permute(0, 2, 3, 1), r(3, 16, 40, 2).permute(0, 2, 3, 1)), (r(3, 40, 2, 40)[..., 1:17], r(40, 3, 2, 16).transpose(0, 1)),
                  (r(3, 40, 2, 32)[..., ::2], r(1, 1, 1, 16).expand(3, 40, 2, 16))):
        got = []
        for keep in (lambda v: v, lambda v: v.contiguous()):
            leaves = [v.detach().requires_grad_(True) for v in (keep(x), torch.ones(16, device=_dev()), torch.zeros(16, device=_dev()))]
            y = sed_amd.group_norm_act(leaves[0], 4, leaves[1], leaves[2], activation="silu")
            got.append([y, *torch.autograd.grad(y, leaves, keep(dy))])
        assert all(torch.equal(a, b) for a, b in zip(*got))


def _norm_relu(shape, groups, dtype, seed, frames=None):
    """relu, whose slope jumps where u = 0.  Values of x whose u lies within four errors of the corner move by a tenth of the spread,
    before anything is run, until none is left (moving one moves its group's statistics, hence a few rounds)."""
    import sed_amd
    rng = np.random.default_rng(seed)
    c = shape[-1]
    four = (shape[0], shape[1], int(np.prod(shape[2:-1])), c)
    w, rw = _rounded(1 + 0.3 * rng.standard_normal(c), torch.float32)
    b, rb = _rounded(0.3 * rng.standard_normal(c), torch.float32)
    dy, rdy = _rounded(rng.standard_normal(shape), dtype)
    v = rng.standard_normal(shape)
    near = 1e-3  # more than four times the error of u at these sizes, as the assertion below checks
    for _ in range(20):
        x, rx = _rounded(v, dtype)
        q = rx.reshape(four)
        u = np.full(four, np.inf)
        for k in range(shape[0]):
            own = shape[1] if frames is None else frames[k]
            if own:
                z = q[k, :own].reshape(own * four[2], groups, -1)
                hat = (z - z.mean((0, 2), keepdims=True)) / np.sqrt(z.var((0, 2), keepdims=True) + 1e-5)
                u[k, :own] = hat.reshape(own, four[2], c) * rw + rb
        bad = np.abs(u) < near
        if not bad.any():
            break
        v = v + 0.1 * bad.reshape(shape)
    o, clear = S.group_norm(rx.reshape(four), groups, rw, rb, 1e-5, "relu", frames, rdy.reshape(four))
    assert clear > 1
    fr = None if frames is None else torch.tensor(frames, dtype=torch.int32, device=_dev())
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = sed_amd.group_norm_act(x, groups, w, b, activation="relu", frames=fr)
    _close(y, o["y"][0].reshape(shape), o["y"][1].reshape(shape), "y")
    for k, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
        s = shape if k == "dx" else (c,)
        _close(got, o[k][0].reshape(s), o[k][1].reshape(s), k)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("shape,groups,frames", (((3, 9000, 32), 4, (9000, 5, 4501)), ((2, 900, 3, 30), 6, (1, 900)), ((1, 901, 33), 3, None), ((2, 433, 3, 64), 8, None),
                                                 ((2, 33, 96), 2, (33, 7)), ((3, 7, 24), 1, (7, 0, 2)), ((1, 4, 4096), 1, None), ((600, 3, 16), 2, None), ((1, 2000, 64), 1, None)))
def test_norm_relu(shape, groups, frames, dtype):
    """Every kernel with relu: walks with whole vectors and single channels, groups held whole with 4 and 8 channels a lane."""
    _norm_relu(shape, groups, dtype, sum(shape), frames)


def test_conv_of_many_clips_without_a_state():
    """Clips x rows of state x channels past 2^32 where no state is given or asked for: nothing of that size is launched."""
    import sed_amd
    nb, d, W, pick = 150000, 4096, 8, [0, 77777, 149999]
    assert nb * (W - 1) * d >= 1 << 32
    g = torch.Generator(device=_dev()).manual_seed(2)
    x = torch.zeros(nb, 1, d, dtype=torch.float16, device=_dev())
    x[pick] = torch.randn(3, 1, d, generator=g, device=_dev()).half()
    w, b = torch.randn(d, W, generator=g, device=_dev()), torch.randn(d, generator=g, device=_dev())
    y = sed_amd.causal_conv(x, w, b, activation="silu")
    assert torch.equal(y[pick], sed_amd.causal_conv(x[pick], w, b, activation="silu"))
    del y
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dy = torch.zeros(nb, 1, d, dtype=torch.float16, device=_dev())
    dy[pick] = torch.randn(3, 1, d, generator=g, device=_dev()).half()
    dx, dw, db = torch.autograd.grad(sed_amd.causal_conv(*leaves, activation="silu"), leaves, dy)
    alone = []
    for i in pick:
        few = [x.detach()[i:i + 1].requires_grad_(True), w, b]
        alone.append(torch.autograd.grad(sed_amd.causal_conv(*few, activation="silu"), few, dy[i:i + 1]))
    assert torch.equal(dx[pick], torch.cat([t[0] for t in alone]))
    for k, got in ((1, dw), (2, db)):  # zeros add nothing; three clips' terms in some order, here and there
        terms = torch.stack([t[k].double() for t in alone])
        assert ((got.double() - terms.sum(0)).abs() <= 2 * U * terms.abs().sum(0)).all()


def test_norm_of_many_groups_held_whole():
    """Clips x groups past 2^24, each held by one workgroup: the walks' joining launch is not needed, so its grid sets no limit."""
    import sed_amd
    nb, groups, cg, pick = 65535, 258, 8, [0, 40001, 65534]
    c = groups * cg
    assert nb * groups > 1 << 24
    rng = np.random.default_rng(6)
    x, rx = _rounded(rng.standard_normal((3, 1, c)), torch.float32)
    dy, rdy = _rounded(rng.standard_normal((3, 1, c)), torch.float32)
    w, rw = _rounded(1 + 0.3 * rng.standard_normal(c), torch.float32)
    b, rb = _rounded(0.3 * rng.standard_normal(c), torch.float32)
    bx, bdy = (torch.zeros(nb, 1, c, device=_dev()) for _ in range(2))
    bx[pick], bdy[pick] = x, dy
    leaves = [t.requires_grad_(True) for t in (bx, w, b)]
    y = sed_amd.group_norm_act(bx, groups, w, b, activation="silu")
    o, _ = S.group_norm(rx.reshape(3, 1, 1, c), groups, rw, rb, 1e-5, "silu", None, rdy.reshape(3, 1, 1, c))
    _close(y[pick], o["y"][0].reshape(3, 1, c), o["y"][1].reshape(3, 1, c), "y")
    grads = torch.autograd.grad(y, leaves, bdy)  # clips without a gradient add nothing to w and b
    _close(grads[0][pick], o["dx"][0].reshape(3, 1, c), o["dx"][1].reshape(3, 1, c), "dx")
    for k, got in zip(("dw", "db"), grads[1:]):
        _close(got, o[k][0], o[k][1], k)


def test_scan_gradient_of_more_rows_than_a_grid_has_threads():
    """dB and dC of clips x frames x states past 2^32 values together: all clips but three are zeros."""
    import sed_amd
    nb, n, ns, pick = (1 << 18) + 8, 256, 32, [3, 1 << 17, (1 << 18) + 7]
    assert nb * n * 2 * ns >= 1 << 32
    small, ref, rng = _scan_inputs(3, n, 1, 1, ns, torch.bfloat16, 31, gate=False)
    dy, rdy = _rounded(rng.standard_normal((3, n, 1)), torch.bfloat16)
    big = dict(small)
    for k in ("x", "dt", "B", "C"):
        big[k] = torch.zeros(nb, *small[k].shape[1:], dtype=torch.bfloat16, device=_dev())
        big[k][pick] = small[k]
    bdy = torch.zeros(nb, n, 1, dtype=torch.bfloat16, device=_dev())
    bdy[pick] = dy
    leaves = {k: t.requires_grad_(True) for k, t in big.items()}
    args = dict(leaves)
    y = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, softplus=True)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), bdy)))
    o = S.scan(**ref, use_softplus=True, dy=rdy)
    _close(y[pick], o["y"][0], _scan_bound(o, "y", 3, n, 1), "y")
    for k in ("x", "dt", "B", "C"):
        _close(grads[k][pick], o[NAMES[k]][0], _scan_bound(o, NAMES[k], 3, n, 1), NAMES[k])
    for k in ("A", "D", "dt_bias"):  # zeros add nothing to a sum
        _close(grads[k], o[NAMES[k]][0], _scan_bound(o, NAMES[k], 3, n, 1), NAMES[k])
    rest = grads["B"][(1 << 18) - 100000:(1 << 18)]
    assert (rest == 0).all()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("n,ns,d", ((40, 16, 7), (600, 16, 64), (50, 4, 12), (3000, 8, 5)))
def test_scan_steps_masked_by_the_lowest_value(n, ns, d, dtype):
    """dt of the type's lowest value behind a softplus is no step at all, z of it a closed gate: the state passes, every output is finite."""
    import sed_amd
    dev, ref, rng = _scan_inputs(2, n, d, 1, ns, dtype, n + d, state=True)
    low = torch.finfo(dtype).min
    hit = rng.random((2, n, d)) < 0.3
    for k, where in (("dt", hit), ("z", np.roll(hit, 1, 1))):
        dev[k][torch.from_numpy(where).to(_dev())] = low
        ref[k][where] = low
    dy, rdy = _rounded(rng.standard_normal((2, n, d)), dtype)
    dl, rdl = _rounded(rng.standard_normal((2, d, ns)), torch.float32)
    leaves = {k: t.requires_grad_(True) for k, t in dev.items()}
    args = dict(leaves)
    y, last = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, softplus=True, return_state=True)
    with np.errstate(over="ignore"):
        o = S.scan(**ref, use_softplus=True, dy=rdy, dlast=rdl)
    _close(y, o["y"][0], _scan_bound(o, "y", 2, n, d), "y")
    _close(last, o["last"][0], _scan_bound(o, "last", 2, n, d), "last")
    for (k, t), got in zip(leaves.items(), torch.autograd.grad([y, last], list(leaves.values()), [dy, dl])):
        _close(got, o[NAMES[k]][0], _scan_bound(o, NAMES[k], 2, n, d), NAMES[k])


@pytest.mark.parametrize("reverse", (False, True))
@pytest.mark.parametrize("n,d,ns", ((40, 6, 16), (700, 64, 16), (50, 12, 4), (3000, 5, 8), (90, 9, 1), (200, 20, 32)))
def test_scan_infinities_reach_later_frames_of_their_channel_only(n, d, ns, reverse):
    """A value of x that is no number: other channels and clips, the frames walked before it and the gradient of x, which does not read x,
    keep their bits; dB and dC do in the frames walked before."""
    import sed_amd
    dev, _, rng = _scan_inputs(2, n, d, 1, ns, torch.float32, n, gate=False, state=True)
    dy = torch.from_numpy(rng.standard_normal((2, n, d)).astype(np.float32)).to(_dev())
    t0, c0, got = n // 3, d // 2, []
    for bad in (None, float("nan"), float("inf")):
        leaves = {k: t.clone() for k, t in dev.items()}
        if bad is not None:
            leaves["x"][0, t0, c0] = bad
        for t in leaves.values():
            t.requires_grad_(True)
        args = dict(leaves)
        y = sed_amd.gated_scan(*[args.pop(k) for k in ("x", "dt", "A", "B", "C")], **args, softplus=True, reverse=reverse)
        got.append((y, *torch.autograd.grad(y, [leaves["x"], leaves["B"], leaves["C"]], dy)))
    before = torch.arange(n, device=_dev()) > t0 if reverse else torch.arange(n, device=_dev()) < t0
    rest = torch.arange(d, device=_dev()) != c0
    y, dx, dB, dC = got[0]
    for by, bdx, bdB, bdC in got[1:]:
        assert torch.equal(by[1], y[1]) and torch.equal(by[0][:, rest], y[0][:, rest]) and torch.equal(by[0][before], y[0][before])
        assert not by[0, t0, c0].isfinite()
        assert torch.equal(bdx, dx)
        assert torch.equal(bdB[1], dB[1]) and torch.equal(bdC[1], dC[1]) and torch.equal(bdB[0][before], dB[0][before]) and torch.equal(bdC[0][before], dC[0][before])
