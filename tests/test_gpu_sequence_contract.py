"""GPU tests of what the sequence operators promise beside their values on ordinary data: derivatives that would be wrong are refused,
limits and strides are those the documentation names, extreme parameters and recordings keep their digits."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_sequence import _dev, _scan_inputs

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
