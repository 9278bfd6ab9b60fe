"""The bounds that hold the residual-block norms' kernels (tests/norm_bounds.py), on the CPU: plain f32 arithmetic stays within them, the
gradients are autograd's, and no gradient can be lost without leaving them."""
import pytest
import torch

from tests import memory_ops_reference as ref
from tests import norm_bounds as nb


def _f32(x, kind, act, post=True, pre=True):
    """The same in plain f32 torch, by autograd: rows of f32 whatever the inputs' type."""
    leaves = {k: x[k].float().detach().clone().requires_grad_() for k in ("x", "f", "gate") + nb.PARAMS if x[k] is not None}
    y, h = ref.residual_norm(leaves["x"], leaves["f"], leaves.get("gate"), act, {k: leaves.get(k) for k in nb.PARAMS}, kind, post, pre, 1e-6)
    grads = torch.autograd.grad([y, h], list(leaves.values()), [x["dy"].float(), x["dh"].float()])
    return {"y": y, "h": h, **{"d" + k: g for k, g in zip(leaves, grads)}}


@pytest.mark.parametrize("n,d,act,params,strided", nb.SHAPES)
@pytest.mark.parametrize("kind", ["layer_norm", "rms_norm"])
def test_f32_is_within_and_a_lost_gradient_is_not(n, d, act, params, strided, kind):
    x = nb.inputs("cpu", n, d, torch.float32, n + d, act, params, strided)
    want = nb.block(x["x"], x["f"], x["gate"], act, {p: x[p] for p in nb.PARAMS}, kind, True, True, 1e-6, x["dy"], x["dh"])
    got = _f32(x, kind, act)
    assert set(want) == set(got)
    assert nb.outside(got, want, nb.U) is None
    for half in (nb.U, 2.0 ** -8):
        for name in want:
            # two columns' layer norm is their two signs: it has no gradient to lose (eps apart)
            if name in ("y", "h") or (name == "df" and d == 2 and kind == "layer_norm"):
                continue
            lost = dict(got, **{name: torch.zeros_like(got[name])})
            assert (nb.outside(lost, want, half) or [None])[0] == name, name
            if 2 < n < 1000 and n * d <= 1 << 19 and got[name].dim() == 1:        # and a column sum without one of the rows
                terms = nb.block(*(t[1:] if t is not None else None for t in (x["x"], x["f"], x["gate"])), act, {p: x[p] for p in nb.PARAMS}, kind, True,
                                 True, 1e-6, x["dy"][1:], x["dh"][1:])
                assert (nb.outside(dict(got, **{name: terms[name][0]}), want, half) or [None])[0] == name, name


@pytest.mark.parametrize("kind", ["layer_norm", "rms_norm"])
def test_values_are_autograds(kind):
    x = nb.inputs("cpu", 13, 40, torch.float64, 3, "silu", True, False)
    x.update({k: x[k].double() for k in nb.PARAMS})
    want = nb.block(x["x"], x["f"], x["gate"], "silu", {p: x[p] for p in nb.PARAMS}, kind, True, True, 1e-6, x["dy"], x["dh"])
    leaves = {k: x[k].detach().clone().requires_grad_() for k in ("x", "f", "gate") + nb.PARAMS}
    y, h = ref.residual_norm(leaves["x"], leaves["f"], leaves["gate"], "silu", leaves, kind, True, True, 1e-6)
    grads = torch.autograd.grad([y, h], list(leaves.values()), [x["dy"], x["dh"]])
    for name, g in [("y", y), ("h", h)] + [("d" + k, g) for k, g in zip(leaves, grads)]:
        assert float((want[name][0] - g.detach()).abs().max()) <= 1e-10, name
