"""GPU tests (-m gpu) of the residual-block norms against 64 bits within bounds that follow every value (tests/norm_bounds.py, whose CPU tests
show that a gradient that is lost leaves them)."""
import itertools

import pytest
import torch

from tests import norm_bounds as nb
from tests.test_memory_ops_gpu import BF16, F16, F32, HALF

pytestmark = pytest.mark.gpu


def _check(x, kind, act, post=True, pre=True, use_dy=True, use_dh=True):
    from purejaxql_amd import ops
    params = {p: x[p] for p in nb.PARAMS}
    if not post:
        params["post_scale"] = params["post_bias"] = None
    if not pre:
        params["pre_scale"] = params["pre_bias"] = None
    dy, dh = (x["dy"] if use_dy else None), (x["dh"] if use_dh and pre else None)
    kw = dict(gate=x["gate"], gate_act=act, norm_type=kind, post=post, pre=pre, **params)
    y, h = ops.residual_norm(x["x"], x["f"], **kw)
    got = {"y": y, "h": h}
    want = nb.block(x["x"], x["f"], x["gate"], act, params, kind, post, pre, 1e-6, dy, dh)
    if dy is not None or dh is not None:
        got.update({"d" + k: g for k, g in ops.residual_norm_grad(x["x"], x["f"], dy, dh, **kw).items()})
    assert {k for k, g in got.items() if g is not None} == set(want)
    assert nb.outside(got, want, HALF[x["x"].dtype]) is None


@pytest.mark.parametrize("n,d,act,params,strided", nb.SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["layer_norm", "rms_norm"])
def test_norms_within_their_bounds(gpu, n, d, act, params, strided, dtype, kind):
    _check(nb.inputs(gpu, n, d, dtype, n + d, act, params, strided), kind, act)


@pytest.mark.parametrize("kind,post,pre,use_dy,use_dh", [c for c in itertools.product(["layer_norm", "rms_norm"], *[[True, False]] * 4)
                                                         if c[3] or (c[4] and c[2])])
@pytest.mark.parametrize("n,d", [(37, 96), (300, 1500), (260, 4500)])
def test_options_within_their_bounds(gpu, kind, post, pre, use_dy, use_dh, n, d):
    _check(nb.inputs(gpu, n, d, BF16 if n == 300 else F32, n, "silu", True, n == 37), kind, "silu", post, pre, use_dy, use_dh)
