"""GPU tests (-m gpu) of the sequence-memory operators where less than f32 would show, at the ends of their ranges, and of every form of
a kernel where one form can go wrong alone.  Tolerances count half steps: u = 2^-24 (f32), h = 2^-8 (bf16), 2^-11 (f16)."""
import pytest
import torch

from tests import memory_ops_reference as ref
from tests.test_memory_ops_gpu import BF16, HALF, U, _abs, _attn_inputs, _close, _d

pytestmark = pytest.mark.gpu


# ---- attention -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t,m,h,dk,dv", [(1, 3, 2, 64, 64), (1, 600, 4, 128, 128), (20, 3, 2, 32, 32), (32, 40, 3, 128, 128), (20, 5, 2, 96, 64), (75, 3, 2, 64, 128),
                                         (130, 2, 3, 128, 96), (75, 3, 2, 33, 50), (900, 1, 2, 64, 128), (700, 1, 2, 128, 33)])
def test_bf16_outputs_are_rounded_once(gpu, t, m, h, dk, dv):
    """Sums and states are f32 and an output is rounded to bf16 once: with the f32 bound e = (2 T + Dk + Dv + 16) u abs on the sum, the
    stored value is off by e + h (|sum| + e).  Nothing is relative to h abs."""
    from purejaxql_amd import ops
    x = _attn_inputs(gpu, t, m, h, dk, dv, BF16, t + dk, True, 0.01)
    q, k, v, decay, state, reset, scale = x["q"], x["k"], x["v"], x["decay"], x["state"], x["reset"], dk ** -0.5
    n, half = (2 * t + dk + dv + 16) * U, HALF[BF16]
    out, new = ops.decay_attention(q, k, v, decay, state=state, reset=reset, scale=scale)
    r_out, r_new = ref.attention(_d(q), _d(k), _d(v), _d(decay), _d(state), reset, scale)
    a_out, a_new = ref.attention(_abs(q), _abs(k), _abs(v), _d(decay), _abs(state), reset, scale)
    _close(out, r_out, n * a_out + half * (r_out.abs() + n * a_out), "out")
    _close(new, r_new, n * a_new + 1e-30, "state")
    got = ops.decay_attention_grad(q, k, v, decay, x["dout"], dstate_out=x["dstate"], state=state, reset=reset, scale=scale)
    want = ref.attention_grad(_d(q), _d(k), _d(v), _d(decay), _d(x["dout"]), _d(x["dstate"]), _d(state), reset, scale)
    most = ref.attention_grad(_abs(q), _abs(k), _abs(v), _d(decay), _abs(x["dout"]), _abs(x["dstate"]), _abs(state), reset, scale)
    for name, g, w, a in zip(("dq", "dk", "dv"), got, want, most):
        _close(g, w, n * a + half * (w.abs() + n * a), name)
    _close(got[3], want[3], n * most[3] + 1e-30, "dstate")


@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128), (96, 72), (67, 128)])
def test_a_row_steps_alike_alone_and_among_many(gpu, dk, dv):
    """An env acts the same whatever runs beside it: a row's step has the same bits in a batch of 5 rows and in one of 700."""
    from purejaxql_amd import ops
    for dtype in (BF16, torch.float32):
        x = _attn_inputs(gpu, 1, 700, 4, dk, dv, dtype, dk + dv, True, 0.3)
        few, many = x["state"][:5].clone(), x["state"].clone()
        args = [x[n][0] for n in ("q", "k", "v")]
        a = ops.decay_attention_step(*(z[:5] for z in args), x["decay"], few, reset=x["reset"][0, :5], scale=0.3)
        b = ops.decay_attention_step(*args, x["decay"], many, reset=x["reset"][0], scale=0.3)
        assert torch.equal(a, b[:5]) and torch.equal(few, many[:5]), dtype
