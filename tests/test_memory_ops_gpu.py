"""GPU tests (-m gpu) of the sequence-memory operators against their definitions in float64 (tests/memory_ops_reference.py).

Tolerances, derived before the first run, with u = 2^-24 (f32's half step) and h = half a step of the tensor's type (bf16 2^-8, f16
2^-11).  "abs" is the reference's sum of the absolute values of the same terms.
  attention, f32: every term passes at most 2 roundings per step it is carried (decay, addition; in the chunked form fewer) and one per
    product and addition over the head width: (2 T + Dk + Dv + 16) u abs.
  attention, bf16: the weights between two steps of a chunk, or the state, are an operand of a matrix product in bf16: h abs, and what
    is added to a state is split in bf16 pieces, at least two: h^2 abs; the output is rounded once: h |ref|.  States are f32: no last term.
  norms: the terms of a row's sums are of one row: (D + 32) u of the largest intermediate; see rn_tol.
  log probabilities: x = logit / temperature has |x| u, the exponent of e^(x - m) as much again, the sum A u at most; see lp_tol.
"""
import itertools
import math

import numpy as np
import pytest
import torch

from tests import memory_ops_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _close(got, want, tol, what):
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    over = (got - want).abs() - tol
    assert got.numel() == 0 or float(over.max()) <= 0.0, (what, float(over.max()), int((over > 0).sum()), got.numel(), float((got - want).abs().max()))


# ---- attention -----------------------------------------------------------------------------------------------------------------
def _attn_inputs(gpu, t, m, h, dk, dv, dtype, seed, state=True, resets=0.1, spread=False):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)

    def normal(*shape, dt=dtype, s=1.0):
        return (torch.randn(*shape, generator=gen, device=gpu) * s).to(dt)

    def wide(d, s=1.0):
        if not spread:
            return normal(t, m, h, d, s=s)
        return normal(t, h, m, 3 * d + 5, s=s)[..., d:2 * d].transpose(1, 2)     # a slice of a wider projection, rows and heads swapped

    x = {"q": wide(dk), "k": wide(dk, dk ** -0.5), "v": wide(dv), "dout": wide(dv)}
    x["decay"] = 1.0 - torch.exp2(-torch.linspace(1.0, 9.0, h, device=gpu)) if h > 1 else torch.full((1,), 0.96875, device=gpu)
    x["state"] = normal(m, h, dk, dv, dt=F32, s=0.5) if state else None
    x["dstate"] = normal(m, h, dk, dv, dt=F32, s=0.5) if state else None
    x["reset"] = (torch.rand(t, m, generator=gen, device=gpu) < resets).to(torch.uint8) if resets else None
    return x


def _d(x):
    return None if x is None else x.double()


def _abs(x):
    return None if x is None else x.double().abs()


def _attn_check(x, scale, grad=True):
    from purejaxql_amd import ops
    q, k, v, decay, state, reset = (x[n] for n in ("q", "k", "v", "decay", "state", "reset"))
    dt, t, dk, dv = q.dtype, q.shape[0], q.shape[-1], v.shape[-1]
    out, new = ops.decay_attention(q, k, v, decay, state=state, reset=reset, scale=scale)
    r_out, r_new = ref.attention(_d(q), _d(k), _d(v), _d(decay), _d(state), reset, scale)
    a_out, a_new = ref.attention(_abs(q), _abs(k), _abs(v), _d(decay), _abs(state), reset, scale)
    n, h = (2 * t + dk + dv + 16) * U, (HALF[dt] if dt != F32 else 0.0)
    _close(out, r_out, (n + h + h * h) * a_out + h * r_out.abs(), "out")
    _close(new, r_new, (n + h * h) * a_new + 1e-30, "state")
    if not grad:
        return
    got = ops.decay_attention_grad(q, k, v, decay, x["dout"], dstate_out=x["dstate"], state=state, reset=reset, scale=scale)
    want = ref.attention_grad(_d(q), _d(k), _d(v), _d(decay), _d(x["dout"]), _d(x["dstate"]), _d(state), reset, scale)
    most = ref.attention_grad(_abs(q), _abs(k), _abs(v), _d(decay), _abs(x["dout"]), _abs(x["dstate"]), _abs(state), reset, scale)
    for name, g, w, a in zip(("dq", "dk", "dv"), got, want, most):
        assert g.dtype == dt and g.is_contiguous()
        _close(g, w, (n + h + h * h) * a + h * w.abs(), name)
    if state is None:
        assert got[3] is None
    else:
        _close(got[3], want[3], (n + h * h) * most[3] + 1e-30, "dstate")


ATTN_SHAPES = [(1, 1, 1, 1, 1), (1, 5, 3, 32, 32), (2, 3, 2, 16, 48), (7, 2, 3, 33, 17), (31, 3, 1, 64, 64), (32, 9, 4, 32, 32),
               (64, 2, 2, 128, 128), (65, 2, 3, 48, 80), (129, 3, 2, 128, 40), (200, 1, 2, 96, 128), (513, 2, 1, 7, 100)]


@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decay_attention_and_gradient(gpu, shape, dtype):
    _attn_check(_attn_inputs(gpu, *shape, dtype, seed=sum(shape)), scale=shape[3] ** -0.5)


@pytest.mark.parametrize("dk,dv", [(96, 96), (80, 16), (24, 88), (72, 64), (96, 128), (128, 72), (88, 40)])
@pytest.mark.parametrize("t,m,h", [(20, 3, 2), (33, 40, 3), (300, 2, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decay_attention_widths_between_powers_of_two(gpu, t, m, h, dk, dv, dtype):
    _attn_check(_attn_inputs(gpu, t, m, h, dk, dv, dtype, dk + dv, True, 0.02), scale=dk ** -0.5)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("state,resets,spread", [(False, 0.0, False), (True, 0.0, True), (False, 0.5, True), (True, 1.0, False)])
def test_decay_attention_states_resets_strides(gpu, dtype, state, resets, spread):
    _attn_check(_attn_inputs(gpu, 75, 3, 3, 40, 64, dtype, 5, state, resets, spread), scale=0.7)


@pytest.mark.parametrize("t,m,h,dk,dv,dtype", [(3000, 1, 1, 64, 64, BF16), (2049, 2, 1, 32, 128, F32), (4100, 1, 2, 128, 64, BF16),
                                               (1500, 1, 3, 128, 128, F32)])
def test_long_windows_of_few_rows(gpu, t, m, h, dk, dv, dtype):
    """What a launch of few rows does (the time axis may be cut): with resets far apart, near, and none."""
    for resets in (0.0, 0.0007, 0.03):
        _attn_check(_attn_inputs(gpu, t, m, h, dk, dv, dtype, t, True, resets), scale=dk ** -0.5)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decays_at_their_limits(gpu, dtype):
    """decay 0 (only the step itself), 1 (a plain sum), the smallest step below 1."""
    x = _attn_inputs(gpu, 100, 2, 3, 32, 32, dtype, 3, True, 0.02)
    x["decay"] = torch.tensor([0.0, 1.0, 1.0 - 2.0 ** -24], device=gpu)
    _attn_check(x, 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_non_finite_steps_stay_in_their_episode(gpu, dtype, bad):
    """A reset drops a NaN state; a NaN or infinity in k or v reaches the steps behind it in its episode and no others, and in q its own."""
    from purejaxql_amd import ops
    t, m = 150, 2
    x = _attn_inputs(gpu, t, m, 2, 32, 48, dtype, 9, True, 0.0)
    reset = torch.zeros(t, m, dtype=torch.uint8, device=gpu)
    reset[0, 0] = 1
    reset[70, 0] = 1
    x["state"][0] = math.nan
    x["k"][40, 0, 0, 3] = bad
    x["v"][41, 0, 1, 5] = bad
    x["q"][100, 0, 1, 2] = bad
    out, new = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"], state=x["state"], reset=reset)
    fine = torch.isfinite(out).all(-1)
    want = torch.ones(t, m, 2, dtype=torch.bool, device=gpu)
    want[40:70, 0, 0] = False
    want[41:70, 0, 1] = False
    want[100, 0, 1] = False
    assert torch.equal(fine, want) and bool(torch.isfinite(new).all())
    clean = {n: x[n].clone() for n in ("q", "k", "v")}
    for n in clean:
        clean[n][~torch.isfinite(clean[n])] = 0
    state = x["state"].clone()
    state[0] = 0
    out2, new2 = ops.decay_attention(clean["q"], clean["k"], clean["v"], x["decay"], state=state, reset=reset)
    r_out, _ = ref.attention(*(clean[n].double() for n in ("q", "k", "v")), x["decay"].double(), state.double(), reset)
    a_out, _ = ref.attention(*(clean[n].double().abs() for n in ("q", "k", "v")), x["decay"].double(), state.double().abs(), reset)
    h = HALF[dtype] if dtype != F32 else 0.0
    tol = ((2 * t + 96) * U + h + h * h) * a_out + h * r_out.abs()
    keep = want[..., None].expand_as(out)
    _close(out[keep], r_out[keep], tol[keep], "the rest")
    # the gradient of the later episode does not see the earlier one's steps either
    dq, dk, dv, ds = ops.decay_attention_grad(x["q"], x["k"], x["v"], x["decay"], x["dout"], dstate_out=x["dstate"], state=x["state"], reset=reset)
    assert bool(torch.isfinite(dv[101:, 0]).all()) and bool(torch.isfinite(dk[101:, 0]).all()) and bool(torch.isfinite(dq[70:, 0]).all())
    assert bool((ds[0] == 0).all())
    for g in (dq, dk, dv):
        assert bool(torch.isfinite(g[:, 1]).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,h,dk,dv", [(1, 1, 128, 128), (130, 4, 32, 32), (33, 3, 20, 50)])
def test_steps_in_place_are_the_window(gpu, dtype, m, h, dk, dv):
    """Acting step by step on one state buffer gives the window's outputs and final state."""
    from purejaxql_amd import ops
    t = 9
    x = _attn_inputs(gpu, t, m, h, dk, dv, dtype, 21, True, 0.2)
    state = x["state"].clone()
    outs = [ops.decay_attention_step(x["q"][i], x["k"][i], x["v"][i], x["decay"], state, reset=x["reset"][i].bool(), scale=0.3) for i in range(t)]
    args = [x[n].double() for n in ("q", "k", "v", "decay", "state")]
    r_out, r_new = ref.attention(*args, x["reset"], 0.3)
    a_out, a_new = ref.attention(*[a.abs() for a in args], x["reset"], 0.3)
    h_ = HALF[dtype] if dtype != F32 else 0.0
    n = (2 * t + dk + dv + 16) * U
    _close(torch.stack(outs), r_out, (n + h_ + h_ * h_) * a_out + h_ * r_out.abs(), "out")
    _close(state, r_new, (n + h_ * h_) * a_new + 1e-30, "state")


@pytest.mark.parametrize("dk,dv,m,h", [(128, 128, 525, 4), (96, 72, 300, 7), (8, 128, 1100, 2), (67, 128, 130, 16)])
def test_steps_in_place_of_many_wide_rows(gpu, dk, dv, m, h):
    """Steps of so many wide bf16 rows that they go by another kernel than those of few: still the window's outputs and state."""
    from purejaxql_amd import ops
    t = 3
    x = _attn_inputs(gpu, t, m, h, dk, dv, BF16, 22, True, 0.3)
    state = x["state"].clone()
    outs = [ops.decay_attention_step(x["q"][i], x["k"][i], x["v"][i], x["decay"], state, reset=x["reset"][i], scale=0.3) for i in range(t)]
    args = [x[n].double() for n in ("q", "k", "v", "decay", "state")]
    r_out, r_new = ref.attention(*args, x["reset"], 0.3)
    a_out, a_new = ref.attention(*[a.abs() for a in args], x["reset"], 0.3)
    n, h_ = (2 * t + dk + dv + 16) * U, HALF[BF16]
    _close(torch.stack(outs), r_out, (n + h_ + h_ * h_) * a_out + h_ * r_out.abs(), "out")
    _close(state, r_new, (n + h_ * h_) * a_new + 1e-30, "state")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,d", [(20, 32), (75, 64), (40, 128)])
def test_products_that_overflow_behind_a_step_or_episode(gpu, dtype, t, d):
    """k of a step times q of an earlier one, or of another episode, is no term of any sum, though it is larger than a float."""
    x = _attn_inputs(gpu, t, 2, 2, d, d, dtype, 6, True, 0.0)
    x["q"][2, 0] *= 2.0 ** 100
    x["k"][5, 0] *= 2.0 ** 100
    x["reset"] = torch.zeros(t, 2, dtype=torch.uint8, device=gpu)
    x["reset"][8, 1] = 1
    x["k"][7, 1] *= 2.0 ** 100
    x["q"][9, 1] *= 2.0 ** 100
    x["dstate"] = None
    _attn_check(x, scale=1.0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,m,h,dk,dv", [(700, 1, 2, 33, 50), (333, 3, 1, 64, 64), (260, 2, 3, 128, 96)])
def test_long_windows_off_sixteen_bytes(gpu, dtype, t, m, h, dk, dv):
    """Slices that start off 16 bytes, few rows and a long window: element by element, the time axis cut."""
    x = _attn_inputs(gpu, t, m, h, dk, dv, dtype, 31, True, 0.004, spread=True)
    for n in ("q", "k", "v", "dout"):
        wide = torch.zeros(t, m, h, x[n].shape[-1] + 1, dtype=dtype, device=gpu)
        wide[..., 1:] = x[n]
        x[n] = wide[..., 1:]
    _attn_check(x, scale=dk ** -0.5)


def test_calls_on_two_streams_at_once(gpu):
    """Two calls in flight together, of the same sizes with workspaces of their own, give what each gives alone."""
    from purejaxql_amd import ops
    xs = [_attn_inputs(gpu, 900, 1, 3, 64, 64, BF16, s, True, 0.002) for s in (1, 2)]
    ls = [_logit_inputs(gpu, 2, 70000, BF16, s, True) for s in (3, 4)]
    ns = [_norm_inputs(gpu, 700, 4500, F32, s, "silu", True) for s in (5, 6)]

    def run(x, l, n):
        o = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"], state=x["state"], reset=x["reset"])
        g = ops.decay_attention_grad(x["q"], x["k"], x["v"], x["decay"], x["dout"], state=x["state"], reset=x["reset"])
        p = ops.action_logprobs(l["logits"], l["actions"], mask=l["mask"], top=5)
        r = ops.residual_norm_grad(n["x"], n["f"], n["dy"], n["dh"], gate=n["gate"], gate_act="silu", **{k: n[k] for k in NORM_PARAMS})
        return [*o, *g, *p, *r.values()]

    want = [run(*a) for a in zip(xs, ls, ns)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, a in zip(streams, zip(xs, ls, ns)):
            with torch.cuda.stream(st):
                got.append(run(*a))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_attention_lengths_of_zero(gpu):
    from purejaxql_amd import ops
    x = _attn_inputs(gpu, 0, 3, 2, 16, 8, F32, 1, True, 0.0)
    out, new = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"], state=x["state"])
    assert out.shape == (0, 3, 2, 8) and torch.equal(new, x["state"])
    _, new = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"])
    assert bool((new == 0).all())
    dq, dk, dv, ds = ops.decay_attention_grad(x["q"], x["k"], x["v"], x["decay"], x["dout"], dstate_out=x["dstate"], state=x["state"])
    assert torch.equal(ds, x["dstate"]) and dq.shape == (0, 3, 2, 16) and dv.shape == (0, 3, 2, 8)
    y = _attn_inputs(gpu, 4, 0, 2, 16, 8, F32, 1, True, 0.0)
    out, new = ops.decay_attention(y["q"], y["k"], y["v"], y["decay"], state=y["state"])
    assert out.shape == (4, 0, 2, 8) and new.shape == (0, 2, 16, 8)


def test_expanded_heads_and_rows_have_a_gradient_each(gpu):
    """k and v shared by the heads (stride 0): every head gets its own gradient, the caller's sum is the shared tensor's."""
    from purejaxql_amd import ops
    t, m, h, d = 40, 2, 3, 32
    x = _attn_inputs(gpu, t, m, h, d, d, F32, 4, True, 0.05)
    k1, v1 = x["k"][:, :, :1].contiguous(), x["v"][:, :, :1].contiguous()
    k, v = k1.expand(t, m, h, d), v1.expand(t, m, h, d)
    got = ops.decay_attention_grad(x["q"], k, v, x["decay"], x["dout"], state=x["state"], reset=x["reset"])
    leaves = [x["q"].double().requires_grad_(), k1.double().requires_grad_(), v1.double().requires_grad_()]
    o, _ = ref.attention(leaves[0], leaves[1].expand(t, m, h, d), leaves[2].expand(t, m, h, d), x["decay"].double(), x["state"].double(), x["reset"])
    want = torch.autograd.grad(o, leaves, x["dout"].double())
    most = ref.attention_grad(*(z.double().abs() for z in (x["q"], k, v)), x["decay"].double(), x["dout"].double().abs(), None,
                              x["state"].double().abs(), x["reset"])
    n = (2 * t + 2 * d + 16 + h) * U
    _close(got[0], want[0], n * most[0], "dq")
    _close(got[1].sum(2, keepdim=True), want[1], n * most[1].sum(2, keepdim=True), "dk")
    _close(got[2].sum(2, keepdim=True), want[2], n * most[2].sum(2, keepdim=True), "dv")


def test_attention_gradient_against_differences(gpu):
    """Directional derivatives of the definition in 64 bits (central differences, error O(step^2)) against the kernel's gradient."""
    from purejaxql_amd import ops
    x = _attn_inputs(gpu, 90, 2, 2, 24, 40, F32, 17, True, 0.03)
    got = ops.decay_attention_grad(x["q"], x["k"], x["v"], x["decay"], x["dout"], dstate_out=x["dstate"], state=x["state"], reset=x["reset"], scale=0.5)
    base = {n: x[n].double() for n in ("q", "k", "v", "state")}

    def loss(z):
        o, s = ref.attention(z["q"], z["k"], z["v"], x["decay"].double(), z["state"], x["reset"], 0.5)
        return float((o * x["dout"].double()).sum() + (s * x["dstate"].double()).sum())

    gen = torch.Generator(device=gpu)
    gen.manual_seed(1)
    for name, g in zip(("q", "k", "v", "state"), got):
        d = torch.randn(base[name].shape, generator=gen, device=gpu, dtype=torch.float64)
        step = 1e-4     # the loss is linear in each input alone: the difference is exact up to 64-bit rounding
        up, down = dict(base), dict(base)
        up[name], down[name] = base[name] + step * d, base[name] - step * d
        diff = (loss(up) - loss(down)) / (2 * step)
        size = float((g.double().abs() * d.abs()).sum())
        assert abs(diff - float((g.double() * d).sum())) <= 1e-5 * size, (name, diff, float((g.double() * d).sum()), size)


def test_offsets_past_32_bits(gpu):
    """Rows of a cache that lie more than 2^32 elements apart: strides are 64-bit."""
    from purejaxql_amd import ops
    far = 1 << 31
    if torch.cuda.mem_get_info()[0] < 40 * (1 << 30):
        pytest.skip("needs 40 GB")
    big = torch.zeros(2 * far + 4096, dtype=BF16, device=gpu)
    t, m, h, d = 5, 3, 1, 16
    x = _attn_inputs(gpu, t, m, h, d, d, BF16, 2, False, 0.0)
    views = {}
    for i, n in enumerate(("q", "k", "v")):
        views[n] = big[i * 512:].as_strided((t, m, h, d), (32, far, d, 1))
        views[n].copy_(x[n])
    out, new = ops.decay_attention(views["q"], views["k"], views["v"], x["decay"])
    want, wnew = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"])
    assert torch.equal(out, want) and torch.equal(new, wnew)


# ---- norms ---------------------------------------------------------------------------------------------------------------------
def _norm_inputs(gpu, n, d, dtype, seed, gate_act, params, strided=False):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)

    def normal(*shape, dt=dtype, s=1.0):
        return (torch.randn(*shape, generator=gen, device=gpu) * s).to(dt)

    def rows(s=1.0):
        return normal(n, 2 * d + 3, s=s)[:, d:2 * d] if strided else normal(n, d, s=s)

    x = {"x": rows(2.0), "f": rows(0.7), "gate": rows() if gate_act != "none" else None, "dy": rows(), "dh": rows()}
    for name in ("res_scale", "post_scale", "post_bias", "pre_scale", "pre_bias"):
        x[name] = normal(d, dt=F32, s=0.3) + (0.0 if name.endswith("bias") else 0.8) if params else None
    return x


NORM_PARAMS = ("res_scale", "post_scale", "post_bias", "pre_scale", "pre_bias")


def _norm_check(x, kind, gate_act, post=True, pre=True, eps=1e-6, use_dy=True, use_dh=True):
    """rn_tol: a normalised value carries the rounding of its row's two sums ((D + 4) u relative, taken pairwise by 64 lanes far less)
    and a handful of operations on itself; it is amplified by |row| / sqrt(var + eps) where the mean is subtracted.  The rows here
    have means near 0 (amplification below 4), so (D + 32) u (|value| + 4 max|row|) holds with room; gradients chain three such steps."""
    from purejaxql_amd import ops
    n, d = x["x"].shape
    dt = x["x"].dtype
    params = {p: x[p] for p in NORM_PARAMS}
    if not post:
        params["post_scale"] = params["post_bias"] = None
    if not pre:
        params["pre_scale"] = params["pre_bias"] = None
    kw = dict(gate=x["gate"], gate_act=gate_act, norm_type=kind, post=post, pre=pre, eps=eps, **params)
    y, h = ops.residual_norm(x["x"], x["f"], **kw)
    leaves = {k: x[k].double().detach().requires_grad_() for k in ("x", "f", "gate") if x[k] is not None}
    leaves.update({k: v.double().detach().requires_grad_() for k, v in params.items() if v is not None})
    p64 = {k: leaves.get(k) for k in NORM_PARAMS}
    ry, rh = ref.residual_norm(leaves["x"], leaves["f"], leaves.get("gate"), gate_act, p64, kind, post, pre, eps)
    half = HALF[dt] if dt != F32 else U

    def tol(w, chain):
        rowmax = w.abs().amax(-1, keepdim=True) if w.dim() == 2 and w.numel() else w.abs().amax() if w.numel() else w
        return half * w.abs() + chain * (d + 32) * U * (w.abs() + 4 * rowmax) + 1e-30

    _close(y, ry.detach(), tol(ry.detach(), 2), "y")
    if pre:
        _close(h, rh.detach(), tol(rh.detach(), 4), "h")
    else:
        assert h is None
    dy, dh = (x["dy"] if use_dy else None), (x["dh"] if use_dh and pre else None)
    if dy is None and dh is None:
        return
    got = ops.residual_norm_grad(x["x"], x["f"], dy, dh, **kw)
    outs, gs = [], []
    if dy is not None:
        outs.append(ry)
        gs.append(dy.double())
    if dh is not None:
        outs.append(rh)
        gs.append(dh.double())
    want = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs, allow_unused=True)))
    # The gradient of a norm is (dz - z mean(dz z) - mean(dz)) / sqrt(var + eps), z the normalised row with sum z^2 <= D: each of the
    # three terms is at most sqrt(D) max|dz| (Cauchy-Schwarz) and carries (D + 32) u of itself, whatever is left of their sum -- for
    # one or two columns almost nothing is, the gradient there being of the order of eps.  So its error is bounded by
    # lost(dz) = 3 (D + 32) u sqrt(D) max|dz| / sqrt(var + eps), which is passed on by factors of at most |scale act| or |scale n slope|.
    def lost(dz, row):
        c = row if kind == "rms_norm" else row - row.mean(-1, keepdim=True)
        return 3 * (d + 32) * U * math.sqrt(d) * dz.abs().amax(-1, keepdim=True) / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)

    one = torch.ones(d, dtype=torch.float64, device=x["x"].device)
    scale = {k: (leaves[k].detach() if k in leaves else one) for k in ("res_scale", "post_scale", "pre_scale")}
    extra = {"x": lost(dh.double() * scale["pre_scale"], ry.detach()) if dh is not None else 0.0 * ry.detach()}
    g64 = leaves["gate"].detach() if gate_act != "none" else None
    act = one.expand(n, d) if g64 is None else torch.sigmoid(g64) * (1.0 if gate_act == "sigmoid" else g64)
    factor = (scale["res_scale"] * act * scale["post_scale"]).abs()
    most = (want["x"].abs() + extra["x"]) * factor
    extra["f"] = (extra["x"] * factor).amax(-1, keepdim=True)
    if post:
        f64 = leaves["f"].detach()
        c = f64 if kind == "rms_norm" else f64 - f64.mean(-1, keepdim=True)
        extra["f"] = lost(most, f64) + 3 * math.sqrt(d) * extra["f"] / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if g64 is not None:       # slopes of sigmoid and silu are at most 1.1
        nn = ref.normed(leaves["f"].detach(), kind, eps) if post else leaves["f"].detach()
        nn = nn * scale["post_scale"] + (leaves["post_bias"].detach() if "post_bias" in leaves else 0.0)
        extra["gate"] = extra["x"] * (scale["res_scale"] * nn).abs() * 1.1
    for name in ("x", "f", "gate"):
        if x[name] is not None:
            assert got[name].dtype == dt and got[name].is_contiguous()
            w = want[name] if want[name] is not None else torch.zeros_like(leaves[name])
            _close(got[name], w, tol(w, 16) + extra[name], "d" + name)
        else:
            assert got[name] is None
    for name in NORM_PARAMS:
        if params[name] is None:
            assert got[name] is None
            continue
        w = want[name] if want[name] is not None else torch.zeros_like(leaves[name])
        # a sum over n rows of terms that are bounded by the products of the factors' largest values
        size = 16 * (d + n + 64) * U * math.sqrt(n) * (float(x["dy"].double().abs().max()) + 8 * float(x["dh"].double().abs().max())) * 16
        _close(got[name], w, torch.full_like(w, size) + 0 * w, "d" + name)


@pytest.mark.parametrize("n,d", [(1, 1), (3, 2), (5, 64), (130, 128), (7, 333), (33, 1024), (6, 1025), (9, 4096), (2, 4095), (3, 8192), (4, 5001)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_residual_norm_sizes(gpu, n, d, dtype):
    kind, act = ("layer_norm", "silu") if (n + d) % 2 else ("rms_norm", "sigmoid")
    if d == 1:
        kind = "rms_norm"     # the layer norm of one column is 0 whatever the column holds
    _norm_check(_norm_inputs(gpu, n, d, dtype, n * d, act, True), kind, act)


@pytest.mark.parametrize("kind,act,params,post,pre,strided", itertools.product(
    ["layer_norm", "rms_norm"], ["none", "silu"], [True, False], [True, False], [True, False], [False, True]))
def test_residual_norm_options(gpu, kind, act, params, post, pre, strided):
    _norm_check(_norm_inputs(gpu, 37, 96, F32, 3, act, params, strided), kind, act, post, pre)


@pytest.mark.parametrize("n,d,dtype,params,strided", [(900, 4100, F32, True, False), (300, 5001, BF16, True, True), (520, 6000, F16, False, False),
                                                      (70, 8191, F32, True, True)])
def test_residual_norm_wide_rows(gpu, n, d, dtype, params, strided):
    """Rows over 4096 columns: the parameter gradients come from a second look at the rows."""
    _norm_check(_norm_inputs(gpu, n, d, dtype, d, "silu", params, strided), "layer_norm", "silu")


@pytest.mark.parametrize("use_dy,use_dh", [(True, False), (False, True)])
def test_residual_norm_one_gradient(gpu, use_dy, use_dh):
    _norm_check(_norm_inputs(gpu, 50, 200, BF16, 8, "sigmoid", True), "layer_norm", "sigmoid", use_dy=use_dy, use_dh=use_dh)


def test_residual_norm_of_constant_rows_and_no_rows(gpu):
    """A row without variance is all zeros behind its norm (eps keeps the root); no rows give no outputs and zero parameter gradients."""
    from purejaxql_amd import ops
    f = torch.full((4, 256), 3.0, device=gpu)
    x = torch.zeros(4, 256, device=gpu)
    y, h = ops.residual_norm(x, f)
    assert bool((y == 0).all()) and bool((h == 0).all())
    e = torch.empty(0, 64, device=gpu)
    s = torch.ones(64, device=gpu)
    y, h = ops.residual_norm(e, e, post_scale=s)
    assert y.shape == (0, 64) and h.shape == (0, 64)
    g = ops.residual_norm_grad(e, e, e, e, post_scale=s)
    assert bool((g["post_scale"] == 0).all()) and g["x"].shape == (0, 64)


def test_residual_norm_many_rows_and_leading_indexes(gpu):
    """More rows than workgroups (parameter gradients walk), a [T, M, D] tensor, the same bits in every run."""
    from purejaxql_amd import ops
    x = _norm_inputs(gpu, 8000, 160, F32, 5, "silu", True)
    _norm_check(x, "layer_norm", "silu")
    kw = dict(gate_act="silu", **{p: x[p] for p in NORM_PARAMS})
    three = {k: x[k].view(40, 200, 160) for k in ("x", "f", "gate", "dy", "dh")}
    a = ops.residual_norm_grad(x["x"], x["f"], x["dy"], x["dh"], gate=x["gate"], **kw)
    for _ in range(3):
        b = ops.residual_norm_grad(three["x"], three["f"], three["dy"], three["dh"], gate=three["gate"], **kw)
        for k in a:
            assert torch.equal(a[k].reshape(-1), b[k].reshape(-1)), k


def test_residual_norm_gradient_against_differences(gpu):
    from purejaxql_amd import ops
    x = _norm_inputs(gpu, 6, 80, F32, 12, "silu", True)
    kw = dict(gate_act="silu", **{p: x[p] for p in NORM_PARAMS})
    got = ops.residual_norm_grad(x["x"], x["f"], x["dy"], x["dh"], gate=x["gate"], **kw)
    base = {k: x[k].double() for k in ("x", "f", "gate") + NORM_PARAMS}

    def loss(z):
        y, h = ref.residual_norm(z["x"], z["f"], z["gate"], "silu", z, "layer_norm", True, True, 1e-6)
        return float((y * x["dy"].double()).sum() + (h * x["dh"].double()).sum())

    gen = torch.Generator(device=gpu)
    gen.manual_seed(3)
    for name in base:
        d = torch.randn(base[name].shape, generator=gen, device=gpu, dtype=torch.float64)
        up, down = dict(base), dict(base)
        up[name], down[name] = base[name] + 1e-5 * d, base[name] - 1e-5 * d
        diff = (loss(up) - loss(down)) / 2e-5      # error of the difference: step^2 times a third derivative of order 1
        size = float((got[name].double().abs() * d.abs()).sum())
        assert abs(diff - float((got[name].double() * d).sum())) <= 2e-5 * size, (name, diff, size)


# ---- log probabilities -----------------------------------------------------------------------------------------------------------
def _logit_inputs(gpu, n, a, dtype, seed, masked, strided=False, scale=2.5):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)
    x = {"logits": (torch.randn(n, a + (5 if strided else 0), generator=gen, device=gpu) * scale).to(dtype)[:, :a]}
    x["actions"] = torch.randint(0, a, (n,), generator=gen, device=gpu, dtype=torch.int32)
    x["mask"] = (torch.rand(n, a, generator=gen, device=gpu) < 0.7).to(torch.uint8) if masked else None
    for k in ("dlogp", "dentropy", "dlse"):
        x[k] = torch.randn(n, generator=gen, device=gpu)
    return x


def _logp_check(x, temperature, top, grad=True):
    """lp_tol: x = logit / temperature is off by |x| u, as is the exponent of e^(x - m): e = 4 (max|x| + 1) u relative on every term
    of a sum; A terms add (64 + A / 64) u at most (a lane's running sum, then six joins).  The entropy weighs it by |log p|."""
    from purejaxql_amd import ops
    logits, actions, mask = x["logits"], x["actions"], x["mask"]
    n, a = logits.shape
    dt = logits.dtype
    got = ops.action_logprobs(logits, actions, mask=mask, temperature=temperature, top=top)
    want = ref.logprobs(logits.cpu(), actions.cpu(), None if mask is None else mask.cpu(), temperature, top)
    big = float(torch.where(torch.isfinite(logits), logits, torch.zeros_like(logits)).double().abs().max()) / temperature if logits.numel() else 0.0
    e = 4 * (big + 1) * U + (64 + a / 64) * U
    names = ("logp", "entropy", "lse", "top_logp")
    for name, g, w in zip(names, got[:4], want[:4]):
        g = g.double().cpu()
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(torch.isinf(g), torch.isinf(w)), name
        ok = torch.isfinite(w)
        assert torch.equal(g[~ok & ~torch.isnan(w)], w[~ok & ~torch.isnan(w)]), name
        wide = 1.0 + math.log(a) + 2 * big if name == "entropy" else 1.0
        _close(g[ok], w[ok], e * wide + 4 * U * w[ok].abs(), name)
    assert torch.equal(got[4].cpu(), want[4]), "top_action"
    if not grad:
        return
    d = ops.action_logprobs_grad(logits, actions, got[2], got[1], x["dlogp"], x["dentropy"], x["dlse"], mask=mask, temperature=temperature)
    z = logits.double() / temperature
    if mask is not None:
        z = z.masked_fill(mask == 0, -math.inf)
    lse, h = want[2].to(z.device)[:, None], want[1].to(z.device)[:, None]
    lp = torch.where(z > -math.inf, z - lse, torch.full_like(z, -math.inf))
    p = torch.exp(lp)
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    hot = (torch.arange(a, device=z.device)[None] == actions[:, None]).double()
    hot = hot * (lp > -math.inf).double()
    has = hot.sum(-1, keepdim=True)
    dlp, dh, dl = (x[k].double()[:, None] for k in ("dlogp", "dentropy", "dlse"))
    w = (dlp * (hot - has * p) - dh * (plogp + p * h) + dl * p) / temperature
    w = torch.where(lp > -math.inf, w, torch.zeros_like(w))
    size = (dlp.abs() * (hot + p) + dh.abs() * (plogp.abs() + p * h.abs()) + dl.abs() * p + dh.abs() * p) / temperature
    half = HALF[dt]
    # f16's subnormal step bounds what a tiny gradient may lose.  A probability below 2^-126, f32's smallest normal number, counts as 0
    # (the kernels take 2^x from the hardware, which has no subnormal results): the gradient loses at most p (|dlogp| + |dlse| +
    # |dentropy| (|log p| + H)) / temperature of it, and p |log p| <= 2^-126 * 126 log 2 below p = 2^-126 (it rises with p up to 1/e).
    floor = 2.0 ** -25 if dt == F16 else 2.0 ** -126 * (dlp.abs() + dl.abs() + dh.abs() * (126 * math.log(2.0) + h.abs().clamp(max=1e6))) / temperature
    _close(d, w, half * w.abs() + (4 * e * (1 + 0) + 16 * U) * size * (1 + math.log(a) + 2 * big) + floor, "dlogits")


@pytest.mark.parametrize("n,a", [(1, 1), (5, 2), (257, 3), (100, 8), (33, 9), (1000, 17), (64, 33), (10, 65), (7, 200), (9, 300), (3, 513), (5, 1024),
                                 (3, 1025), (2, 4097), (1, 9000), (4, 20001), (1300, 1100)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_action_logprobs_sizes(gpu, n, a, dtype):
    n = min(n, 60) if a > 1000 else n     # the reference walks the rows one by one
    _logp_check(_logit_inputs(gpu, n, a, dtype, n + a, (n + a) % 2 == 0, strided=a % 3 == 0), 0.8, min(a, 1 + (n + a) % 16))


def test_action_logprobs_many_rows_of_a_long_axis(gpu):
    """Rows enough that none is cut (a workgroup walks its row), against torch in 64 bits."""
    from purejaxql_amd import ops
    x = _logit_inputs(gpu, 1030, 5000, BF16, 2, False)
    logp, ent, lse, tl, ta = ops.action_logprobs(x["logits"], x["actions"], top=4)
    z = x["logits"].double()
    l64 = torch.logsumexp(z, -1)
    tol = torch.full_like(l64, (4 * (float(z.abs().max()) + 1) + 64 + 5000 / 64) * U)
    _close(lse, l64, tol + 4 * U * l64.abs(), "lse")
    key = z * 1.0 - torch.arange(5000, device=gpu) * 1e-9     # bf16 logits are at least 1e-5 apart unless equal
    assert torch.equal(ta.long(), torch.topk(key, 4).indices)


@pytest.mark.parametrize("a", [17, 300, 5000, 20001])
def test_action_logprobs_rows_at_their_limits(gpu, a):
    """Nothing allowed; one allowed; the type's lowest value; -inf, NaN and +inf in masked and in allowed places; equal logits; actions
    outside the row or not allowed."""
    x = _logit_inputs(gpu, 14, a, F32, 6, True)
    x["mask"][:] = 1
    l, m, act = x["logits"], x["mask"], x["actions"]
    m[0] = 0
    l[0, 3] = math.nan
    m[1] = 0
    m[1, a - 1] = 1
    act[1] = a - 1
    l[2] = torch.finfo(F32).min
    l[3] = -math.inf
    l[3, a // 2] = 1.5
    act[3] = a // 2
    m[4, ::2] = 0
    l[4, ::2] = math.nan
    l[5, ::2] = math.inf
    m[5, ::2] = 0
    l[6] = 0.25
    l[7] = -math.inf
    act[8] = -1
    act[9] = a
    m[10, act[10].item()] = 0
    l[11, ::2] = -math.inf
    l[12, 2] = 80.0
    l[13] = l[13].round()
    _logp_check(x, 1.0, min(a, 16), grad=False)
    keep = [i for i in range(14) if i not in (2,)]
    y = {k: (v[keep].contiguous() if v is not None else None) for k, v in x.items()}
    y["mask"][4 - 1] = m[4]
    _logp_check(y, 1.0, 3)
    bad = _logit_inputs(gpu, 3, a, F32, 7, False)
    bad["logits"][0, 1] = math.nan
    bad["logits"][1, a - 1] = math.inf
    _logp_check(bad, 1.0, 0, grad=False)


def test_action_logprobs_gradient_against_differences(gpu):
    from purejaxql_amd import ops
    x = _logit_inputs(gpu, 6, 40, F32, 3, True)
    x["mask"].scatter_(1, x["actions"].long()[:, None], 1)
    _, ent, lse, _, _ = ops.action_logprobs(x["logits"], x["actions"], mask=x["mask"], temperature=1.3)
    g = ops.action_logprobs_grad(x["logits"], x["actions"], lse, ent, x["dlogp"], x["dentropy"], x["dlse"], mask=x["mask"], temperature=1.3).double()

    def loss(z):
        lp, en, ls, _, _ = ref.logprobs(z.cpu(), x["actions"].cpu(), x["mask"].cpu(), 1.3, 0)
        return float((lp * x["dlogp"].double().cpu()).sum() + (en * x["dentropy"].double().cpu()).sum() + (ls * x["dlse"].double().cpu()).sum())

    gen = torch.Generator(device=gpu)
    gen.manual_seed(4)
    for _ in range(3):
        d = torch.randn(6, 40, generator=gen, device=gpu, dtype=torch.float64)
        z = x["logits"].double()
        diff = (loss(z + 1e-5 * d) - loss(z - 1e-5 * d)) / 2e-5
        assert abs(diff - float((g * d).sum())) <= 2e-5 * float((g.abs() * d.abs()).sum())


@pytest.mark.parametrize("n,a", [(6, 300), (4, 5000), (3, 40001)])
def test_action_logprobs_strided_and_bool_masks(gpu, n, a):
    """A mask of truth values, and one that is a slice of a wider tensor at an odd offset."""
    from purejaxql_amd import ops
    x = _logit_inputs(gpu, n, a, BF16, a, True)
    want = ops.action_logprobs(x["logits"], x["actions"], mask=x["mask"], top=6)
    wide = torch.ones(n, a + 3, dtype=torch.uint8, device=gpu)
    wide[:, 3:] = x["mask"]
    for mask in (x["mask"].bool(), wide[:, 3:]):
        got = ops.action_logprobs(x["logits"], x["actions"], mask=mask, top=6)
        assert all(torch.equal(i, j) for i, j in zip(got, want))
    x["mask"] = wide[:, 3:]
    _logp_check(x, 1.3, 6)


@pytest.mark.parametrize("a", [17, 300, 5000, 70000])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_action_logprobs_beyond_the_largest_float(gpu, a, dtype):
    """logits / temperature overflows: the log probabilities come from differences of logits; lse is infinite and the gradient 0.  A row
    of large logits near each other: no cancellation (differences are exact, the sum of A terms is off by (64 + A / 64) u)."""
    from purejaxql_amd import ops
    big = torch.finfo(dtype).max
    l = torch.empty(3, a, device=gpu)
    l[0], l[1] = -big, big
    l[2] = 2.0 ** 20 + torch.arange(a, device=gpu) % 2 * 2.0 ** 14
    x = l.to(dtype)
    act = torch.tensor([1, 2, 3], dtype=torch.int32, device=gpu)
    logp, ent, lse, top_logp, top = ops.action_logprobs(x, act, temperature=0.25, top=2)
    tol = torch.full((3,), (64 + a / 64 + 64 * math.log(a)) * U, device=gpu)
    want = torch.full((3,), -math.log(a), device=gpu, dtype=torch.float64)
    want[2] = -math.log(a // 2)
    _close(logp, want, tol, "logp")
    _close(ent, -want, tol, "entropy")
    _close(top_logp, want[:, None].expand(3, 2), tol[:, None].expand(3, 2), "top_logp")
    assert top.tolist() == [[0, 1], [0, 1], [1, 3]] and lse[0] == -math.inf and lse[1] == math.inf
    one = torch.ones(3, device=gpu)
    d = ops.action_logprobs_grad(x, act, lse, ent, one, one, one, temperature=0.25)
    assert bool((d[:2] == 0).all()) and bool(torch.isfinite(d).all())


@pytest.mark.parametrize("a", [300, 700, 1500, 3000, 9000, 33001])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_action_logprobs_alternatives_among_equals(gpu, a, dtype):
    """The lowest indexes of 1, 40, 100, 290 and all equal best logits, of fewer allowed than asked for, and of rising and falling rows."""
    gen = torch.Generator(device=gpu)
    gen.manual_seed(a)
    l = torch.randn(9, a, generator=gen, device=gpu) - 8.0
    for i, k in enumerate((1, 40, 100, 290, a)):
        l[i, torch.randperm(a, generator=gen, device=gpu)[:k]] = 4.0
    l[5] = torch.arange(a, device=gpu) / a
    l[6] = -l[5]
    l[7] = -math.inf
    l[7, a // 3:a // 3 + 5] = torch.tensor([-3.0, 0.0, -0.0, -math.inf, 2.0], device=gpu)
    l[8] = torch.finfo(BF16).min
    x = _logit_inputs(gpu, 9, a, dtype, a, False)
    x["logits"] = l.to(dtype)
    from purejaxql_amd import ops
    for top in (1, 8, 16):
        got = ops.action_logprobs(x["logits"], x["actions"], top=top)
        key = x["logits"].double().cpu() + 0.0
        want = torch.sort(key, dim=-1, descending=True, stable=True)
        ids = torch.where(want.values[:, :top] > -math.inf, want.indices[:, :top], torch.full_like(want.indices[:, :top], -1))
        assert torch.equal(got[4].cpu().long(), ids), top


def test_action_logprobs_no_rows(gpu):
    from purejaxql_amd import ops
    e = torch.empty(0, 9, device=gpu)
    act = torch.empty(0, dtype=torch.int32, device=gpu)
    logp, ent, lse, tl, ta = ops.action_logprobs(e, act, top=2)
    assert logp.shape == (0,) and tl.shape == (0, 2) and ta.dtype == torch.int32
    assert ops.action_logprobs_grad(e, act, lse, ent, dlogp=logp).shape == (0, 9)


# ---- together, on streams and in graphs --------------------------------------------------------------------------------------------
def _network(gpu, seed, d=64, h=4, a=6):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)
    w = {n: torch.randn(d, o, generator=gen, device=gpu) * d ** -0.5 for n, o in (("q", d), ("k", d), ("v", d), ("g", d), ("o", d), ("head", a))}
    w.update({n: 1.0 + 0.1 * torch.randn(d, generator=gen, device=gpu) for n in ("res_scale", "post_scale", "pre_scale")})
    w["decay"] = 1.0 - torch.exp2(-torch.linspace(2.0, 5.0, h, device=gpu))
    return w


def _norms(w):
    return {k: w[k] for k in ("res_scale", "post_scale", "pre_scale")}


def _network_forward(w, x, state, reset, actions):
    from purejaxql_amd import ops
    t, m, d = x.shape
    h = w["decay"].numel()
    q, k, v = ((x @ w[n]).view(t, m, h, d // h) for n in "qkv")
    o, new = ops.decay_attention(q, k, v, w["decay"], state=state, reset=reset, scale=(d // h) ** -0.5)
    f, gate = o.reshape(t, m, d) @ w["o"], x @ w["g"]
    y, z = ops.residual_norm(x, f, gate=gate, gate_act="silu", norm_type="rms_norm", **_norms(w))
    logits = (z @ w["head"]).view(t * m, -1)
    logp, ent, lse, top_logp, top = ops.action_logprobs(logits, actions, temperature=0.5, top=2)
    return dict(q=q, k=k, v=v, o=o, new=new, f=f, gate=gate, y=y, z=z, logits=logits, logp=logp, ent=ent, lse=lse, top=top)


def _network_backward(w, x, state, reset, actions, r, dlogp, dent):
    from purejaxql_amd import ops
    t, m, d = x.shape
    g = {}
    dlogits = ops.action_logprobs_grad(r["logits"], actions, r["lse"], r["ent"], dlogp, dent, temperature=0.5).view(t, m, -1)
    g["head"] = r["z"].reshape(t * m, d).t() @ dlogits.view(t * m, -1)
    n = ops.residual_norm_grad(x, r["f"], None, dlogits @ w["head"].t(), gate=r["gate"], gate_act="silu", norm_type="rms_norm", **_norms(w))
    g.update({k: n[k] for k in ("res_scale", "post_scale", "pre_scale")})
    flat = x.reshape(t * m, d)
    dx = n["x"] + n["gate"] @ w["g"].t()
    g["g"] = flat.t() @ n["gate"].view(t * m, d)
    g["o"] = r["o"].reshape(t * m, d).t() @ n["f"].view(t * m, d)
    do = (n["f"] @ w["o"].t()).view_as(r["o"])
    dq, dk, dv, g["state"] = ops.decay_attention_grad(r["q"], r["k"], r["v"], w["decay"], do, state=state, reset=reset, scale=r["q"].shape[-1] ** -0.5)
    for name, dz in (("q", dq), ("k", dk), ("v", dv)):
        g[name] = flat.t() @ dz.view(t * m, d)
        dx = dx + dz.view(t, m, d) @ w[name].t()
    g["x"] = dx
    return g


def _network_inputs(gpu, seed, t=45, m=6, d=64, h=4, a=6):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)
    x = torch.randn(t, m, d, generator=gen, device=gpu)
    state = torch.randn(m, h, d // h, d // h, generator=gen, device=gpu) * 0.3
    reset = (torch.rand(t, m, generator=gen, device=gpu) < 0.05).to(torch.uint8)
    actions = torch.randint(0, a, (t * m,), generator=gen, device=gpu, dtype=torch.int32)
    return x, state, reset, actions, torch.randn(t * m, generator=gen, device=gpu), 0.1 * torch.randn(t * m, generator=gen, device=gpu)


def test_a_memory_network_learns_and_acts(gpu):
    """The operators as a network uses them: a window with its whole gradient against autograd in 64 bits (f32 against 64 bits through
    about ten products of width 64: 1e-4 of the largest gradient), and the same window acted step by step."""
    from purejaxql_amd import ops
    w = _network(gpu, 1)
    x, state, reset, actions, dlogp, dent = _network_inputs(gpu, 2)
    r = _network_forward(w, x, state, reset, actions)
    g = _network_backward(w, x, state, reset, actions, r, dlogp, dent)

    leaves = {n: w[n].double().requires_grad_() for n in w if n != "decay"}
    leaves["x"], leaves["state"] = x.double().requires_grad_(), state.double().requires_grad_()
    t, m, d = x.shape
    h = w["decay"].numel()
    q, k, v = ((leaves["x"] @ leaves[n]).view(t, m, h, d // h) for n in "qkv")
    o, _ = ref.attention(q, k, v, w["decay"].double(), leaves["state"], reset, (d // h) ** -0.5)
    p = {"res_scale": leaves["res_scale"], "post_scale": leaves["post_scale"], "post_bias": None, "pre_scale": leaves["pre_scale"], "pre_bias": None}
    _, z = ref.residual_norm(leaves["x"], o.reshape(t, m, d) @ leaves["o"], leaves["x"] @ leaves["g"], "silu", p, "rms_norm", True, True, 1e-6)
    lp = torch.log_softmax((z @ leaves["head"]).view(t * m, -1) / 0.5, -1)
    loss = (lp.gather(1, actions.long()[:, None])[:, 0] * dlogp.double()).sum() + (-(lp.exp() * lp).sum(-1) * dent.double()).sum()
    want = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    assert set(g) == set(want)
    for n in want:
        _close(g[n], want[n], torch.full_like(want[n], 1e-4 * float(want[n].abs().max())), n)

    s = state.clone()
    for i in range(t):
        q, k, v = ((x[i] @ w[n]).view(m, h, d // h) for n in "qkv")
        o = ops.decay_attention_step(q, k, v, w["decay"], s, reset=reset[i], scale=(d // h) ** -0.5)
        y, z = ops.residual_norm(x[i], o.reshape(m, d) @ w["o"], gate=x[i] @ w["g"], gate_act="silu", norm_type="rms_norm", **_norms(w))
        logp, _, _, _, top = ops.action_logprobs(z @ w["head"], actions[i * m:(i + 1) * m], temperature=0.5, top=2)
        _close(logp, r["logp"][i * m:(i + 1) * m], torch.full((m,), 1e-4), "logp of step %d" % i)
    _close(s, r["new"], torch.full_like(s, 1e-4), "state")


def test_captured_and_replayed_beside_eager_work(gpu):
    """Forward and gradient in one captured graph, replayed on new inputs with eager work and synchronisations between; two graphs of
    different sizes share nothing."""
    w = _network(gpu, 3)
    graphs = []
    for seed, t in ((5, 45), (6, 130)):
        ins = _network_inputs(gpu, seed, t=t)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(2):
                r = _network_forward(w, *ins[:4])
                _network_backward(w, *ins[:4], r, *ins[4:])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            r = _network_forward(w, *ins[:4])
            g = _network_backward(w, *ins[:4], r, *ins[4:])
        graphs.append((graph, ins, r, g, t, st))
    for turn in range(4):
        for graph, ins, r, g, t, st in graphs:
            new = _network_inputs(gpu, 100 + turn, t=t)
            for a, b in zip(ins, new):
                a.copy_(b)
            torch.cuda.synchronize()
            with torch.cuda.stream(st):
                graph.replay()
            torch.cuda.synchronize()
            er = _network_forward(w, *new[:4])
            eg = _network_backward(w, *new[:4], er, *new[4:])
            for n in ("new", "y", "logp", "ent", "top", "o"):
                assert torch.equal(r[n], er[n]), (turn, n)
            for n in ("state", "res_scale", "post_scale", "pre_scale"):
                assert torch.equal(g[n], eg[n]), (turn, n)
            _close(g["x"], eg["x"].double(), torch.full_like(g["x"], 1e-5 * float(eg["x"].abs().max())), "dx")


def test_work_follows_the_current_stream(gpu):
    from purejaxql_amd import ops
    x = _attn_inputs(gpu, 60, 4, 2, 32, 32, F32, 8, True, 0.05)
    want, wnew = ops.decay_attention(x["q"], x["k"], x["v"], x["decay"], state=x["state"], reset=x["reset"])
    side = torch.cuda.Stream()
    y = torch.zeros_like(x["q"])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2000000)
        y.copy_(x["q"])                       # the operator has to run behind this copy
        got, gnew = ops.decay_attention(y, x["k"], x["v"], x["decay"], state=x["state"], reset=x["reset"])
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(gnew, wnew)


def test_numpy_is_not_needed_by_the_operators():
    """The wrappers take torch tensors only (numpy is for the tests)."""
    from purejaxql_amd import ops
    with pytest.raises((ValueError, AttributeError)):
        ops.action_logprobs(np.zeros((2, 3), dtype=np.float32), np.zeros(2, dtype=np.int32))
