"""Thin torch-tensor wrappers over the C ABI (include/pqn_hotpath.h).

Each wrapper passes raw device pointers + torch's current stream; nothing here
computes on the host and nothing falls back to torch/CPU math.
"""
from __future__ import annotations

from ctypes import byref
from typing import Dict, Optional, Tuple

import torch

from . import _lib


def _req(t: torch.Tensor, dtype, name: str):
    if t.dtype != dtype or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{name}: need contiguous CUDA tensor of {dtype}, got {t.dtype} "
                         f"contig={t.is_contiguous()} cuda={t.is_cuda}")


def eps_greedy(q: torch.Tensor, eps: float, key: int, action: Optional[torch.Tensor] = None,
               qmax: Optional[torch.Tensor] = None):
    """jax.vmap(eps_greedy_exploration)(keys, q, eps) (pqn_minatar.py:115-128,196) + max_a q."""
    lib = _lib.load()
    m, a = q.shape
    _req(q, torch.float32, "q")
    if action is None:
        action = torch.empty(m, dtype=torch.int32, device=q.device)
    if qmax is None:
        qmax = torch.empty(m, dtype=torch.float32, device=q.device)
    _lib.check(lib.pqn_eps_greedy(_lib.ptr(q), m, a, float(eps), key, _lib.ptr(action), _lib.ptr(qmax),
                                  _lib.stream_ptr()), "pqn_eps_greedy")
    return action, qmax


def q_lambda(reward: torch.Tensor, done: torch.Tensor, qmax: torch.Tensor, last_q: torch.Tensor, gamma: float,
             lam: float, quirk: bool = True, target: Optional[torch.Tensor] = None):
    """Q(lambda) targets, time-major [T, M] (pqn_minatar.py:237-260)."""
    lib = _lib.load()
    t_len, m = reward.shape
    _req(reward, torch.float32, "reward")
    _req(qmax, torch.float32, "qmax")
    _req(last_q, torch.float32, "last_q")
    if done.dtype == torch.bool:
        done = done.view(torch.uint8)
    _req(done, torch.uint8, "done")
    if target is None:
        target = torch.empty_like(reward)
    _lib.check(lib.pqn_q_lambda(_lib.ptr(reward), _lib.ptr(done), _lib.ptr(qmax), _lib.ptr(last_q), float(gamma),
                                float(lam), t_len, m, 1 if quirk else 0, _lib.ptr(target), _lib.stream_ptr()),
               "pqn_q_lambda")
    return target


def shuffle_permutation(key: int, n: int, device) -> torch.Tensor:
    """jax.random.permutation(key, n) stand-in (pqn_minatar.py:299-315): argsort of
    unique threefry sort keys.  torch.sort is plumbing (rocPRIM radix sort)."""
    lib = _lib.load()
    keys = torch.empty(n, dtype=torch.int64, device=device)
    _lib.check(lib.pqn_shuffle_keys(key, n, _lib.ptr(keys), _lib.stream_ptr()), "pqn_shuffle_keys")
    return torch.sort(keys).indices


class FlatRAdam:
    """optax.chain(clip_by_global_norm(max_norm), radam(lr)) on one flat f32 buffer
    (pqn_minatar.py:140-147,159-162).  The step counter lives on the device."""

    def __init__(self, params: torch.Tensor, lr: float, max_grad_norm: float, lr_decay_steps: float = 0.0,
                 lr_end: float = 1e-20):
        _req(params, torch.float32, "params")
        self.p = params
        self.m = torch.zeros_like(params)
        self.v = torch.zeros_like(params)
        self.count = torch.zeros(1, dtype=torch.int32, device=params.device)
        self.scratch = torch.zeros(1024, dtype=torch.float32, device=params.device)
        self.gnorm = torch.zeros(1, dtype=torch.float32, device=params.device)
        self.lr, self.lr_end, self.lr_steps = float(lr), float(lr_end), float(lr_decay_steps)
        self.max_norm = float(max_grad_norm)

    def step(self, grad: torch.Tensor):
        lib = _lib.load()
        _req(grad, torch.float32, "grad")
        _lib.check(lib.pqn_radam_clip_step(_lib.ptr(self.p), _lib.ptr(grad), _lib.ptr(self.m), _lib.ptr(self.v),
                                           self.p.numel(), _lib.ptr(self.count), self.lr, self.lr_end, self.lr_steps,
                                           self.max_norm, _lib.ptr(self.scratch), _lib.ptr(self.gnorm),
                                           _lib.stream_ptr()), "pqn_radam_clip_step")


# ---- operators of sequence-memory networks: linear attention with a decay per head, the norms around a residual block, log
# probabilities of taken actions.  Functional like the rest of this module: explicit gradients, nothing is recorded by autograd.
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _last_contiguous(t: torch.Tensor, name: str, shape, dtype, index: int):
    """A tensor of this shape and type on GPU `index` whose last index is contiguous; other strides are the caller's."""
    if t.shape != shape or t.dtype != dtype or t.get_device() != index:
        raise ValueError(f"{name}: need {tuple(shape)} of {dtype} on cuda:{index}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    if not t.is_contiguous() and t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the last index must be contiguous, strides are {tuple(t.stride())}")


def _exactly(t: torch.Tensor, name: str, shape, dtype, index: int):
    """A contiguous tensor of this shape and type on GPU `index`."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: need contiguous {tuple(shape)} of {dtype} on cuda:{index}, got {tuple(t.shape)} of {t.dtype} on {t.device} "
                         f"contig={t.is_contiguous()}")


def _on_gpu(t: torch.Tensor, name: str, dtypes):
    if not t.is_cuda or t.dtype not in dtypes:
        raise ValueError(f"{name}: need a CUDA tensor of {' / '.join(str(d) for d in dtypes)}, got {t.dtype} on {t.device}")


def _int32(value: int, name: str) -> int:
    """A size for a 32-bit field of an argument block, which would drop its upper bits silently."""
    if value > 0x7FFFFFFF:
        raise ValueError(f"{name}: up to 2^31 - 1, got {value}")
    return value


def _flags(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.uint8) if t.dtype == torch.bool else t


def _enqueue(fn, args, index: int, what: str):
    """fn(args, stream) on the tensors' own GPU and torch's current stream there."""
    if index == torch.cuda.current_device():
        rc = fn(byref(args), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(byref(args), torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, what)


_ATTN_DTYPES = (torch.float32, torch.bfloat16)


def _attn_args(a, q, k, v, decay, state, reset, scale, step: bool):
    """Checks the common arguments and fills them into `a`; returns (lead shape, state shape)."""
    _on_gpu(q, "q", _ATTN_DTYPES)
    shape, dt, dev = q.shape, q.dtype, q.get_device()
    if len(shape) != (3 if step else 4) or v.dim() != len(shape):
        raise ValueError(f"q, v: need {'[M, H, D]' if step else '[T, M, H, D]'}, got {tuple(q.shape)}, {tuple(v.shape)}")
    m, h, dk = shape[-3:]
    lead, dv = shape[:-1], v.shape[-1]
    if not (0 < dk <= _lib.ATTN_MAX_D and 0 < dv <= _lib.ATTN_MAX_D):
        raise ValueError(f"q, v: head widths of 1 .. {_lib.ATTN_MAX_D}, got {dk} and {dv}")
    if (shape[0] | m | h) >> 31:
        for name, size in zip(("steps", "rows", "heads")[-len(shape) + 1:], shape):
            _int32(size, name)
    _last_contiguous(q, "q", shape, dt, dev)
    _last_contiguous(k, "k", shape, dt, dev)
    _last_contiguous(v, "v", lead + (dv,), dt, dev)
    st = (m, h, dk, dv)
    _exactly(decay, "decay", (h,), torch.float32, dev)
    (a.t_len, a.m, a.heads, a.dk, a.dv, a.dtype, a.scale, a.q, a.k, a.v, a.decay) = (
        1 if step else shape[0], m, h, dk, dv, _DTYPES[dt], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr())
    if step:                         # no time stride
        a.q_stride, a.k_stride, a.v_stride = (0,) + q.stride()[:2], (0,) + k.stride()[:2], (0,) + v.stride()[:2]
    else:
        a.q_stride, a.k_stride, a.v_stride = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    if state is not None:
        _exactly(state, "state", st, torch.float32, dev)
        a.state_in = state.data_ptr()
    if reset is not None:
        if reset.dtype == torch.bool:
            reset = reset.view(torch.uint8)
        _exactly(reset, "reset", lead[:-1], torch.uint8, dev)
        a.reset = reset.data_ptr()
    return lead, st


def _attn_workspace(a, grad: int, device):
    n = _lib.load().pqn_decay_attn_workspace_bytes(byref(a), grad)
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    a.workspace = _lib.ptr(ws)
    return ws


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: Optional[torch.Tensor] = None,
                    reset: Optional[torch.Tensor] = None, scale: float = 1.0, want_state: bool = True):
    """Linear attention with a decay per head over a time-major window, cut at episode ends:

        S_t = decay (1 - reset_t) S_{t-1} + k_t v_t^T,   out_t = scale S_t^T q_t

    q, k [T, M, H, Dk], v [T, M, H, Dv] (f32 or bf16, Dk and Dv up to 128, any strides with a contiguous last index), decay f32 [H]
    in [0, 1], state f32 [M, H, Dk, Dv] (None: zeros), reset u8 / bool [T, M] (the flag comes BEFORE its step: done of the step
    before; what it drops may be NaN).  Returns (out [T, M, H, Dv], the state behind the last step or None).  A NaN or infinity in
    q, k, v reaches the steps behind it in its episode and no others.  Autograd records nothing: the gradient is decay_attention_grad."""
    lib = _lib.load()
    a = _lib.DecayAttnArgs()
    lead, st = _attn_args(a, q, k, v, decay, state, reset, scale, False)
    out = torch.empty_like(v, memory_format=torch.contiguous_format)
    new = torch.empty(st, dtype=torch.float32, device=q.device) if want_state else None
    a.out, a.state_out = out.data_ptr(), _lib.ptr(new)
    ws = _attn_workspace(a, 0, q.device)  # noqa: F841 (held until the launch is enqueued)
    _enqueue(lib.pqn_decay_attn, a, q.get_device(), "pqn_decay_attn")
    return out, new


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
                         reset: Optional[torch.Tensor] = None, scale: float = 1.0) -> torch.Tensor:
    """One step of decay_attention for acting: q, k [M, H, Dk], v [M, H, Dv], reset [M]; `state` is advanced in place, with
    the same bits whatever other rows there are.  Returns out [M, H, Dv]; autograd records nothing."""
    lib = _lib.load()
    if state is None:
        raise ValueError("state: a step advances a state, pass zeros for a new one")
    a = _lib.DecayAttnArgs()
    lead, _ = _attn_args(a, q, k, v, decay, state, reset, scale, True)
    out = torch.empty_like(v, memory_format=torch.contiguous_format)
    a.out, a.state_out = out.data_ptr(), a.state_in
    _enqueue(lib.pqn_decay_attn, a, q.get_device(), "pqn_decay_attn")
    return out


def decay_attention_grad(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, dout: torch.Tensor,
                         dstate_out: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                         reset: Optional[torch.Tensor] = None, scale: float = 1.0):
    """Gradients of decay_attention from those of its outputs (dout like out; dstate_out like the returned state, None: zeros).
    Returns (dq, dk, dv, dstate), contiguous, in the inputs' types; dstate is None without a state.  Every head and row has its own
    gradient, also where q, k or v were expanded over them (the caller sums).  decay is a constant: it has no gradient."""
    lib = _lib.load()
    a = _lib.DecayAttnArgs()
    lead, st = _attn_args(a, q, k, v, decay, state, reset, scale, False)
    _last_contiguous(dout, "dout", lead + (a.dv,), q.dtype, q.get_device())
    if dstate_out is not None:
        _exactly(dstate_out, "dstate_out", st, torch.float32, q.get_device())
    a.dout, a.dout_stride, a.dstate_out = dout.data_ptr(), dout.stride()[:-1], _lib.ptr(dstate_out)
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    dstate = torch.empty(st, dtype=torch.float32, device=q.device) if state is not None else None
    a.dq, a.dk_out, a.dv_out, a.dstate_in = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(dstate)
    ws = _attn_workspace(a, 1, q.device)  # noqa: F841
    _enqueue(lib.pqn_decay_attn_grad, a, q.get_device(), "pqn_decay_attn_grad")
    return dq, dk, dv, dstate


_NORMS = {"layer_norm": 0, "rms_norm": 1}
_GATES = {"none": 0, "sigmoid": 1, "silu": 2}
_NORM_PARAMS = ("res_scale", "post_scale", "post_bias", "pre_scale", "pre_bias")


def _rows(t: torch.Tensor, name: str, shape, dtype, index: int) -> Tuple[torch.Tensor, int]:
    """t as rows of its last index: (tensor that holds them, stride between rows)."""
    _last_contiguous(t, name, shape, dtype, index)
    if t.dim() == 2:
        return t, t.stride(0)
    t = t.reshape(-1, shape[-1])    # a view wherever the rows are evenly spaced, else a copy
    return t, t.stride(0)


def _norm_args(x, f, gate, gate_act, params, norm_type, post, pre, eps):
    _on_gpu(x, "x", _DTYPES)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x: need [..., D] with D >= 1, got {tuple(x.shape)}")
    if norm_type not in _NORMS or gate_act not in _GATES:
        raise ValueError(f"norm_type: one of {sorted(_NORMS)}, gate_act: one of {sorted(_GATES)}; got {norm_type!r}, {gate_act!r}")
    if (gate is None) != (gate_act == "none"):
        raise ValueError("gate and gate_act go together: a gate tensor with 'sigmoid' or 'silu', neither with 'none'")
    shape, d, dt, dev = x.shape, x.shape[-1], x.dtype, x.get_device()
    if d >> 31:
        _int32(d, "D")
    a = _lib.ResidualNormArgs()
    x, a.x_stride = _rows(x, "x", shape, dt, dev)
    f, a.f_stride = _rows(f, "f", shape, dt, dev)
    if gate is not None:
        gate, a.gate_stride = _rows(gate, "gate", shape, dt, dev)
        a.gate = gate.data_ptr()
    for name, p in params.items():
        if p is not None:
            _exactly(p, name, (d,), torch.float32, dev)
            setattr(a, name, p.data_ptr())
    a.n, a.d, a.dtype, a.norm, a.gate_act = x.shape[0], d, _DTYPES[dt], _NORMS[norm_type], _GATES[gate_act]
    a.post, a.pre, a.eps = post, pre, eps
    a.x, a.f = x.data_ptr(), f.data_ptr()
    return a, shape, (x, f, gate)


def residual_norm(x: torch.Tensor, f: torch.Tensor, gate: Optional[torch.Tensor] = None, gate_act: str = "none",
                  res_scale: Optional[torch.Tensor] = None, post_scale: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, pre_scale: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, norm_type: str = "layer_norm", post: bool = True, pre: bool = True,
                  eps: float = 1e-6):
    """The norms around a residual block, with the block's gate and residual scale, in one pass:

        y = x + res_scale * act(gate) * (Norm(f) * post_scale + post_bias),   h = Norm(y) * pre_scale + pre_bias

    x the residual stream, f the block's output, gate (act "sigmoid" or "silu") [..., D] in f32, bf16 or f16, D up to 8192; parameters
    f32 [D], None = 1 (scales) or 0 (biases).  norm_type "layer_norm" or "rms_norm"; post=False leaves f as it is, pre=False returns
    no h.  Returns (y, h or None).  Autograd records nothing: the gradient is residual_norm_grad."""
    params = dict(zip(_NORM_PARAMS, (res_scale, post_scale, post_bias, pre_scale, pre_bias)))
    a, shape, keep = _norm_args(x, f, gate, gate_act, params, norm_type, post, pre, eps)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = torch.empty_like(x, memory_format=torch.contiguous_format) if pre else None
    a.y, a.h = y.data_ptr(), _lib.ptr(h)
    _enqueue(_lib.load().pqn_residual_norm, a, x.get_device(), "pqn_residual_norm")
    return y, h


def residual_norm_grad(x: torch.Tensor, f: torch.Tensor, dy: Optional[torch.Tensor], dh: Optional[torch.Tensor],
                       gate: Optional[torch.Tensor] = None, gate_act: str = "none", res_scale: Optional[torch.Tensor] = None,
                       post_scale: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                       pre_scale: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
                       norm_type: str = "layer_norm", post: bool = True, pre: bool = True,
                       eps: float = 1e-6) -> Dict[str, Optional[torch.Tensor]]:
    """Gradients of residual_norm from those of y and h (one may be None: zeros), the other arguments as they were.  Returns a dict
    of x, f, gate (in their type) and of the parameters that were given (f32); None for what was not given."""
    params = dict(zip(_NORM_PARAMS, (res_scale, post_scale, post_bias, pre_scale, pre_bias)))
    a, shape, keep = _norm_args(x, f, gate, gate_act, params, norm_type, post, pre, eps)
    if dy is None and dh is None:
        raise ValueError("dy, dh: at least one of the two gradients is needed")
    if dh is not None and not pre:
        raise ValueError("dh: pre=False has no h")
    held = []
    for name, g in (("dy", dy), ("dh", dh)):
        if g is not None:
            g, stride = _rows(g, name, shape, x.dtype, x.get_device())
            held.append(g)
            setattr(a, name, g.data_ptr())
            setattr(a, name + "_stride", stride)
    got = {"x": torch.empty(shape, dtype=x.dtype, device=x.device), "f": torch.empty(shape, dtype=x.dtype, device=x.device),
           "gate": torch.empty(shape, dtype=x.dtype, device=x.device) if gate is not None else None}
    a.dx, a.df, a.dgate = got["x"].data_ptr(), got["f"].data_ptr(), _lib.ptr(got["gate"])
    for name, p in params.items():
        got[name] = torch.empty_like(p) if p is not None else None
        setattr(a, "d" + name, _lib.ptr(got[name]))
    lib = _lib.load()
    n = lib.pqn_residual_norm_workspace_floats(a.n, a.d)
    ws = torch.empty(n, dtype=torch.float32, device=x.device) if n else None
    a.workspace = _lib.ptr(ws)
    _enqueue(lib.pqn_residual_norm_grad, a, x.get_device(), "pqn_residual_norm_grad")
    return got


def _logprob_args(logits, actions, mask, temperature, top):
    _on_gpu(logits, "logits", _DTYPES)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits: need [N, A] with A >= 1, got {tuple(logits.shape)}")
    n, width = logits.shape
    if (n | width) >> 31:
        _int32(n, "N"), _int32(width, "A")
    dev = logits.get_device()
    _last_contiguous(logits, "logits", (n, width), logits.dtype, dev)
    _exactly(actions, "actions", (n,), torch.int32, dev)
    if not 0 <= top <= min(width, _lib.LOGPROB_MAX_TOP):
        raise ValueError(f"top: need 0 .. {min(width, _lib.LOGPROB_MAX_TOP)} for {width} actions, got {top}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature: must be positive and finite, got {temperature}")
    a = _lib.ActionLogprobsArgs()
    a.n, a.a, a.top, a.dtype, a.temperature = n, width, top, _DTYPES[logits.dtype], temperature
    a.logits, a.logits_stride, a.action = logits.data_ptr(), logits.stride(0), actions.data_ptr()
    if mask is not None:
        mask = _flags(mask)
        _last_contiguous(mask, "mask", (n, width), torch.uint8, dev)
        a.mask, a.mask_stride = mask.data_ptr(), mask.stride(0)
    return a


def action_logprobs(logits: torch.Tensor, actions: torch.Tensor, mask: Optional[torch.Tensor] = None, temperature: float = 1.0,
                    top: int = 0):
    """Log probabilities of the taken actions under softmax(logits / temperature) over the allowed ones -- a Boltzmann policy over q,
    or a policy head -- with the entropy, the logsumexp and the `top` best alternatives.

    logits [N, A] in f32, bf16 or f16 (rows may be strided), actions int32 [N] (outside 0 .. A-1: no action, logp 0), mask u8 / bool
    [N, A] (0 = not allowed, never looked at).  Returns (logp [N], entropy [N], lse [N], top_logp [N, top], top_action i32 [N, top]),
    f32; alternatives in falling order, ties to the lowest index, -inf / -1 where fewer are allowed.  A row that allows nothing has
    lse -inf and entropy 0; one whose logits / temperature overflow has an infinite lse, which has no gradient.
    Autograd records nothing: the gradient is action_logprobs_grad."""
    a = _logprob_args(logits, actions, mask, temperature, top)
    n, dev, f32 = a.n, logits.device, torch.float32
    logp, entropy, lse = torch.empty(3, n, dtype=f32, device=dev).unbind(0)
    top_logp = torch.empty(n, top, dtype=f32, device=dev)
    top_action = torch.empty(n, top, dtype=torch.int32, device=dev)
    a.logp, a.entropy, a.lse, a.top_logp, a.top_action = (t.data_ptr() for t in (logp, entropy, lse, top_logp, top_action))
    lib = _lib.load()
    size = lib.pqn_action_logprobs_workspace_bytes(n, a.a)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    a.workspace = _lib.ptr(ws)
    _enqueue(lib.pqn_action_logprobs, a, dev.index, "pqn_action_logprobs")
    return logp, entropy, lse, top_logp, top_action


def action_logprobs_grad(logits: torch.Tensor, actions: torch.Tensor, lse: torch.Tensor, entropy: torch.Tensor,
                         dlogp: Optional[torch.Tensor] = None, dentropy: Optional[torch.Tensor] = None,
                         dlse: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                         temperature: float = 1.0) -> torch.Tensor:
    """Gradient of action_logprobs with respect to the logits from those of logp, entropy and lse (f32 [N], None: zeros, not all);
    lse and entropy as action_logprobs returned them.  0 where not allowed, and in a row whose lse is infinite and is given a gradient."""
    a = _logprob_args(logits, actions, mask, temperature, 0)
    n, dev = a.n, logits.get_device()
    if dlogp is None and dentropy is None and dlse is None:
        raise ValueError("dlogp, dentropy, dlse: at least one of the gradients is needed")
    for name, t in (("lse", lse), ("entropy", entropy), ("dlogp", dlogp), ("dentropy", dentropy), ("dlse", dlse)):
        if t is not None:
            _exactly(t, name, (n,), torch.float32, dev)
            setattr(a, name, t.data_ptr())
    dlogits = torch.empty(n, a.a, dtype=logits.dtype, device=logits.device)
    a.dlogits = dlogits.data_ptr()
    _enqueue(_lib.load().pqn_action_logprobs_grad, a, dev, "pqn_action_logprobs_grad")
    return dlogits
