"""Refusals of the sequence-memory operators (no GPU needed: every check comes before a launch) and the layout of their argument blocks."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_blocks_match_the_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    from purejaxql_amd import _lib
    blocks = {"pqn_decay_attn_t": _lib.DecayAttnArgs, "pqn_residual_norm_t": _lib.ResidualNormArgs, "pqn_action_logprobs_t": _lib.ActionLogprobsArgs}
    lines = []
    for name, cls in blocks.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f[0]) for f in cls._fields_]
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pqn_hotpath.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    said = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in blocks.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert said == want


def _attn(**kw):
    from purejaxql_amd import _lib
    a = _lib.DecayAttnArgs(t_len=4, m=2, heads=2, dk=16, dv=16, dtype=0, scale=1.0, q=64, k=64, v=64, decay=64, out=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,says", [({"dtype": 2}, "neither f32 nor bf16"), ({"dtype": 7}, "neither"), ({"t_len": -1}, "t_len"), ({"m": -1}, "m must"),
                                     ({"heads": 0}, "heads"), ({"dk": 0}, "head widths"), ({"dk": 129}, "head widths"), ({"dv": 129}, "head widths"),
                                     ({"dv": -3}, "head widths"), ({"q": None}, "NULL q"), ({"v": None}, "NULL q"), ({"decay": None}, "NULL decay"),
                                     ({"out": None}, "NULL out"), ({"m": 1 << 30}, "pairs")])
def test_attention_refusals(kw, says):
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_decay_attn(C.byref(_attn(**kw)), None) == -1
    assert says in lib.pqn_last_error().decode()


@pytest.mark.parametrize("kw", [{"t_len": 1, "m": 1 << 27}, {"t_len": 100, "m": 1 << 25, "dk": 128, "dv": 128}, {"t_len": 100, "m": 1 << 26, "dtype": 1}])
def test_attention_of_more_rows_than_a_launch(kw):
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_decay_attn(C.byref(_attn(**kw)), None) == -1 and "more than one launch" in lib.pqn_last_error().decode()
    kw = dict(kw, dout=64, dq=64, dk_out=64, dv_out=64)
    assert lib.pqn_decay_attn_grad(C.byref(_attn(**kw)), None) == -1 and "more than one launch" in lib.pqn_last_error().decode()


@pytest.mark.parametrize("n,a", [((1 << 31) - 1, 7), (1 << 30, 20), (1 << 28, 60), (1 << 26, 900), (1 << 25, 3000), (1 << 21, 1 << 21)])
def test_log_probabilities_of_more_rows_than_a_launch(n, a):
    from purejaxql_amd import _lib
    lib = _lib.load()
    args = _lib.ActionLogprobsArgs(n=n, a=a, top=0, dtype=1, temperature=1.0, logits=64, logits_stride=a, action=64, logp=64, entropy=64, lse=64,
                                   dlogp=64, dlogits=64, workspace=64)
    assert lib.pqn_action_logprobs(C.byref(args), None) == -1 and "more than one launch" in lib.pqn_last_error().decode()
    if a > 100:
        assert lib.pqn_action_logprobs_grad(C.byref(args), None) == -1 and "more than one launch" in lib.pqn_last_error().decode()


def test_attention_gradient_refusals():
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_decay_attn_grad(C.byref(_attn()), None) == -1 and "NULL dout" in lib.pqn_last_error().decode()
    assert lib.pqn_decay_attn_grad(None, None) == -1 and lib.pqn_decay_attn(None, None) == -1
    # nothing to do is no error, and launches nothing
    assert lib.pqn_decay_attn(C.byref(_attn(m=0)), None) == 0 and lib.pqn_decay_attn_grad(C.byref(_attn(m=0)), None) == 0
    assert lib.pqn_decay_attn(C.byref(_attn(t_len=0)), None) == 0


def _norm(**kw):
    from purejaxql_amd import _lib
    a = _lib.ResidualNormArgs(n=4, d=16, dtype=0, norm=0, gate_act=0, post=1, pre=1, eps=1e-6, x=64, f=64, y=64, h=64, x_stride=16, f_stride=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,says", [({"dtype": 3}, "dtype"), ({"n": -1}, "n must"), ({"d": 0}, "d > 0"), ({"d": 8193}, "up to 8192"), ({"norm": 2}, "norm 2"),
                                     ({"gate_act": 3}, "activation"), ({"eps": -1.0}, "eps"), ({"x": None}, "NULL x"), ({"gate": 64}, "go together"),
                                     ({"gate_act": 1}, "go together"), ({"post": 0, "post_scale": 64}, "without the norm"), ({"h": None}, "h is one"),
                                     ({"pre": 0}, "h is one"), ({"pre": 0, "pre_bias": 64}, "without the norm"), ({"y": None}, "y is an output"),
                                     ({"n": 1 << 31}, "rows")])
def test_norm_refusals(kw, says):
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_residual_norm(C.byref(_norm(**kw)), None) == -1
    assert says in lib.pqn_last_error().decode()


@pytest.mark.parametrize("kw,says", [({}, "are outputs"), ({"dx": 64, "df": 64}, "workspace"), ({"dx": 64, "df": 64, "workspace": 64}, "both NULL"),
                                     ({"dx": 64, "df": 64, "workspace": 64, "pre": 0, "dh": 64}, "without the norm"),
                                     ({"dx": 64, "df": 64, "workspace": 64, "gate": 64, "gate_act": 2}, "are outputs")])
def test_norm_gradient_refusals(kw, says):
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_residual_norm_grad(C.byref(_norm(**kw)), None) == -1
    assert says in lib.pqn_last_error().decode()
    assert lib.pqn_residual_norm(C.byref(_norm(n=0)), None) == 0 and lib.pqn_residual_norm_grad(C.byref(_norm(n=0)), None) == 0


def _logp(**kw):
    from purejaxql_amd import _lib
    a = _lib.ActionLogprobsArgs(n=4, a=8, top=0, dtype=0, temperature=1.0, logits=64, logits_stride=8, action=64, logp=64, entropy=64, lse=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,says", [({"dtype": -1}, "dtype"), ({"n": -1}, "n must"), ({"a": 0}, "a > 0"), ({"top": 9}, "top must"), ({"top": -1}, "top must"),
                                     ({"a": 100, "top": 17}, "top must"), ({"temperature": 0.0}, "temperature"), ({"temperature": -1.0}, "temperature"),
                                     ({"temperature": float("inf")}, "temperature"), ({"temperature": float("nan")}, "temperature"),
                                     ({"temperature": 1e-44}, "temperature"), ({"logits": None}, "NULL logits"), ({"logp": None}, "NULL logp"),
                                     ({"top": 2}, "NULL top_logp"), ({"a": 100000}, "NULL workspace"), ({"a": 100000, "workspace": 68}, "aligned"),
                                     ({"a": (1 << 30) + 1}, "columns")])
def test_logprob_refusals(kw, says):
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_action_logprobs(C.byref(_logp(**kw)), None) == -1
    assert says in lib.pqn_last_error().decode()


def test_logprob_gradient_refusals():
    from purejaxql_amd import _lib
    lib = _lib.load()
    assert lib.pqn_action_logprobs_grad(C.byref(_logp()), None) == -1 and "dlogits" in lib.pqn_last_error().decode()
    assert lib.pqn_action_logprobs_grad(C.byref(_logp(dlogits=64)), None) == -1 and "all NULL" in lib.pqn_last_error().decode()
    assert lib.pqn_action_logprobs_grad(C.byref(_logp(n=0)), None) == 0 and lib.pqn_action_logprobs(C.byref(_logp(n=0)), None) == 0


def test_wrappers_refuse_what_the_kernels_do_not_take():
    """Host tensors (there is no CPU form), and on the way to a launch wrong shapes, types and options."""
    from purejaxql_amd import ops
    q = torch.zeros(4, 2, 2, 16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.decay_attention(q, q, q, torch.ones(2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.residual_norm(q, q)
    with pytest.raises(ValueError, match="CUDA"):
        ops.action_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="a step advances"):
        ops.decay_attention_step(q[0], q[0], q[0], torch.ones(2), None)
