"""Sizes beyond the 32-bit fields of the sequence-memory operators' argument blocks, and temperatures at the ends of f32, are refused on
the host (no GPU needed: the tensors are stand-ins with a shape and no memory, and every check comes before a launch)."""
import ctypes as C

import pytest
import torch


class _Shape:
    """What the checks read of a GPU tensor."""
    is_cuda, dtype, device = True, torch.float32, torch.device("cuda", 0)

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 64

    def stride(self, i=None):
        s = [1]
        for n in reversed(self.shape[1:]):
            s.insert(0, s[0] * max(1, n))
        return tuple(s) if i is None else s[i]


BIG = [(1 << 31), (1 << 32) + 5]


@pytest.mark.parametrize("big", BIG)
@pytest.mark.parametrize("where", ["steps", "rows", "heads"])
def test_attention_sizes_beyond_32_bits(big, where):
    from purejaxql_amd import _lib, ops
    t, m, h = (big if where == n else 2 for n in ("steps", "rows", "heads"))
    q = _Shape(t, m, h, 4)
    with pytest.raises(ValueError, match=where):
        ops._attn_args(_lib.DecayAttnArgs(), q, q, q, _Shape(h), None, None, 1.0, False)
    if where != "steps":
        q = _Shape(m, h, 4)
        with pytest.raises(ValueError, match=where):
            ops._attn_args(_lib.DecayAttnArgs(), q, q, q, _Shape(h), None, None, 1.0, True)


@pytest.mark.parametrize("big", BIG)
def test_norm_and_logit_sizes_beyond_32_bits(big):
    from purejaxql_amd import ops
    x = _Shape(2, big)
    with pytest.raises(ValueError, match="D: up to"):
        ops._norm_args(x, x, None, "none", {}, "layer_norm", True, True, 1e-6)
    for n, a, says in ((big, 3, "N: up to"), (3, big, "A: up to")):
        with pytest.raises(ValueError, match=says):
            ops._logprob_args(_Shape(n, a), _Shape(n, dtype=torch.int32), None, 1.0, 0)


def test_the_largest_sizes_reach_the_library():
    """2^31 - 1 rows pass the wrappers' check (and the library answers for itself)."""
    from purejaxql_amd import ops
    n = (1 << 31) - 1
    a = ops._logprob_args(_Shape(n, 3), _Shape(n, dtype=torch.int32), None, 1.0, 0)
    assert a.n == n and a.a == 3


@pytest.mark.parametrize("temperature", [3.0e-39, 3.5e-39, 4.2e-39])
def test_temperatures_whose_scale_is_no_float(temperature):
    """1 / temperature is a float there, log2 e / temperature is not: the largest logit itself would come out as 0 * infinity."""
    from purejaxql_amd import _lib
    lib = _lib.load()
    a = _lib.ActionLogprobsArgs(n=4, a=8, top=0, dtype=0, temperature=temperature, logits=64, logits_stride=8, action=64, logp=64, entropy=64, lse=64,
                                dlogp=64, dlogits=64)
    for fn in (lib.pqn_action_logprobs, lib.pqn_action_logprobs_grad):
        a.n = 0                        # nothing would be launched, were it let through
        assert fn(C.byref(a), None) == -1 and "temperature" in lib.pqn_last_error().decode()
    a.temperature = 4.3e-39
    assert lib.pqn_action_logprobs(C.byref(a), None) == 0
