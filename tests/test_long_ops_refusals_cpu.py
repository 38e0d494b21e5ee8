"""Calls of the long-sequence operators that are refused whatever the device: forward-mode tangents, transforms, and tensors on the host under a trace or a mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad
from torch.utils._python_dispatch import TorchDispatchMode

from dl_templates_amd.paged_cache import paged_append_, paged_attention
from dl_templates_amd.rope_axes import rope_axes_qk, rope_axes_qk_
from dl_templates_amd.window_attn import window_attention


def tensors():
    x, cache = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 16, dtype=torch.bfloat16)
    return x, cache, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32), [torch.zeros(5, 8, 2)]


def calls(x):
    """Every operator on `x` as q, or as k for the append."""
    _, cache, pages, seq, pos, tables = tensors()
    other = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16)
    return {
        "window": lambda: window_attention(x, other, other, 4), "rotation": lambda: rope_axes_qk(x, None, pos, tables)[0], "in place": lambda: rope_axes_qk_(x, None, pos, tables)[0],
        "append": lambda: paged_append_(cache, cache.clone(), x, other, pages, seq, None, (None, tables, "halves"), other), "paged": lambda: paged_attention(x, cache, cache, pages, seq),
    }


NAMES = ["window", "rotation", "in place", "append", "paged"]


@pytest.mark.parametrize("name", ["in place", "append", "paged"])
def test_tangents(name):
    x = torch.ones(1, 2, 4, 16, dtype=torch.bfloat16)
    with fwd_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            calls(fwd_ad.make_dual(x, torch.ones_like(x)))[name]()
    assert (x == 1).all()


@pytest.mark.parametrize("name", NAMES)
def test_transforms(name):
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.vmap(lambda x: calls(x)[name]())(torch.zeros(3, 1, 2, 4, 16, dtype=torch.bfloat16))


@pytest.mark.parametrize("name", NAMES)
def test_host_tensors_under_a_trace_and_a_mode(name):
    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    x = tensors()[0]
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        torch.jit.trace(lambda x: calls(x)[name](), (x,), check_trace=False)
    with Seen(), pytest.raises(RuntimeError, match="ROCm GPU only"):
        calls(x)[name]()
