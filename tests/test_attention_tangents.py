"""The attention operators, and those around them, have no forward-mode
derivative: inputs that carry a tangent are refused, not answered without one.
Refused before the device is looked at, so no GPU is needed."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import copy_on_write_sdm_amd as cow
from test_attention_host import cache, ints


def calls():
    """Each operator's call, by an input of it."""

    q, k = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)
    rotation, norm = cow.HeadRotation(64, device="cpu"), torch.zeros(64)
    x, w, b, r = torch.zeros(5, 16), torch.zeros(7, 16), torch.zeros(7), torch.zeros(5, 7)
    rotate = lambda **kw: cow.rotate_heads(**{**dict(                           # noqa: E731
        query=q, key=k, positions=ints(5), rotation=rotation, query_norm=norm,
        key_norm=norm), **kw})
    linear = lambda **kw: cow.linear(**{**dict(x=x, weight=w, bias=b, residual=r),  # noqa: E731
                                        **kw})
    for name, t in (("x", x), ("weight", w), ("bias", b), ("residual", r)):
        yield f"linear-{name}", t, lambda t, name=name: linear(**{name: t})
    for name, t in (("query", q), ("key", k), ("query_norm", norm), ("key_norm", norm)):
        yield f"rotate_heads-{name}", t, lambda t, name=name: rotate(**{name: t})
    yield "prompt", k, lambda t: cow.prompt_attention(q, k, t, ints(2))
    yield "write", k, lambda t: cow.write_kv_cache(k, t, ints(5), *cache())
    yield "cached", q, lambda t: cow.cached_attention(t[None], *cache(), ints(1, 2), ints(1))


@pytest.mark.parametrize("name,tensor,call", calls(), ids=[c[0] for c in calls()])
def test_inputs_with_a_tangent(name, tensor, call):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(tensor, torch.ones_like(tensor))
        for off in (False, True):
            with torch.set_grad_enabled(not off), pytest.raises(RuntimeError,
                                                                match="forward-mode"):
                call(dual)
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(forward_ad.unpack_dual(dual).primal)
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(tensor)
