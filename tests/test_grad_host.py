"""Autograd at the layers' calls, without a GPU: what has no backward pass says so."""
import types

import pytest
import torch
from torch.autograd import forward_ad

import tilus_b200
from tilus_b200 import BlockNorm, Int8Linear, QuantizedLinear, grad, norm, ops
from tilus_b200 import dtypes as D
from tilus_b200 import linear as linear_module


@pytest.fixture
def plain(monkeypatch):
    """The operators, in elementary operations on the CPU."""
    cast = lambda x: (x.detach().float().round().to(torch.int8), torch.ones(x.shape[0]))  # noqa: E731
    dot = lambda a, b, a_sf, b_sf: (a.float() @ b.float().t()) * a_sf[:, None] * b_sf  # noqa: E731
    monkeypatch.setattr(ops, "per_token_cast_int8", cast)
    monkeypatch.setattr(ops, "int8_matmul", lambda a, b, a_sf, b_sf, bias=None, out_dtype=None, **_: dot(a, b, a_sf, b_sf).to(out_dtype))
    monkeypatch.setattr(ops, "int8_gate_up", lambda a, b, a_sf, b_sf, out_dtype=None, **_: dot(a, b, a_sf, b_sf)[:, ::2].to(out_dtype))
    monkeypatch.setattr(ops, "block_norm", lambda block, residual, weight, **_: (block * weight, block.clone()))
    stub = types.SimpleNamespace(linear=lambda x, qw, sc, layer: x.detach() * 2)
    monkeypatch.setattr(linear_module, "native", lambda: stub)


def _calls():
    x = torch.ones(3, 128, dtype=torch.float16)
    layer = Int8Linear("float16", 128, 32)
    return x, (layer, layer.forward_swiglu, QuantizedLinear("float16", D.int4b, 32, 128, 64))


def test_activations_that_require_a_gradient(plain):
    x, calls = _calls()
    for call in calls:
        want = call(x)
        assert not want.requires_grad
        y = x.clone().requires_grad_()
        got = call(y)
        assert got.requires_grad and torch.equal(got, want)
        with pytest.raises(RuntimeError, match="no gradient with respect to its activations"):
            got.float().sum().backward()
        with torch.no_grad():
            assert not call(y).requires_grad
        assert not call(y.detach()).requires_grad


def test_tangents_are_not_dropped(plain):
    x, calls = _calls()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls[:2]:
            with pytest.raises(RuntimeError):
                call(dual)
            call(x)
        with pytest.raises(RuntimeError):
            norm.block_norm(dual, None, torch.ones(128, dtype=torch.float16))
    assert not grad.followed(x, None)


def test_the_exported_norm_is_the_differentiable_one(monkeypatch):
    assert tilus_b200.block_norm is norm.block_norm
    monkeypatch.setattr(ops, "block_norm", lambda block, residual, weight, **_: (block * weight, block.clone()))
    x, new = tilus_b200.block_norm(torch.ones(2, 8), None, torch.ones(8, requires_grad=True))
    assert x.requires_grad and new.requires_grad
    x, new = BlockNorm("float16", 8)(torch.ones(2, 8, dtype=torch.float16), None)
    assert x.requires_grad
    with torch.no_grad():
        assert not tilus_b200.block_norm(torch.ones(2, 8), None, torch.ones(8, requires_grad=True))[0].requires_grad
