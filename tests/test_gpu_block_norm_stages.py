"""Block norms where a CTA takes several rows through few stages of shared memory, or through gates of several runs of rows.

The gradient's kernel has four stages for narrow rows, two for 32-bit residuals of some 6400 to 9600 channels and 16-bit ones of 9600 to
14400, and one above; with one or two the sum of block block is not taken a row ahead.  The forms and tolerances are those of
test_gpu_block_norm."""
import pytest
import torch

from tests.test_gpu_block_norm import EPS, _check_gradients, _close, _formula, _make
from tilus_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,wide", [(400, 8192, True), (333, 6408, True), (450, 12288, False), (460, 9608, False), (500, 14272, True),
                                      (600, 16384, False), (450, 16384, True), (2000, 4608, True), (3000, 1032, False)])
@pytest.mark.parametrize("post,gates", [(True, 1), (True, 0), (False, 1)])
def test_gradients_of_several_rows_to_a_cta(T, D, wide, post, gates):
    _check_gradients(_make(T, D, torch.bfloat16 if T % 100 else torch.float16, wide=wide, post=post, gates=gates, seed=D, grads=True), 0.75)


@pytest.mark.parametrize("T,D,wide,gates", [(400, 8192, True, 5), (500, 14272, True, 5), (462, 12288, False, 7), (600, 16384, False, 25),
                                            (450, 14272, True, 150), (300, 14272, True, 300), (900, 8192, True, 300), (320, 12288, False, 160)])
def test_gradients_of_several_gates_in_few_stages(T, D, wide, gates):
    """The last of them have more gates than CTAs: each CTA takes gate after gate through the same stages."""
    _check_gradients(_make(T, D, torch.bfloat16, wide=wide, post=True, gates=gates, seed=gates, grads=True), 1.0)


def test_gradients_in_one_stage_without_the_new_residuals():
    s = _make(400, 14272, torch.bfloat16, wide=True, post=True, gates=1, grads=True)
    s["grad_new"] = None
    _check_gradients(s, 0.75)
    s = _make(400, 16384, torch.float16, residual=False, post=True, gates=5, grads=True)
    _check_gradients(s, 0.75)


@pytest.mark.parametrize("T,D,gates", [(900, 4096, 3), (1200, 2304, 600), (888, 3080, 888), (2664, 2056, 2)])
@pytest.mark.parametrize("post", [True, False])
def test_several_gates_where_rows_are_copied_ahead(T, D, gates, post):
    s = _make(T, D, torch.bfloat16, post=post, gates=gates, seed=T)
    x, new = ops.block_norm(**s, residual_scale=0.75, eps=EPS)
    want_x, want_new, size_x, size_new = _formula(s, 0.75)
    _close(x, want_x, size_x)
    _close(new, want_new, size_new)
    codes, sf, again = ops.block_norm_cast_int8(**s, residual_scale=0.75, eps=EPS)
    assert torch.equal(again, new)
    for got, want in zip((codes, sf), ops.per_token_cast_int8(x)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("T,D,wide", [(450, 14272, True), (500, 12288, False)])
def test_the_same_bits_through_few_stages(T, D, wide):
    s = _make(T, D, torch.bfloat16, wide=wide, post=True, gates=5, grads=True)
    call = lambda: ops.block_norm_backward(s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"],  # noqa: E731
                                           post_weight=s["post_weight"], gate=s["gate"])
    first = call()
    for _ in range(5):
        assert all(torch.equal(x, y) for x, y in zip(first, call()))
    assert ops.device_status(ops.get_workspace("cuda", 256)) == [0, 0, 0, 0]
