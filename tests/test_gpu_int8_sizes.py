"""8-bit products at the ends of their range, against the definitions in 64 bits."""
import pytest
import torch

from tests.test_gpu_int8 import _check, _exact
from tilus_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 17])
def test_nearly_2_to_the_31_columns(M):
    N, K = 2 ** 31 - 16, 16
    gen = torch.Generator(device="cuda").manual_seed(M)
    a = torch.randint(-128, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    b = torch.zeros(N, K, device="cuda", dtype=torch.int8)
    places = [0, N // 2 - 7, N - 40]
    for p in places:
        b[p:p + 40] = torch.randint(-128, 128, (40, K), generator=gen, device="cuda", dtype=torch.int8)
    a_sf, b_sf = torch.rand(M, generator=gen, device="cuda") + 0.5, torch.full((N,), 0.0625, device="cuda")
    out = ops.int8_matmul(a, b, a_sf, b_sf, out_dtype=torch.bfloat16)
    assert out.shape == (M, N)
    for p in places:
        want = _exact(a, b[p:p + 40], a_sf, b_sf[p:p + 40])
        _check(out[:, p:p + 40], want, torch.bfloat16, 4 * 2.0 ** -24 * want.abs())


def test_nearly_2_to_the_31_rows():
    M, N, K = 2 ** 31 - 1, 16, 16
    gen = torch.Generator(device="cuda").manual_seed(0)
    a = torch.zeros(M, K, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (N, K), generator=gen, device="cuda", dtype=torch.int8)
    places = [0, M // 2 - 7, M - 300]
    for p in places:
        a[p:p + 300] = torch.randint(-128, 128, (300, K), generator=gen, device="cuda", dtype=torch.int8)
    a_sf, b_sf = torch.full((M,), 0.0625, device="cuda"), torch.rand(N, generator=gen, device="cuda") + 0.5
    out = ops.int8_matmul(a, b, a_sf, b_sf)
    for p in places:
        want = _exact(a[p:p + 300], b, a_sf[p:p + 300], b_sf)
        _check(out[p:p + 300], want, torch.float16, 4 * 2.0 ** -24 * want.abs())
