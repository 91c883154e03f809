"""8-bit products, casts and their sums at the ends of their range, against the definitions in 64 bits."""
import pytest
import torch

from tests.test_gpu_int8 import F64, _cast_by_definition, _check, _exact
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


def test_cast_of_nearly_2_to_the_31_rows():
    T = 2 ** 31 - 1
    x = torch.zeros(T, 8, device="cuda", dtype=torch.float16)
    places = [0, T // 2 - 7, T - 50]
    for p in places:
        x[p:p + 50] = torch.randn(50, 8, device="cuda").half()
    codes, sf = ops.per_token_cast_int8(x)
    for p in places:
        want, want_sf = _cast_by_definition(x[p:p + 50])
        assert torch.equal(codes[p:p + 50], want) and torch.equal(sf[p:p + 50], want_sf)


@pytest.mark.parametrize("M,N", [(1, 16), (9, 64), (40, 512), (129, 1024), (260, 64), (700, 272)])
@pytest.mark.parametrize("gated", [False, True])
def test_every_product_of_the_longest_sums_counts(M, N, gated):
    """Partial sums of up to 2^30 that cancel to a small integer, which float16 holds: nothing is lost, nothing there twice.  (The
    shapes go to each kernel, and to the stream kernel with and without a split of K.)"""
    K, rows = 131056, 2 * N if gated else N
    gen = torch.Generator(device="cuda").manual_seed(M)
    half = (K - 16) // 2
    a = torch.full((M, K), -128, device="cuda", dtype=torch.int8)
    b = torch.full((rows, K), 127, device="cuda", dtype=torch.int8)
    b[:, :half] = -127
    a[:, -16:] = torch.randint(-8, 8, (M, 16), generator=gen, device="cuda", dtype=torch.int8)
    b[:, -16:] = torch.randint(-8, 8, (rows, 16), generator=gen, device="cuda", dtype=torch.int8)
    sums = a[:, -16:].to(F64) @ b[:, -16:].to(F64).t()  # at most 16 * 8 * 8
    one = torch.ones(M, device="cuda")
    if gated:
        got = ops.int8_gate_up(a, b, one, torch.full((rows,), 2.0 ** -8, device="cuda"))
        g, u = (sums * 2.0 ** -8).chunk(2, dim=1)
        want = g * torch.sigmoid(g) * u
        _check(got, want, torch.float16, want.abs() * (14 + 1.2 * g.abs()) * 2.0 ** -23)
    else:
        got = ops.int8_matmul(a, b, one, torch.ones(rows, device="cuda"))
        assert torch.equal(got.to(F64), sums)
