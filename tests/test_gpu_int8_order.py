"""When a product of 8-bit integers may read its operand B: not before the kernel in front of it has ended, unless the caller says
that B has been complete since before that kernel."""
import ctypes
import threading

import pytest
import torch

from tilus_b200 import Int8Linear, QuantizedLinear, _lib, ops
from tilus_b200 import dtypes as D

pytestmark = pytest.mark.gpu
NAMES = ("per_token_cast_int", "igemm", "igemm_swiglu", "block_norm", "block_norm_scratch_bytes", "block_norm_backward")


def _operands(M, rows, K, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-128, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (rows, K), generator=gen, device="cuda", dtype=torch.int8)
    return a, b, (torch.rand(M, generator=gen, device="cuda") + 0.5) / 73, (torch.rand(rows, generator=gen, device="cuda") + 0.5) / (73 * K ** 0.5)


@pytest.fixture
def told(monkeypatch):
    """What the products are told about B: their C entries are replaced by ones that note `early_b` and launch nothing."""
    lib, native, seen = _lib.load(), _lib.native(), []

    def noting(name, place):
        restype, argtypes = _lib.SYMBOLS["b200q_" + name]

        def call(*args):
            seen.append(args[place])
            return 0

        return ctypes.CFUNCTYPE(restype, *argtypes)(call)

    fakes = dict(igemm=noting("igemm", 13), igemm_swiglu=noting("igemm_swiglu", 14))
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
    real = [address(getattr(lib, "b200q_" + n)) for n in NAMES]
    native.bind_int8(*(address(fakes[n]) if n in fakes else a for n, a in zip(NAMES, real)))
    yield seen
    native.bind_int8(*real)


def test_products_are_not_told_that_b_is_at_rest(told):
    """Whatever stands in front, in whatever order: kernels of others, casts on this and other streams, refused calls."""
    a, b, a_sf, b_sf = _operands(4, 64, 128)
    w = torch.randn(64, 128, device="cuda").half()
    ops.int8_matmul(a, b, a_sf, b_sf)
    ops.int8_gate_up(a, b, a_sf, b_sf)
    ops.int8_matmul(a, torch.neg(b), a_sf, b_sf)
    codes, sf = ops.per_token_cast_int8(w)
    ops.int8_matmul(a, b, a_sf, b_sf)  # (another B)
    ops.int8_matmul(a, codes, a_sf, sf)
    codes, sf = ops.per_token_cast_int8(w)
    with pytest.raises(ValueError):
        ops.int8_matmul(a, b, a_sf[:3], b_sf)
    ops.int8_matmul(a, codes, a_sf, sf)
    layer = Int8Linear(torch.float16, 128, 64).cuda()
    layer.forward_cast(a, a_sf)
    layer.forward_swiglu(a, a_sf)
    assert len(told) >= 7 and not any(told)


def test_products_are_told_what_the_caller_says(told):
    a, b, a_sf, b_sf = _operands(4, 64, 128)
    ops.int8_matmul(a, b, a_sf, b_sf, early_b=True)
    ops.int8_gate_up(a, b, a_sf, b_sf, early_b=True)
    layer = Int8Linear(torch.float16, 128, 64).cuda()
    layer.forward_cast(a, a_sf, early_b=True)
    layer.forward_swiglu(a, a_sf, early_b=True)
    x = torch.zeros(4, 128, dtype=torch.float16, device="cuda")
    layer(x)  # (its own cast stands between the weights and the product)
    layer.forward_swiglu(x)
    assert told == [1] * 6


class _Negated(torch.nn.Module):
    def forward(self, w):
        return torch.neg(w)


@pytest.mark.parametrize("M", [1, 40])
def test_weights_computed_on_access(M):
    """A parametrization's kernel runs when the layer's weight is asked for: that is before the cast in front of the product."""
    torch.manual_seed(0)
    layer = Int8Linear(torch.float16, 1024, 4096).cuda()
    layer.load_and_quantize(torch.randn(4096, 1024) / 32)
    x = torch.randn(M, 1024, device="cuda").half()
    want, want_gated = -layer(x), layer.forward_swiglu(x)
    torch.nn.utils.parametrize.register_parametrization(layer, "weight", _Negated(), unsafe=True)
    for _ in range(10):
        assert torch.equal(layer(x), want)
    assert not torch.equal(layer.forward_swiglu(x), want_gated)


@pytest.mark.parametrize("M", [1, 8, 40, 200, 300])
@pytest.mark.parametrize("N", [256, 8192])
def test_b_by_elementwise_kernels_right_in_front(M, N):
    """B is the output of an elementwise kernel of another library, the last one before the product, and of a product's own operands
    nothing else changes."""
    a, b, a_sf, b_sf = _operands(M, N, 1040, seed=1)
    other = torch.randint_like(b, -128, 128)
    flags = torch.rand(b.shape, device="cuda") < 0.5
    forms = (lambda: torch.bitwise_not(other, out=b), lambda: torch.where(flags, other, torch.zeros_like(b), out=b),
             lambda: torch.bitwise_xor(other, 85, out=b))
    wants = []
    for form in forms:
        form()
        torch.cuda.synchronize()
        wants.append(ops.int8_matmul(a, b, a_sf, b_sf))
        torch.cuda.synchronize()
    for i in range(30):
        forms[i % 3]()
        assert torch.equal(ops.int8_matmul(a, b, a_sf, b_sf), wants[i % 3])


@pytest.mark.parametrize("M", [1, 40])
def test_a_refused_call_between_a_cast_and_its_product(M):
    torch.manual_seed(4)
    w = torch.randn(8192, 2048, device="cuda").half()
    x, x_sf = ops.per_token_cast_int8(torch.randn(M, 2048, device="cuda").half())
    bad = torch.zeros(M * 8192 + 4, dtype=torch.float16, device="cuda")[4:].view(M, 8192)
    wants = []
    for sign in (1, -1):
        codes, sf = ops.per_token_cast_int8(w * sign)
        torch.cuda.synchronize()
        wants.append(ops.int8_matmul(x, codes, x_sf, sf))
    negative = -w
    torch.cuda.synchronize()
    for i in range(20):
        codes, sf = ops.per_token_cast_int8(negative if i % 2 else w)
        with pytest.raises(_lib.B200QError):
            ops.int8_matmul(x, codes, x_sf, sf, out=bad)
        assert torch.equal(ops.int8_matmul(x, codes, x_sf, sf), wants[i % 2])


def test_two_threads_on_one_stream():
    """Each casts weights of its own and multiplies by them, on the same stream."""
    torch.manual_seed(5)
    x, x_sf = ops.per_token_cast_int8(torch.randn(4, 1024, device="cuda").half())
    sets = [[(s * torch.randn(2048, 1024, device="cuda")).half() for s in (1, 2)] for _ in range(2)]
    wants = []
    for pair in sets:
        wants.append([])
        for w in pair:
            codes, sf = ops.per_token_cast_int8(w)
            torch.cuda.synchronize()
            wants[-1].append(ops.int8_matmul(x, codes, x_sf, sf))
    torch.cuda.synchronize()
    got = [[], []]

    def work(k):
        for i in range(60):
            codes, sf = ops.per_token_cast_int8(sets[k][i % 2])
            got[k].append((i % 2, ops.int8_matmul(x, codes, x_sf, sf)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 60 and all(torch.equal(out, wants[k][i]) for i, out in got[k])


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("behind", ["cast", "product"])
def test_an_event_behind_a_cast_with_more_on_its_stream(M, behind):
    """A graph whose main stream waits for an event right behind the cast of the weights, after which the other stream goes on."""
    torch.manual_seed(6)
    w, more = torch.randn(4096, 2048, device="cuda").half(), torch.randn(64, 2048, device="cuda").half()
    x, x_sf = ops.per_token_cast_int8(torch.randn(M, 2048, device="cuda").half())
    b, b_sf = ops.per_token_cast_int8(more)
    codes, sf = ops.per_token_cast_int8(w)
    torch.cuda.synchronize()
    want = ops.int8_matmul(x, codes, x_sf, sf)
    static = torch.zeros_like(w)
    side, g, event = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            codes, sf = ops.per_token_cast_int8(static)
            event.record()
            last = ops.per_token_cast_int8(more) if behind == "cast" else ops.int8_matmul(x, b, x_sf, b_sf)
        torch.cuda.current_stream().wait_event(event)
        out = ops.int8_matmul(x, codes, x_sf, sf)
        torch.cuda.current_stream().wait_stream(side)
    for sign in (1, -1, 1, -1):
        static.copy_(w * sign)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want * sign)
    del last


@pytest.mark.parametrize("M", [1, 40])
def test_early_reads_of_weights_at_rest(M):
    """With early_b, behind a cast: the same bits, also where the cast is of the stream's latest weights of another product."""
    a, b, a_sf, b_sf = _operands(M, 4096, 2048, seed=7)
    x = torch.randn(M, 2048, device="cuda").half()
    codes, sf = ops.per_token_cast_int8(x)
    want, want_gated = ops.int8_matmul(codes, b, sf, b_sf), ops.int8_gate_up(codes, b, sf, b_sf)
    torch.cuda.synchronize()
    for _ in range(10):
        codes, sf = ops.per_token_cast_int8(x)
        assert torch.equal(ops.int8_matmul(codes, b, sf, b_sf, early_b=True), want)
        codes, sf = ops.per_token_cast_int8(x)
        assert torch.equal(ops.int8_gate_up(codes, b, sf, b_sf, early_b=True), want_gated)


def test_between_a_weight_only_product_and_a_cast():
    """A layer whose successor starts early in front of a layer that casts: all read what was written."""
    torch.manual_seed(8)
    first = QuantizedLinear("float16", D.int4b, 128, 1024, 1024).cuda()
    first.load_and_quantize(torch.randn(1024, 1024) / 32)
    second = Int8Linear("float16", 1024, 2048).cuda()
    second.load_and_quantize(torch.randn(2048, 1024) / 32)
    x = torch.randn(8, 1024, device="cuda").half()
    h = first(x)
    torch.cuda.synchronize()
    want = second(h)
    torch.cuda.synchronize()
    for _ in range(20):
        assert torch.equal(second(first(x)), want)


@pytest.mark.parametrize("gated", [False, True])
def test_an_output_that_autograd_has_saved(gated):
    """Writing to `out` counts as a change of it, and it must not want a gradient itself."""
    a, b, a_sf, b_sf = _operands(4, 64, 128)
    call = ops.int8_gate_up if gated else ops.int8_matmul
    out = call(a, b, a_sf, b_sf)
    weight = torch.ones_like(out, requires_grad=True)
    y = (out * weight).sum()
    before = out._version
    call(a, b, a_sf, b_sf, out=out)
    after = out._version
    assert after > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="must not require a gradient"):
        call(a, b, a_sf, b_sf, out=weight)
    with torch.no_grad():
        call(a, b, a_sf, b_sf, out=weight)
    with torch.inference_mode():
        static = call(a, b, a_sf, b_sf)
        call(a, b, a_sf, b_sf, out=static)
    assert torch.equal(weight, static) and torch.equal(out, static)
