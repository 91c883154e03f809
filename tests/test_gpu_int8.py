"""8-bit integer products, the per-token int8 cast and the layer made of them, against the definitions in 64 bits.

The sums are exact integers.  What the kernels round: a sum's conversion to float32 and the two or three float32 operations
behind it (2^-24 of the value each), and the output (half a step: eps / 2).  The gated form adds float32's fast
exponential (2 + 1.2 |g| units in the last place) and quotient (2).  The tolerances below count these."""
import ctypes

import pytest
import torch

from tests.launches import launches
from tilus_b200 import Int8Linear, QuantizedLinear, _lib, ops
from tilus_b200 import dtypes as D

pytestmark = pytest.mark.gpu
F64 = torch.float64


def _operands(M, rows, K, seed=0, extreme=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-128, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (rows, K), generator=gen, device="cuda", dtype=torch.int8)
    if extreme:
        a.fill_(-128)
        b.fill_(-128)
    a_sf = (torch.rand(M, generator=gen, device="cuda") + 0.5) / 73
    b_sf = (torch.rand(rows, generator=gen, device="cuda") + 0.5) / (73 * K ** 0.5)
    return a, b, a_sf, b_sf


def _exact(a, b, a_sf, b_sf):
    return (a.to(F64) @ b.to(F64).t()) * a_sf.to(F64)[:, None] * b_sf.to(F64)


def _half_step(want, dtype):
    """Half a step of the output's type at each value, subnormals' included."""
    info = torch.finfo(dtype)
    return (want.abs() * info.eps / 2).clamp(min=info.tiny * info.eps / 2)


def _check(got, want, dtype, more):
    assert got.dtype == dtype and got.shape == want.shape
    err = (got.to(F64) - want).abs()
    bound = _half_step(want, dtype) * (1 + 1e-6) + more
    assert bool((err <= bound).all()), float((err / bound).max())


def _gated(c, clamp):
    g, u = c.chunk(2, dim=1)
    if clamp is not None:
        g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
    want = g * torch.sigmoid(g) * u
    return want, want.abs() * (14 + 1.2 * g.abs()) * 2.0 ** -23


SHAPES = [(1, 16, 16), (1, 128, 128), (2, 144, 144), (8, 2048, 4096), (16, 80, 1040), (17, 272, 256), (63, 512, 144),
          (64, 1040, 2048), (65, 400, 384), (100, 11008, 4224), (256, 304, 1024),
          (257, 16, 16), (300, 272, 144), (511, 256, 128), (700, 1296, 2064), (2049, 2048, 256)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_int8_matmul(M, N, K, dtype):
    a, b, a_sf, b_sf = _operands(M, N, K, seed=M)
    bias = torch.randn(N, device="cuda").to(dtype) if K % 32 == 16 else None
    got = ops.int8_matmul(a, b, a_sf, b_sf, bias=bias, out_dtype=dtype)
    c = _exact(a, b, a_sf, b_sf)
    want = c if bias is None else c + bias.to(F64)
    _check(got, want, dtype, 4 * 2.0 ** -24 * (c.abs() + want.abs()))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,clamp", [(torch.float16, None), (torch.bfloat16, 0.75)], ids=["f16", "bf16_clamp"])
def test_int8_gate_up(M, N, K, dtype, clamp):
    a, b, a_sf, b_sf = _operands(M, 2 * N, K, seed=M)
    got = ops.int8_gate_up(a, b, a_sf, b_sf, out_dtype=dtype, swiglu_clamp_value=clamp)
    want, more = _gated(_exact(a, b, a_sf, b_sf), clamp)
    _check(got, want, dtype, more)


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_steep_gates_and_outputs_out_of_range(M, gated):
    """Sums scaled to thousands: gates whose exponential leaves float32's range, and outputs past float16's."""
    a, b, a_sf, b_sf = _operands(M, 64, 512, seed=3)
    b_sf *= 3000.0
    c = _exact(a, b, a_sf, b_sf)
    if gated:
        got = ops.int8_gate_up(a, b, a_sf, b_sf, out_dtype=torch.bfloat16)
        want, more = _gated(c, None)
        _check(got, want, torch.bfloat16, more + 1e-30)  # (quotients by more than 2^126 may be zero)
    else:
        got = ops.int8_matmul(a, b, a_sf * 100, b_sf, out_dtype=torch.float16)
        want = c.mul(100).to(torch.float32).to(torch.float16)
        assert bool(torch.isinf(got).any()) and bool((torch.isinf(got) == torch.isinf(want)).all())


@pytest.mark.parametrize("M", [1, 260])
def test_the_largest_sums_are_exact(M):
    """K = 131056 of the largest products: 128 * 128 * K is just below 2^31."""
    K, N = 131056, 16
    a, b, a_sf, b_sf = _operands(M, N, K, extreme=True)
    got = ops.int8_matmul(a, b, torch.ones_like(a_sf), torch.full_like(b_sf, 2.0 ** -16), out_dtype=torch.bfloat16)
    assert bool((got.to(F64) == torch.tensor(16384.0 * K / 65536).to(torch.bfloat16).item()).all())
    b[:, 1] = 127
    a[:, 1] = 127
    want = 16384 * (K - 1) + 127 * 127
    got = ops.int8_matmul(a, b, torch.ones_like(a_sf), torch.full_like(b_sf, 2.0 ** -16), out_dtype=torch.bfloat16)
    assert bool((got.to(F64) == torch.tensor(want / 65536.0, dtype=F64).to(torch.bfloat16).item()).all())


def _planned(a, b, a_sf, b_sf, out, gated, **edit):
    M, K = a.shape
    N = b.shape[0] // (2 if gated else 1)
    lib, pl = _lib.load(), _lib.IgemmPlan()
    _lib.check(lib.b200q_igemm_plan(M, N, K, int(gated), ctypes.byref(pl)))
    for k, v in edit.items():
        setattr(pl, k, v)
    ws = ops.get_workspace("cuda", 256)
    return lib.b200q_igemm_planned(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), a_sf.data_ptr(), b_sf.data_ptr(), None,
                                   out.data_ptr(), out.stride(0), M, N, K, ops.act_code(out.dtype), int(gated), 0, 0.0, 1,
                                   ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream, ctypes.byref(pl))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 272, 2064), (13, 48, 16), (40, 400, 1040), (130, 144, 304), (200, 272, 1040), (256, 80, 2048),
                                   (256, 16, 1040), (261, 144, 2064), (528, 272, 400)])
def test_every_plan_gives_the_same_bits(M, N, K, gated):
    """The sums being exact, neither the kernel nor the split of K changes a result."""
    a, b, a_sf, b_sf = _operands(M, N * (2 if gated else 1), K, seed=5)
    first = None
    edits = [dict(kernel=1, width=w, ctas=c) for w, c in ((256, 2), (256, 6), (128, 4), (128, 148))]
    if M <= 256:
        edits += [dict(kernel=2, width=w, cluster=c, stages=s)
                  for w, c, s in ((8, 1, 4), (16, 1, 1), (16, 1, 16), (24, 1, 2), (40, 1, 2), (48, 1, 3), (56, 1, 2), (80, 1, 3), (120, 1, 2),
                                  (128, 1, 2), (8, 2, 2), (16, 2, 2), (24, 2, 2), (32, 2, 4), (56, 2, 3), (112, 2, 1), (128, 2, 1),
                                  (40, 3, 2), (48, 3, 2), (16, 4, 2), (72, 4, 2), (96, 4, 2), (128, 4, 3), (80, 5, 5), (112, 7, 2), (64, 8, 1),
                                  (88, 8, 2), (128, 8, 4))
                  if c <= -(-K // 128) and (M <= 64 or c < 5 and s < 16)]  # (what shared memory holds)
    if M <= 16:
        edits += [dict(kernel=3, ctas=c) for c in (1, 3, 300)]
    for edit in edits:
        out = torch.full((M, N), float("nan"), dtype=torch.float16, device="cuda")
        assert _planned(a, b, a_sf, b_sf, out, gated, **edit) == _lib.ST_OK, edit
        first = out if first is None else first
        assert torch.equal(out, first), edit
    assert ops.device_status(ops.get_workspace("cuda", 256)) == [0, 0, 0, 0]


def test_plans_that_cannot_run_are_refused():
    a, b, a_sf, b_sf = _operands(8, 256, 512)
    out = torch.empty(8, 256, dtype=torch.float16, device="cuda")
    good = {1: dict(kernel=1, width=256, ctas=2), 2: dict(kernel=2, width=64, cluster=2, stages=2),
            3: dict(kernel=3, ctas=16)}
    for edit in good.values():
        assert _planned(a, b, a_sf, b_sf, out, False, **edit) == _lib.ST_OK
    for kernel, edit in ((1, dict(kernel=0)), (1, dict(kernel=4)), (1, dict(width=64)), (1, dict(ctas=3)), (1, dict(ctas=0)),
                         (1, dict(ctas=4096)), (2, dict(cluster=9)),
                         (2, dict(cluster=5)), (2, dict(cluster=0)), (2, dict(stages=0)), (2, dict(stages=17)), (2, dict(width=60)), (2, dict(cluster=1, width=4)),
                         (2, dict(width=0)), (2, dict(width=264)), (3, dict(ctas=0))):
        assert _planned(a, b, a_sf, b_sf, out, False, **{**good[kernel], **edit}) == _lib.ST_UNSUPPORTED, edit
    a, b, a_sf, b_sf = _operands(17, 256, 512)
    out = torch.empty(17, 256, dtype=torch.float16, device="cuda")
    assert _planned(a, b, a_sf, b_sf, out, False, **good[3]) == _lib.ST_UNSUPPORTED


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_strided_operands_and_output(M, gated):
    """Rows out of wider matrices on all sides; what lies beside the output stays."""
    N, K = 272, 400
    rows = N * (2 if gated else 1)
    a, b, a_sf, b_sf = _operands(M, rows, K + 48)
    a, b = a[:, 16:16 + K], b[:, 32:32 + K]
    wide = torch.full((M + 2, N + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[1:M + 1, 8:8 + N]
    if gated:
        assert ops.int8_gate_up(a, b, a_sf, b_sf, out_dtype=torch.bfloat16, out=out) is not None
        want = ops.int8_gate_up(a.contiguous(), b.contiguous(), a_sf, b_sf, out_dtype=torch.bfloat16)
    else:
        ops.int8_matmul(a, b, a_sf, b_sf, out_dtype=torch.bfloat16, out=out)
        want = ops.int8_matmul(a.contiguous(), b.contiguous(), a_sf, b_sf, out_dtype=torch.bfloat16)
    assert torch.equal(out, want)
    wide[1:M + 1, 8:8 + N] = 7.0
    assert bool((wide == 7.0).all())


def test_an_output_of_more_than_2_to_the_31_elements():
    M, N, K = 40000, 57344, 16
    a, b, a_sf, b_sf = _operands(M, N, K)
    got = ops.int8_matmul(a, b, a_sf, b_sf)
    for rows in (slice(0, 2), slice(37440, 37460), slice(M - 2, M)):
        want = _exact(a[rows], b, a_sf[rows], b_sf)
        _check(got[rows], want, torch.float16, 4 * 2.0 ** -24 * want.abs())


def test_no_rows():
    a, b, a_sf, b_sf = _operands(4, 32, 64)
    assert ops.int8_matmul(a[:0], b, a_sf[:0], b_sf).shape == (0, 32)
    assert ops.int8_gate_up(a[:0], b, a_sf[:0], b_sf).shape == (0, 16)
    codes, sf = ops.per_token_cast_int8(torch.empty(0, 64, dtype=torch.float16, device="cuda"))
    assert codes.shape == (0, 64) and sf.shape == (0,)


# ---- the cast -------------------------------------------------------------------------------------------------
def _cast_by_definition(x):
    """Quotients and the product rounded to float32 once each, from their exact values (a product of 16 and 24 bits is one
    in 64); the code to the nearest even."""
    x = x.to(F64)
    top = x.abs().amax(1)
    zero = top < 2.0 ** -100
    inv = (127.0 / top.clamp(min=1e-30)).float().to(F64)
    codes = (x * inv[:, None]).float().to(F64).round()
    codes[zero] = 0
    return codes.to(torch.int8), torch.where(zero, torch.ones_like(top), top / 127.0).float()


@pytest.mark.parametrize("T,D", [(1, 8), (1, 4096), (5, 248), (7, 264), (3, 520), (130, 2056), (33, 4104), (9, 14336), (300, 5120),
                                 (2, 16392), (3, 32768), (2, 40008)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_per_token_cast_int8(T, D, dtype):
    torch.manual_seed(D)
    x = (torch.randn(T, D, device="cuda") * 2).to(dtype)
    x[0, 0] = 0
    if T > 2:
        x[1] = 0
        x[2] *= 1e-4
    codes, sf = ops.per_token_cast_int8(x)
    want, want_sf = _cast_by_definition(x)
    assert torch.equal(sf, want_sf) and torch.equal(codes, want)


def test_cast_of_values_on_the_border_of_two_codes():
    """Multiples of half a code: ties go to the even one."""
    x = torch.arange(-254, 255, device="cuda", dtype=torch.float32)[None] / 2
    x = torch.nn.functional.pad(x, (0, 3)).to(torch.float16)  # 512 channels, largest magnitude 127: the scale is 1
    codes, sf = ops.per_token_cast_int8(x)
    assert float(sf) == 1.0 and torch.equal(codes, x.float().round().to(torch.int8))


def test_cast_of_rows_with_nan_infinities_and_tiny_values():
    x = torch.ones(6, 72, dtype=torch.bfloat16, device="cuda")
    x[0, 3] = float("nan")
    x[1, 5] = float("-inf")
    x[2, :] = 1e-38
    x[3, 7] = float("inf")
    x[3, 8] = float("nan")
    x[4] = -0.0
    codes, sf = ops.per_token_cast_int8(x)
    assert bool(torch.isnan(sf[0])) and float(sf[1]) == float("inf") and bool(torch.isnan(sf[3]))
    assert sf[2] == 1 and sf[4] == 1 and bool((codes[[0, 1, 2, 3, 4]] == 0).all()) and bool((codes[5] == 127).all())
    w = torch.ones(16, 80, dtype=torch.int8, device="cuda")
    out = ops.int8_matmul(torch.nn.functional.pad(codes, (0, 8)), w, sf, torch.ones(16, device="cuda"))
    assert bool(torch.isnan(out[[0, 1, 3]]).all()) and bool((out[[2, 4]] == 0).all()) and bool((out[5] == 72).all())


def test_cast_of_strided_rows_and_of_more_than_2_to_the_31_values():
    torch.manual_seed(0)
    x = torch.randn(50, 1000, device="cuda").half()[:, 8:528]
    codes, sf = ops.per_token_cast_int8(x)
    want, want_sf = _cast_by_definition(x)
    assert torch.equal(codes, want) and torch.equal(sf, want_sf)
    x = torch.empty(140000, 16384, dtype=torch.float16, device="cuda")
    x[:2] = 1.5
    x[131072:] = torch.randn(16384, device="cuda").half()
    codes, sf = ops.per_token_cast_int8(x)
    want, want_sf = _cast_by_definition(x[131072:131074])
    assert torch.equal(codes[139990:139992], want) and torch.equal(sf[139990:139992], want_sf)
    assert bool((codes[1] == 127).all())


# ---- the calls in a program -----------------------------------------------------------------------------------
def test_products_read_what_the_kernel_before_them_writes():
    """Both operands come from casts right in front of the product on its stream (which starts setting up before they end)."""
    torch.manual_seed(1)
    for M in (4, 300):
        w = torch.randn(2048, 1024, device="cuda").half()
        x = torch.randn(M, 1024, device="cuda").half()
        wc, wsf = ops.per_token_cast_int8(w)
        xc, xsf = ops.per_token_cast_int8(x)
        torch.cuda.synchronize()
        want = ops.int8_matmul(xc, wc, xsf, wsf)
        for _ in range(20):
            a, a_sf = ops.per_token_cast_int8(x)
            b, b_sf = ops.per_token_cast_int8(w)
            assert torch.equal(ops.int8_matmul(a, b, a_sf, b_sf), want)


@pytest.mark.parametrize("M", [1, 8, 40, 300, 257])
def test_operands_that_other_kernels_write_right_before(M):
    """B and its scales by kernels of another library, on the same stream, directly in front of the product."""
    a, b, a_sf, b_sf = _operands(M, 2064, 1040, seed=1)
    others = [_operands(M, 2064, 1040, seed=s) for s in (2, 3)]
    wants = [ops.int8_matmul(*o) for o in others]
    torch.cuda.synchronize()
    for i in range(40):
        for dst, src in zip((a, a_sf, b_sf, b), others[i % 2][:1] + others[i % 2][2:] + others[i % 2][1:2]):
            dst.copy_(src)
        assert torch.equal(ops.int8_matmul(a, b, a_sf, b_sf), wants[i % 2])


@pytest.mark.parametrize("M", [1, 40])
def test_weights_cast_in_front_of_a_product_that_starts_its_successor_early(M):
    """Between the cast and the product a weight-only product runs, which lets its successor start before the cast has ended."""
    torch.manual_seed(6)
    w = torch.randn(8192, 2048, device="cuda").half()
    x, x_sf = ops.per_token_cast_int8(torch.randn(M, 2048, device="cuda").half())
    between = QuantizedLinear("float16", D.int4b, 128, 1024, 1024).cuda()
    small = torch.randn(16, 1024, device="cuda").half()
    want = []
    for sign in (1, -1):
        c, sf = ops.per_token_cast_int8(sign * w)
        torch.cuda.synchronize()
        want.append(ops.int8_matmul(x, c, x_sf, sf))
    between(small)
    torch.cuda.synchronize()
    for i in range(20):
        c, sf = ops.per_token_cast_int8(w if i % 2 == 0 else -w)
        between(small)
        assert torch.equal(ops.int8_matmul(x, c, x_sf, sf), want[i % 2])


def test_codes_of_a_norm_as_weights():
    """What the norm casts may be B of the product right behind it as well."""
    torch.manual_seed(5)
    block, weight = torch.randn(512, 1024, device="cuda").half(), torch.ones(1024, device="cuda").half()
    x, x_sf = ops.per_token_cast_int8(torch.randn(3, 1024, device="cuda").half())
    codes, sf, _ = ops.block_norm_cast_int8(block, None, weight)
    torch.cuda.synchronize()
    want = ops.int8_matmul(x, codes, x_sf, sf)
    for _ in range(20):
        c, s, _ = ops.block_norm_cast_int8(block, None, weight)
        assert torch.equal(ops.int8_matmul(x, c, x_sf, s), want)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_weights_cast_on_another_stream_of_a_captured_graph(M):
    """A graph of two joined streams: one casts the weights, the other the activations, and multiplies."""
    torch.manual_seed(3)
    w, x = torch.randn(4096, 2048, device="cuda").half(), torch.randn(M, 2048, device="cuda").half()
    want = ops.int8_matmul(*[t for pair in zip(ops.per_token_cast_int8(x), ops.per_token_cast_int8(w)) for t in pair])
    static_w, static_x = torch.zeros_like(w), torch.zeros_like(x)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            wc, wsf = ops.per_token_cast_int8(static_w)
        xc, xsf = ops.per_token_cast_int8(static_x)
        torch.cuda.current_stream().wait_stream(side)
        out = ops.int8_matmul(xc, wc, xsf, wsf)
    for sign in (1, -1, 1, -1):  # each replay has to see its own weights
        static_w.copy_(w * sign)
        static_x.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want * sign)


def test_products_on_two_streams_at_once():
    """Clusters, pairs and two CTAs to an SM of two streams next to one another."""
    shapes = [(64, 1024, 8192, False), (200, 528, 4096, False), (64, 28672, 1024, True), (300, 2048, 1024, False), (9, 4096, 8192, False)]
    sets = [_operands(m, n, k, seed=i) for i, (m, n, k, _) in enumerate(shapes)]
    call = lambda o, gated: ops.int8_gate_up(*o) if gated else ops.int8_matmul(*o)
    wants = [call(o, s[3]) for o, s in zip(sets, shapes)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(40):
        for k, stream in enumerate(streams):
            j = (i + 2 * k) % len(shapes)
            with torch.cuda.stream(stream):
                got.append((j, call(sets[j], shapes[j][3])))
    torch.cuda.synchronize()
    assert all(torch.equal(out, wants[j]) for j, out in got)


def test_other_streams_and_captured_graphs():
    torch.manual_seed(2)
    layer = Int8Linear(torch.bfloat16, 1024, 2048).cuda()
    layer.load_and_quantize(torch.randn(2048, 1024) / 32)
    x = torch.randn(40, 1024, device="cuda").bfloat16()
    want = layer(x)
    want_gated = layer.forward_swiglu(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    static = torch.zeros_like(x)
    for _ in range(2):  # two graphs, replayed on two streams at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = layer(static), layer.forward_swiglu(static)
        graphs.append((g, outs))
    static.copy_(x)
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _), stream in zip(graphs, (side, torch.cuda.Stream())):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, (out, out_gated) in graphs:
        assert torch.equal(out, want) and torch.equal(out_gated, want_gated)


@pytest.mark.parametrize("M,name", [(1, "int8_row_kernel"), (17, "int8_stream_kernel"), (128, "int8_stream_kernel"), (300, "int8_pair_kernel")])
def test_which_kernels_a_layer_launches(M, name):
    layer = Int8Linear(torch.float16, 1024, 4096).cuda()
    x = torch.zeros(M, 1024, dtype=torch.float16, device="cuda")
    layer(x), layer.forward_swiglu(x)
    names = launches(lambda: layer(x), lambda: layer.forward_swiglu(x))
    assert ["cast_int_kernel" in n or name in n for n, _ in names] == [True] * 4 and name in names[1][0] and name in names[3][0]
    assert all(early for _, early in names[1:])


def test_layer_against_dense_weights():
    """The error of 8 bits on both sides: each rounding is off by half a step of absmax / 127, independently, so a sum of K
    products is off by about sqrt(K) times what one is; six deviations hold for every one of 64 * 512 outputs."""
    torch.manual_seed(3)
    K, N, M = 1024, 512, 64
    w, x, bias = torch.randn(N, K) / 32, torch.randn(2, M // 2, K), torch.randn(N)
    layer = Int8Linear("float16", K, N, bias=True)
    layer = layer.cuda()
    layer.load_and_quantize(w.half(), bias)
    out = layer(x.half().cuda())
    assert out.shape == (2, M // 2, N)
    want = x.half().to(F64).view(M, K) @ w.half().to(F64).t() + bias.half().to(F64)
    step_x, step_w = x.half().abs().amax(-1).view(M, 1) / 127, w.half().abs().amax(-1) / 127
    sigma = (K / 12) ** 0.5 * ((step_x * w.std()) ** 2 + (step_w * x.std()) ** 2).sqrt()
    err = (out.view(M, N).cpu().to(F64) - want).abs()
    assert bool((err <= 6 * sigma.to(F64) + want.abs() * 2.0 ** -11).all())
    assert layer.half().scales.dtype == torch.float32 and torch.equal(layer(x.half().cuda()), out)
    copy = Int8Linear("float16", K, N, bias=True).cuda()
    copy.load_state_dict(layer.state_dict())
    assert torch.equal(copy(x.half().cuda()), out)


def test_refusals():
    a, b, a_sf, b_sf = _operands(4, 32, 64)
    for bad in (dict(a=a.float()), dict(b=b.half()), dict(a_sf=a_sf.half()), dict(bias=torch.zeros(32, device="cuda")),
                dict(out=torch.empty(4, 32, device="cuda")), dict(out_dtype=torch.float32)):
        with pytest.raises(TypeError):
            ops.int8_matmul(**{**dict(a=a, b=b, a_sf=a_sf, b_sf=b_sf), **bad})
    for bad in (dict(a=a.cpu()), dict(b=b.cpu()), dict(a=a[0]), dict(a=a.t().contiguous().t()), dict(b=b[:, :48]), dict(a_sf=a_sf[:3]),
                dict(b_sf=torch.ones(64, device="cuda")[::2]), dict(out=torch.empty(4, 16, dtype=torch.float16, device="cuda")),
                dict(bias=torch.zeros(16, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            ops.int8_matmul(**{**dict(a=a, b=b, a_sf=a_sf, b_sf=b_sf), **bad})
    unaligned = torch.zeros(4 * 80 + 8, dtype=torch.int8, device="cuda")
    for bad in (dict(a=unaligned[8:328].view(4, 80)[:, :64]), dict(a=a[:1].expand(4, 64)), dict(a=unaligned[:288].view(4, 72)[:, :64])):
        with pytest.raises(_lib.B200QError) as e:
            ops.int8_matmul(**{**dict(a=a, b=b, a_sf=a_sf, b_sf=b_sf), **bad})
        assert e.value.status == _lib.ST_INVALID_ARG
    for m, n, k in ((4, 24, 64), (4, 32, 72), (1, 16, 131072)):
        with pytest.raises(_lib.B200QError) as e:
            ops.int8_matmul(*_operands(m, n, k))
        assert e.value.status == _lib.ST_UNSUPPORTED
    with pytest.raises(ValueError):
        ops.int8_gate_up(a, b[:31], a_sf, b_sf[:31])
    with pytest.raises(_lib.B200QError):
        ops.int8_gate_up(a, b, a_sf, b_sf, swiglu_clamp_value=float("nan"))
    x = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    for bad, error in ((x.float(), TypeError), (x.cpu(), ValueError), (x[0], ValueError), (x.t().contiguous().t(), ValueError),
                       (x[:, :60], _lib.B200QError), (x[:, 4:60], _lib.B200QError)):
        with pytest.raises(error):
            ops.per_token_cast_int8(bad)
    layer = Int8Linear(torch.float16, 64, 32, bias=True).cuda()
    with pytest.raises(ValueError):
        layer.forward_swiglu(x)
    with pytest.raises(TypeError):
        layer(x.bfloat16())
    with pytest.raises(ValueError):
        layer(x[:, :32])
