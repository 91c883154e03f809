"""Block norms (forward, with the int8 cast, and gradients) against their formulas in 64 bits.

Tolerances: everything but the outputs is float32, where each operation is off by 2^-24 of its result.  A statistic
sums at most 64 values in a row (per thread, then over lanes and warps), so with what follows it no value is off by more than
some 100 such roundings of the terms it is made of; `_close` takes 128, of the sum of the terms' magnitudes (a value may be
smaller than its terms), and half a step of the output's type.  Sums over tokens add up to `tokens` terms in a row."""
import pytest
import torch

from tests.launches import launches
from tilus_b200 import BlockNorm, Int8Linear, _lib, norm, ops

pytestmark = pytest.mark.gpu
F64 = torch.float64
EPS = 1e-5


def _make(T, D, dtype, wide=False, post=False, gates=0, residual=True, seed=0, grads=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    rtype = torch.float32 if wide else dtype
    s = dict(block=(n(T, D) * 2).to(dtype), residual=(n(T, D) * 3).to(rtype) if residual else None, weight=(1 + 0.3 * n(D)).to(dtype),
             post_weight=(1 + 0.3 * n(D)).to(dtype) if post else None,
             gate=None if not gates else (0.6 * n(*((D,) if gates == 1 else (gates, D)))).to(dtype))
    if grads:
        s["grad_x"] = n(T, D).to(dtype)
        s["grad_new"] = n(T, D).to(rtype if residual else dtype)
    return s


def _formula(s, scale, eps=EPS):
    """x, the new residual, and the sums of the magnitudes of their terms."""
    up = lambda t: None if t is None else t.to(F64)  # noqa: E731
    block, residual, weight, post, gate = (up(s[k]) for k in ("block", "residual", "weight", "post_weight", "gate"))
    T, D = block.shape
    n = block
    if post is not None:
        n = block * torch.rsqrt(block.square().mean(1, keepdim=True) + eps) * post
    if gate is not None:
        n = n * gate.view(-1, D).repeat_interleave(T // gate.view(-1, D).shape[0], 0)
    old = scale * residual if residual is not None else torch.zeros_like(block)
    r = old + n
    inv = torch.rsqrt(r.square().mean(1, keepdim=True) + eps) * weight
    size = old.abs() + n.abs()
    return r * inv, r, size * inv.abs(), size


def _close(got, want, size, roundings=128):
    assert got.shape == want.shape
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 2.0 ** -24
    bound = (want.abs() + size * roundings * 2.0 ** -24) * half + size * roundings * 2.0 ** -24
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    err = (got.to(F64) - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


CASES = [(1, 8), (1, 4096), (3, 264), (5, 512), (7, 520), (2, 1000), (130, 2048), (1030, 520), (1030, 1032), (1100, 2056), (900, 4096), (33, 4104), (64, 5120), (3, 8192), (2, 8200), (6, 16384)]
FORMS = [dict(), dict(post=True, gates=1), dict(wide=True, gates=1), dict(wide=True, post=True), dict(residual=False, post=True)]


@pytest.mark.parametrize("T,D", CASES)
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_block_norm(T, D, form, dtype):
    s = _make(T, D, dtype, seed=D, **FORMS[form])
    scale = 0.75
    x, new = ops.block_norm(**s, residual_scale=scale, eps=EPS)
    want_x, want_new, size_x, size_new = _formula(s, scale)
    assert x.dtype == dtype and new.dtype == (s["residual"].dtype if s["residual"] is not None else dtype)
    _close(x, want_x, size_x)
    _close(new, want_new, size_new)
    codes, sf, new2 = ops.block_norm_cast_int8(**s, residual_scale=scale, eps=EPS)
    assert torch.equal(new2, new)
    for got, want in zip((codes, sf), ops.per_token_cast_int8(x)):  # the codes are those of the two calls
        assert torch.equal(got, want)


@pytest.mark.parametrize("T,gates", [(6, 2), (12, 12), (300, 3), (64, 1)])
def test_gates_of_several_runs_of_tokens(T, gates):
    s = _make(T, 520, torch.bfloat16, gates=gates if gates > 1 else 0)
    if gates == 1:  # [1, hidden] is a gate for all tokens too
        s["gate"] = torch.randn(1, 520, device="cuda").bfloat16()
    x, new = ops.block_norm(**s, eps=EPS)
    want_x, want_new, size_x, size_new = _formula(s, 1.0)
    _close(x, want_x, size_x)
    _close(new, want_new, size_new)


def _gradients(s, scale, eps=EPS):
    """The formulas' gradients and the sums of the magnitudes of their terms."""
    up = lambda t: None if t is None else t.to(F64)  # noqa: E731
    block, residual, w, post, gate, dx, dnew = (up(s[k]) for k in ("block", "residual", "weight", "post_weight", "gate", "grad_x", "grad_new"))
    T, D = block.shape
    one = torch.ones(1, D, dtype=F64, device="cuda")
    G = 1 if gate is None else gate.view(-1, D).shape[0]
    grow = one if gate is None else gate.view(-1, D).repeat_interleave(T // G, 0)
    s1 = torch.rsqrt(block.square().mean(1, keepdim=True) + eps) if post is not None else torch.ones(T, 1, dtype=F64, device="cuda")
    p = one if post is None else post
    bh = block * s1
    n = bh * p
    old = scale * residual if residual is not None else torch.zeros_like(block)
    r = old + grow * n
    s2 = torch.rsqrt(r.square().mean(1, keepdim=True) + eps)
    xh, xh_size = r * s2, (old.abs() + (grow * n).abs()) * s2
    e = dx * w
    dnew = torch.zeros_like(dx) if dnew is None else dnew
    dr = dnew + s2 * (e - xh * (e * xh).mean(1, keepdim=True))
    dr_size = dnew.abs() + s2 * (e.abs() + xh_size * (e.abs() * xh_size).mean(1, keepdim=True))
    dn, dn_size = grow * dr, grow.abs() * dr_size
    f, f_size = dn * p, dn_size * p.abs()
    db, db_size = f, f_size
    if post is not None:
        db = s1 * (f - bh * (f * bh).mean(1, keepdim=True))
        db_size = s1 * (f_size + bh.abs() * (f_size * bh.abs()).mean(1, keepdim=True))
    runs = lambda t: t.view(G, T // G, D).sum(1)  # noqa: E731
    return {"block": (db, db_size), "residual": (scale * dr, abs(scale) * dr_size),
            "weight": ((dx * xh).sum(0), (dx.abs() * xh_size).sum(0)),
            "post_weight": ((dn * bh).sum(0), (dn_size * bh.abs()).sum(0)), "gate": (runs(dr * n), runs(dr_size * n.abs()))}


def _check_gradients(s, scale, **kw):
    got = ops.block_norm_backward(s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"], post_weight=s["post_weight"],
                                  gate=s["gate"], residual_scale=scale, eps=EPS)
    want = _gradients(s, scale)
    T = s["block"].shape[0]
    for name, g in zip(("block", "residual", "weight", "post_weight", "gate"), got):
        operand = s[name]
        assert (g is None) == (operand is None), name
        if g is None:
            continue
        sums = name not in ("block", "residual")
        assert g.dtype == (torch.float32 if sums else operand.dtype) and g.shape == operand.shape
        value, size = (t.view(g.shape) for t in want[name])
        _close(g, value, size, roundings=256 + (T if sums else 0))
    return got


@pytest.mark.parametrize("T,D", CASES + [(1, 16384), (700, 264), (1030, 1024)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_gradients(T, D, form):
    dtype = torch.bfloat16 if form % 2 else torch.float16
    s = _make(T, D, dtype, seed=T + D, grads=True, **FORMS[form])
    _check_gradients(s, 0.75)


@pytest.mark.parametrize("T,gates,post", [(6, 2, True), (640, 640, False), (600, 300, True), (301, 7, True), (64, 2, False), (96, 24, True),
                                          (120, 30, True), (75, 25, False)])
def test_gradients_of_several_gates(T, gates, post):
    _check_gradients(_make(T, 264, torch.bfloat16, wide=True, post=post, gates=gates, grads=True), 1.0)


@pytest.mark.parametrize("T,gates", [(9, 1), (60, 3), (90, 30), (5, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_gradients_of_gates_of_wide_rows(T, gates, dtype):
    """Above 4096 channels the sums are taken over pairs of them."""
    _check_gradients(_make(T, 4168, dtype, post=True, gates=gates, grads=True), 0.5)


def test_gradients_without_one_of_the_new_residual():
    s = _make(40, 1000, torch.float16, post=True, gates=1, grads=True)
    s["grad_new"] = None
    _check_gradients(s, 1.25)


@pytest.mark.parametrize("name", ["block", "residual", "weight", "post_weight", "gate"])
def test_gradients_against_differences(name):
    """Central differences of the formula in 64 bits along a random direction, of which the kernel's gradient gives the slope.
    Truncation and cancellation are below 1e-6 of it at this step; the outputs' type is off by 2^-12 a value at random."""
    s = _make(24, 264, torch.float16, wide=True, post=True, gates=3, grads=True)
    got = dict(zip(("block", "residual", "weight", "post_weight", "gate"), _check_gradients(s, 0.75)))
    torch.manual_seed(7)
    direction = torch.randn(s[name].shape, device="cuda", dtype=F64)

    def value(h):
        t = dict(s)
        t[name] = s[name].to(F64) + h * direction
        x, new, _, _ = _formula(t, 0.75)
        return float((x * s["grad_x"].to(F64)).sum() + (new * s["grad_new"].to(F64)).sum())

    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    terms = got[name].to(F64) * direction
    assert abs(float(terms.sum()) - slope) <= 1e-5 * abs(slope) + 2.0 ** -11 * float(terms.norm()) + 1e-4


def test_the_same_call_gives_the_same_bits():
    s = _make(900, 4096, torch.bfloat16, post=True, gates=3, grads=True)
    args = (s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"])
    first = ops.block_norm_backward(*args, post_weight=s["post_weight"], gate=s["gate"])
    for _ in range(5):
        again = ops.block_norm_backward(*args, post_weight=s["post_weight"], gate=s["gate"])
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_zero_rows_and_rows_with_nan_stay_among_themselves():
    s = _make(5, 1024, torch.float16, post=True, gates=1, grads=True)
    s["block"][1] = 0
    s["residual"][1] = 0
    s["block"][3, 5] = float("nan")
    x, new = ops.block_norm(**{k: v for k, v in s.items() if not k.startswith("grad")}, eps=EPS)
    assert bool((x[1] == 0).all()) and bool((new[1] == 0).all()) and bool(torch.isnan(x[3]).all())
    assert bool(torch.isfinite(x[[0, 2, 4]]).all())
    got = ops.block_norm_backward(s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"], post_weight=s["post_weight"],
                                  gate=s["gate"], eps=EPS)
    assert bool(torch.isfinite(got[0][[0, 2, 4]]).all()) and bool(torch.isnan(got[0][3]).all())
    # both norms' inverse deviations are eps^-1/2 = 316 in the row of zeros: gradients of some 1e5, of which float16 holds up to 65504
    value = _gradients(s, 1.0)["block"][0][1].abs()
    assert bool(torch.isfinite(got[0][1][value < 65000]).all()) and bool(torch.isinf(got[0][1][value > 66000]).all())
    codes, sf, _ = ops.block_norm_cast_int8(**{k: v for k, v in s.items() if not k.startswith("grad")}, eps=EPS)
    assert bool(torch.isnan(sf[3])) and float(sf[1]) == 1.0 and bool((codes[[1, 3]] == 0).all())


def test_strided_rows():
    s = _make(50, 1040, torch.bfloat16, wide=True, grads=True)
    s = {k: v[:, 16:536] if v is not None and v.dim() == 2 else v[16:536].clone() if v is not None else None for k, v in s.items()}
    s["gate"] = torch.randn(5, 1024, device="cuda").bfloat16()[:, 8:528]
    x, new = ops.block_norm(**{k: v for k, v in s.items() if not k.startswith("grad")}, eps=EPS)
    want_x, want_new, size_x, size_new = _formula(s, 1.0)
    _close(x, want_x, size_x)
    _close(new, want_new, size_new)
    _check_gradients(s, 1.0)


def test_no_tokens():
    s = _make(4, 64, torch.float16, post=True, gates=1, grads=True)
    cut = {k: v[:0] if k in ("block", "residual", "grad_x", "grad_new") else v for k, v in s.items()}
    x, new = ops.block_norm(**{k: v for k, v in cut.items() if not k.startswith("grad")})
    assert x.shape == new.shape == (0, 64)
    got = ops.block_norm_backward(cut["grad_x"], cut["grad_new"], cut["block"], cut["residual"], cut["weight"],
                                  post_weight=cut["post_weight"], gate=cut["gate"])
    assert got[0].shape == (0, 64) and all(bool((g == 0).all()) for g in got[2:])


def test_more_than_2_to_the_31_values():
    T, D = 140000, 16384
    block = torch.zeros(T, D, dtype=torch.float16, device="cuda")
    block[-3:] = torch.randn(3, D, device="cuda").half()
    block[-3, 0] = 3.0
    weight = torch.ones(D, dtype=torch.float16, device="cuda")
    x, new = ops.block_norm(block, None, weight, eps=EPS)
    tail = dict(block=block[-3:], residual=None, weight=weight, post_weight=None, gate=None)
    want_x, want_new, size_x, size_new = _formula(tail, 1.0)
    _close(x[-3:], want_x, size_x)
    _close(new[-3:], want_new, size_new)
    del x, new
    got = ops.block_norm_backward(block, None, block, None, weight, eps=EPS)[0]
    tail |= dict(grad_x=block[-3:], grad_new=None)
    value, size = _gradients(tail, 1.0)["block"]
    _close(got[-3:], value, size, 256)


# ---- the module, and the operators together -------------------------------------------------------------------
def test_module_and_autograd():
    m = BlockNorm(torch.bfloat16, 520, post_norm=True, gated=True, residual_scale=0.75, eps=EPS).cuda()
    s = _make(12, 520, torch.bfloat16, wide=True, post=True, gates=1, grads=True)
    with torch.no_grad():
        for k, v in (("weight", m.weight), ("post_weight", m.post_weight), ("gate", m.gate)):
            v.copy_(s[k])
    block = s["block"].view(3, 4, 520).clone().requires_grad_()
    residual = s["residual"].view(3, 4, 520).clone().requires_grad_()
    x, new = m(block, residual)
    assert x.shape == new.shape == block.shape
    torch.autograd.backward([x, new], [s["grad_x"].view_as(x), s["grad_new"].view_as(new)])
    want = ops.block_norm_backward(s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"], post_weight=s["post_weight"],
                                   gate=s["gate"], residual_scale=0.75, eps=EPS)
    assert torch.equal(block.grad.view(12, 520), want[0]) and torch.equal(residual.grad.view(12, 520), want[1])
    for p, g in ((m.weight, want[2]), (m.post_weight, want[3]), (m.gate, want[4])):
        assert torch.equal(p.grad, g.to(torch.bfloat16))
    # the gradient of a sum is an expanded one; an output that nothing uses has none
    m.zero_grad()
    m(block.detach(), residual.detach())[0].float().sum().backward()
    ones = torch.ones(12, 520, dtype=torch.bfloat16, device="cuda")
    want = ops.block_norm_backward(ones, None, s["block"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                                   residual_scale=0.75, eps=EPS)
    assert torch.equal(m.weight.grad, want[2].to(torch.bfloat16))


def test_capture():
    """The operators are captured; recording gradients under capture is refused before anything is."""
    s = _make(33, 1024, torch.float16, post=True, gates=1, grads=True)
    names = ("block", "residual", "weight", "post_weight", "gate")
    want = ops.block_norm(**{k: s[k] for k in names}), ops.block_norm_backward(
        s["grad_x"], s["grad_new"], s["block"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"])
    static = {k: torch.zeros_like(v) for k, v in s.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.block_norm(**{k: static[k] for k in names}), ops.block_norm_backward(
            static["grad_x"], static["grad_new"], static["block"], static["residual"], static["weight"],
            post_weight=static["post_weight"], gate=static["gate"])
    for k in s:
        static[k].copy_(s[k])
    g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want[0] + want[1], got[0] + got[1]):
        assert torch.equal(w, o)
    weight = s["weight"].clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            norm.block_norm(s["block"], s["residual"], weight)
        with torch.no_grad():
            x, _ = norm.block_norm(s["block"], s["residual"], weight)
    g.replay()
    assert torch.equal(x, ops.block_norm(s["block"], s["residual"], s["weight"])[0])


@pytest.mark.parametrize("T", [1, 40, 600])
def test_a_feed_forward_block(T):
    """Norm and cast, gate_up with SwiGLU, cast, down, and the norm behind it, as a decoder runs them: against the same steps in
    64 bits with the same roundings between them.  A code next to a border may fall to its other side where the steps before
    differ in the last bits; that moves an output by one product of K, so the sums are compared by their norm."""
    torch.manual_seed(T)
    D, H = 1024, 2064
    pre, behind = (BlockNorm(torch.bfloat16, D, post_norm=True, residual_scale=0.9).cuda() for _ in range(2))
    up, down = Int8Linear(torch.bfloat16, D, 2 * H).cuda(), Int8Linear(torch.bfloat16, H, D).cuda()
    up.load_and_quantize(torch.randn(2 * H, D) / 32)
    down.load_and_quantize(torch.randn(D, H) / 45)
    block, residual = torch.randn(T, D, device="cuda").bfloat16(), torch.randn(T, D, device="cuda").bfloat16()

    def run():
        x, sf, res = pre.forward_cast(block, residual)
        h = up.forward_swiglu(x, sf)
        return behind(down(h), res)

    with torch.no_grad():
        x, new = run()
        names = [n for n, _ in launches(run)]
    assert len(names) == 5 and sum("norm_kernel" in n for n in names) == 2 and "cast_int_kernel" in names[2]

    def dot(v, layer):
        top = v.abs().amax(1, keepdim=True)
        codes = (v * (127.0 / top).float().to(F64)).float().to(F64).round()
        return (codes @ layer.weight.to(F64).t()) * (top / 127).float().to(F64) * layer.scales.to(F64)

    s = dict(block=block, residual=residual, weight=pre.weight.data, post_weight=pre.post_weight.data, gate=None)
    v, r, _, _ = _formula(s, 0.9, 1e-6)
    h, _ = (lambda c: (c[:, :H] * torch.sigmoid(c[:, :H]) * c[:, H:], None))(dot(v.bfloat16().to(F64), up))
    c = dot(h.bfloat16().to(F64), down)
    s |= dict(block=c.bfloat16(), residual=r.bfloat16(), weight=behind.weight.data, post_weight=behind.post_weight.data)
    want_x, want_new, _, _ = _formula(s, 0.9, 1e-6)
    # outputs in bf16 (2^-9 at random) of operands in bf16 (as much again)
    assert float((x.to(F64) - want_x).norm() / want_x.norm()) <= 2.0 ** -8
    assert float((new.to(F64) - want_new).norm() / want_new.norm()) <= 2.0 ** -8


def test_refusals():
    s = _make(4, 64, torch.float16, post=True, gates=1)
    call = lambda **bad: ops.block_norm(**{**s, **bad})  # noqa: E731
    cuda = dict(device="cuda", dtype=torch.float16)
    for bad in (dict(block=s["block"].float()), dict(residual=s["residual"].bfloat16()), dict(weight=s["weight"].float()),
                dict(post_weight=s["post_weight"].bfloat16()), dict(gate=s["gate"].float())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(block=s["block"].cpu()), dict(block=s["block"][0]), dict(residual=s["residual"][:3]),
                dict(weight=torch.ones(63, **cuda)), dict(weight=torch.ones(128, **cuda)[::2]), dict(gate=torch.ones(3, 64, **cuda)),
                dict(gate=torch.ones(32, **cuda)), dict(gate=torch.ones(1, 1, 64, **cuda)), dict(gate=torch.ones(0, 64, **cuda)),
                dict(block=s["block"].t().contiguous().t())):
        with pytest.raises(ValueError):
            call(**bad)
    for n in (60, 16392):
        with pytest.raises(_lib.B200QError) as e:
            ops.block_norm(torch.zeros(2, n, **cuda), None, torch.ones(n, **cuda))
        assert e.value.status == _lib.ST_UNSUPPORTED
    odd = torch.zeros(4 * 64 + 4, **cuda)[4:].view(4, 64)
    with pytest.raises(_lib.B200QError):
        call(block=odd)
    with pytest.raises(_lib.B200QError):
        call(residual=s["residual"][:1].expand(4, 64))
    g = torch.zeros(4, 64, **cuda)
    back = lambda gx, gn: ops.block_norm_backward(gx, gn, s["block"], s["residual"], s["weight"])  # noqa: E731
    for gx, gn, error in ((g.float(), None, TypeError), (g[:3], None, ValueError), (g, g.float(), TypeError), (g, g[:3], ValueError),
                          (g[:1].expand(4, 64), None, _lib.B200QError), (g.cpu(), None, ValueError)):
        with pytest.raises(error):
            back(gx, gn)
    m = BlockNorm(torch.float16, 64).cuda()
    with pytest.raises(ValueError):
        m(s["block"][:, :32], None)
    with pytest.raises(ValueError):
        m(s["block"], s["residual"][:2])
