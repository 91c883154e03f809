"""The 8-bit integer operators and block norms without a GPU: what the C ABI and the Python surface refuse, and plans."""
import ctypes

import pytest
import torch

from tilus_b200 import BlockNorm, Int8Linear, _lib, ops


@pytest.fixture(scope="module")
def lib():
    from tilus_b200 import build

    build.build()
    return _lib.load()


def test_plans():
    """Each plan is one that its kernel can run (what the C ABI demands of an edited one)."""
    for gated in (False, True):
        for m in (1, 8, 9, 16, 17, 64, 65, 200, 256, 257, 272, 273, 4096, 4097, 4113, 100000):
            for n in (16, 1040, 4096, 11008, 28672, 151936):
                for k in (16, 144, 4096, 4112, 14336, 131056):
                    p = ops.int8_plan(m, n, k, gated)
                    if p["kernel"] == 1:
                        assert p["width"] in (128, 256) and p["ctas"] % 2 == 0 and 2 <= p["ctas"] <= 148
                        continue
                    if p["kernel"] == 3:
                        assert m <= 16 and 1 <= p["ctas"] <= n // (8 if gated else 16)
                        continue
                    assert p["kernel"] == 2 and m <= 256 and p["rows"] == -(-m // 16) * 16 and 2 <= p["stages"] <= 16
                    assert p["cluster"] in (1, 2, 4, 8) and p["cluster"] <= -(-k // 128)
                    shares = p["ctas"] // p["cluster"]
                    assert p["ctas"] == shares * p["cluster"] and 1 <= shares <= n // 16
                    assert p["width"] == -(-(n // 8) // shares) * 8 and 16 <= p["width"] <= (128 if gated else 256)
    for m, n, k in ((1, 24, 128), (1, 128, 24), (1, 16, 131072)):
        with pytest.raises(_lib.B200QError) as e:
            ops.int8_plan(m, n, k)
        assert e.value.status == _lib.ST_UNSUPPORTED
    with pytest.raises(_lib.B200QError) as e:
        ops.int8_plan(0, 128, 128)
    assert e.value.status == _lib.ST_INVALID_ARG


def test_bad_pointers_are_refused_before_a_launch(lib):
    ok = 4096  # (an address that is never used)
    good = dict(a=ok, lda=128, b=ok, ldb=128, a_sf=ok, b_sf=ok, bias=None, c=ok, ldc=64, M=4, N=64, K=128, act=0, early=1, ws=ok, nbytes=256,
                stream=None)
    for bad, status in ((dict(a=None), 1), (dict(b=None), 1), (dict(a_sf=None), 1), (dict(b_sf=None), 1), (dict(c=None), 1),
                        (dict(a=ok + 8), 1), (dict(b=ok + 8), 1), (dict(c=ok + 8), 1), (dict(b_sf=ok + 8), 1), (dict(bias=ok + 8), 1),
                        (dict(lda=120), 1), (dict(lda=136), 1), (dict(ldb=112), 1), (dict(ldc=60), 1), (dict(ldc=68), 1),
                        (dict(act=2), 2), (dict(N=24), 2), (dict(K=120), 2), (dict(M=0), 1), (dict(ws=None), 3), (dict(nbytes=255), 3),
                        (dict(ws=ok + 16), 3)):
        assert lib.b200q_igemm(*{**good, **bad}.values()) == status, bad
    assert lib.b200q_per_token_cast_int(None, 64, ok, 64, ok, 1, 64, 0, None) == 1
    assert lib.b200q_per_token_cast_int(ok, 64, ok, 64, ok, 1, 60, 0, None) == 2
    assert lib.b200q_per_token_cast_int(ok, 56, ok, 64, ok, 1, 64, 0, None) == 1
    assert lib.b200q_per_token_cast_int(ok + 8, 64, ok, 64, ok, 1, 64, 0, None) == 1
    assert lib.b200q_per_token_cast_int(ok, 64, ok, 64, ok, 1, 64, 2, None) == 2


def _norm(**bad):
    n = _lib.BlockNorm()
    for k, v in {**dict(block=4096, residual=4096, weight=4096, ldb=64, ldr=64, tokens=4, hidden=64, residual_scale=1.0, eps=1e-6),
                 **bad}.items():
        setattr(n, k, v)
    return ctypes.byref(n)


def test_bad_norms_are_refused_before_a_launch(lib):
    ok = 4096
    for bad, status in ((dict(block=None), 1), (dict(weight=None), 1), (dict(block=ok + 8), 1), (dict(residual=ok + 8), 1),
                        (dict(post_weight=ok + 8), 1), (dict(ldb=56), 1), (dict(ldr=68), 1), (dict(tokens=0), 1),
                        (dict(hidden=60), 2), (dict(hidden=16392, ldb=16392, ldr=16392), 2), (dict(act_dtype=2), 2),
                        (dict(gate=ok), 1), (dict(gates=1), 1), (dict(gate=ok, gates=3, ldg=64), 1), (dict(gate=ok, gates=2, ldg=56), 1)):
        assert lib.b200q_block_norm(_norm(**bad), ok, 64, None, None, ok, 64, None) == status, bad
    for x, codes, sf, new, ldx in ((None, None, None, ok, 64), (ok, ok, ok, ok, 64), (None, ok, None, ok, 64), (ok, None, None, None, 64),
                                   (ok, None, None, ok, 56), (ok + 8, None, None, ok, 64)):
        assert lib.b200q_block_norm(_norm(), x, ldx, codes, sf, new, 64, None) == 1
    assert lib.b200q_block_norm(None, ok, 64, None, None, ok, 64, None) == 1
    good = dict(args=_norm(), dx=ok, lddx=64, dn=None, lddn=0, db=ok, lddb=64, dr=ok, lddr=64, dw=ok, dp=None, dg=None, s=ok,
                n=1 << 30, ws=ok, ws_bytes=256, stream=None)
    for bad, status in ((dict(dx=None), 1), (dict(db=None), 1), (dict(dw=None), 1), (dict(dp=ok), 1), (dict(dg=ok), 1),
                        (dict(args=_norm(residual=None)), 1), (dict(lddx=60), 1), (dict(dn=ok, lddn=60), 1), (dict(dw=ok + 8), 1),
                        (dict(s=None), 3), (dict(n=16), 3), (dict(s=ok + 8), 3), (dict(ws=None), 3), (dict(ws_bytes=255), 3)):
        assert lib.b200q_block_norm_backward(*{**good, **bad}.values()) == status, bad
    assert lib.b200q_block_norm_scratch_bytes(4, 60, 0) == 0 and lib.b200q_block_norm_scratch_bytes(4, 64, 3) == 0
    assert lib.b200q_block_norm_scratch_bytes(4, 64, 2) > 0


def test_cpu_tensors_are_refused(lib):
    a, sf = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    x = torch.zeros(4, 64, dtype=torch.float16)
    w = torch.ones(64, dtype=torch.float16)
    for call in (lambda: ops.per_token_cast_int8(x), lambda: ops.int8_matmul(a, a, sf, sf), lambda: ops.int8_gate_up(a, a, sf, sf),
                 lambda: ops.block_norm(x, x, w), lambda: ops.block_norm_cast_int8(x, None, w),
                 lambda: ops.block_norm_backward(x, None, x, x, w), lambda: BlockNorm("float16", 64)(x, None),
                 lambda: Int8Linear("float16", 64, 32)(x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        ops.per_token_cast_int8([1.0])


def test_layers_refuse_sizes_and_keep_their_scales():
    for k, n in ((24, 32), (32, 24), (0, 16), (16, 0)):
        with pytest.raises(ValueError):
            Int8Linear("float16", k, n)
    for d in (0, 12, 16392):
        with pytest.raises(ValueError):
            BlockNorm("float16", d)
    layer = Int8Linear("bfloat16", 32, 64, bias=True).to(torch.float16)
    assert layer.scales.dtype == torch.float32 and layer.weight.dtype == torch.int8
    with pytest.raises(ValueError):
        layer.load_and_quantize(torch.zeros(64, 32))
    with pytest.raises(ValueError):
        layer.load_and_quantize(torch.zeros(32, 64), torch.zeros(64))
