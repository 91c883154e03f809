"""Plans of the 8-bit products at the ends of their range."""
import pytest

from tilus_b200 import ops


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 16, 17, 256, 257, 2 ** 31 - 1])
def test_plans_up_to_the_largest_sizes(M, gated):
    for N in (16, 32768, 2 ** 30 - 16) + (() if gated else (2 ** 31 - 272, 2 ** 31 - 16)):
        for K in (16, 144, 131056):
            p = ops.int8_plan(M, N, K, gated)
            if p["kernel"] == 1:
                assert p["width"] in (128, 256) and p["ctas"] % 2 == 0 and 2 <= p["ctas"] <= 148
            elif p["kernel"] == 3:
                assert M <= 16 and 1 <= p["ctas"] <= N // (8 if gated else 16)
            else:
                shares = p["ctas"] // p["cluster"]
                assert M <= 256 and 1 <= shares <= N // 16 and p["ctas"] == shares * p["cluster"]
                assert p["width"] == -(-(N // 8) // shares) * 8 and 16 <= p["width"] <= (128 if gated else 256)
