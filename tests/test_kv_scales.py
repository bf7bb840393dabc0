"""Attention's scale through the C ABI, without a GPU: one that is not finite, or not with log2 e, is refused (a row that sees no key has to be zeros, and
minus infinity times it would be NaN)."""
import math

import pytest

from tests.test_kv_arguments import ARG, attn, p  # noqa: F401


@pytest.mark.parametrize("chosen", [False, True])
def test_scales(qm, p, chosen):  # noqa: F811
    for scale in (math.nan, math.inf, -math.inf, 2.4e38, -3.4e38):
        assert attn(qm, p, chosen, scale=scale) == ARG and attn(qm, p, chosen, T=0, B=0, scale=scale) == ARG
    for scale in (0.0, -0.0, 1e-45, -0.5, 2.3e38):
        assert attn(qm, p, chosen, T=0, B=0, scale=scale) == 0
