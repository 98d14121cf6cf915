"""cml_moe_route_scored: softmax scores with a balance bias, every row compared; and tokens of one call in several launches.

Biases are spread over [-1, 1] without a grid, so that keys come within 1e-5 of each other at a decision by chance alone, and in none of these rows do they: all are
compared.
"""
import numpy as np
import pytest

from camelid_amd import binding as B
from tests import gpu_util as G
from tests.test_gpu_route_scored import SIGMOID, SOFTMAX, compare, route
from tests.typed_rows import to_bits

pytestmark = pytest.mark.gpu

CASES = [(256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (64, 16, 3, 2, 5), (60, 5, 2, 2, 7), (48, 48, 6, 2, 6), (64, 64, 64, 1, 64), (1024, 64, 9, 2, 20), (1024, 1, 1, 1, 16), (12, 1, 1, 2, 3), (320, 4, 4, 2, 16)]


def inputs(experts, groups):
    rng = np.random.default_rng(experts + groups)
    return (rng.integers(-32, 32, (24, experts)) / 4.0).astype(np.float32), rng.uniform(-1, 1, experts).astype(np.float32)


@pytest.mark.parametrize("quarter", [0, 1])
@pytest.mark.parametrize("renormalise", [0, 1])
@pytest.mark.parametrize("experts,groups,kept,group_top,k", CASES)
def test_softmax_with_bias(experts, groups, kept, group_top, k, renormalise, quarter):
    logits, bias = inputs(experts, groups)
    with G.env(CAMELID_HIP_ROUTE_QUARTER=1 if quarter else 1 << 30):
        compare(SOFTMAX, "f32", to_bits(logits, "f32"), bias, groups, kept, group_top, k, renormalise, 2.5, least=1.0)


@pytest.mark.parametrize("quarter", [0, 1])
def test_tokens_in_several_launches(quarter):
    B.init(0)
    rng = np.random.default_rng(1)
    logits, bias = to_bits(rng.standard_normal((301, 64)), "bf16"), rng.uniform(-0.1, 0.1, 64).astype(np.float32)
    for score in (SOFTMAX, SIGMOID):
        with G.env(CAMELID_HIP_ROUTE_QUARTER=1 if quarter else 1 << 30):
            want = route(score, "bf16", logits, bias, 4, 2, 2, 6, pad=3)
        name = "moe.route.scored.quarter" if quarter else "moe.route.scored"
        before = G.launch_counts().get(name, 0)
        with G.env(CAMELID_HIP_ROUTE_QUARTER=1 if quarter else 1 << 30, CAMELID_HIP_LAUNCH_ITEMS=1024):
            got = route(score, "bf16", logits, bias, 4, 2, 2, 6, pad=3)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        assert G.launch_counts().get(name, 0) - before > 1
