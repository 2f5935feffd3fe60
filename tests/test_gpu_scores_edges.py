"""Choices from rows of scores on the GPU: settings at their borders, against the definitions in 64 bits (scores_oracle)."""
import numpy as np
import pytest

from test_gpu_scores import INF, capi, run_route  # noqa: F401  (capi is a fixture)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ route
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups,kept,k", [(256, 8, 4, 8), (60, 4, 2, 5), (96, 16, 15, 16), (24, 2, 1, 3), (512, 8, 4, 8), (256, 32, 9, 8)])
def test_route_by_groups_with_one_bias_that_is_no_finite_number(capi, sigmoid, E, groups, kept, k):  # noqa: F811
    # one expert's, so that no other group has any; groups that stay and groups that do not lie far apart
    rng = np.random.default_rng(E * 31 + groups)
    x = rng.normal(0, 1, (67, E)).astype(np.float32)
    x += np.repeat(rng.permuted(np.tile(np.linspace(-4, 4, groups), (67, 1)), axis=1), E // groups, axis=1).astype(np.float32)
    bias = rng.uniform(-0.02, 0.02, E).astype(np.float32)
    for odd in (np.nan, -INF, INF):
        for at in (0, E // 2 - 1, E - 1):
            b = bias.copy()
            b[at] = odd
            for top2 in (False, True):
                ids = run_route(capi, x, "f32", k, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=top2, renormalise=not top2)
                assert (ids == at).any(axis=1).all() if odd == INF else not (ids == at).any()
