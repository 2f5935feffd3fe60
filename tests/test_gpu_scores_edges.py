"""Choices from rows of scores on the GPU: settings at their borders, against the definitions in 64 bits (scores_oracle)."""
import numpy as np
import pytest

import scores_oracle as so
import test_gpu_scores as base
from test_gpu_scores import INF, INVALID, Matrix, capi, dev, run_adjust, run_draw, run_route, some_rules  # noqa: F401  (capi is a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def place_by_place(monkeypatch):
    """Infinities and NaN are compared place by place: what is wanted to be -inf is, and nothing else."""
    def near(got, want, error, dtype):
        gone = ~np.isfinite(want)
        assert np.array_equal(got[gone], want[gone], equal_nan=True)
        assert np.isfinite(got[~gone]).all()
        numbers(got, want, error, dtype)

    numbers = base.near
    monkeypatch.setattr(base, "near", near)


# ------------------------------------------------------------------------------------------------ adjust
def with_odd_values(rng, x):
    """Some NaN and infinities among the logits."""
    at = rng.random(x.shape)
    return np.where(at < 0.01, np.nan, np.where(at < 0.02, INF, np.where(at < 0.03, -INF, x))).astype(np.float32)


def test_the_comparison_tells_infinities_apart():
    z = np.zeros(2)
    for got, want in (([5.0, 1.0], [-INF, 1.0]), ([INF, 1.0], [-INF, 1.0]), ([-INF, 1.0], [1.0, 1.0]), ([np.nan, 1.0], [-INF, 1.0]), ([1.0, 1.0], [np.nan, 1.0])):
        with pytest.raises(AssertionError):
            base.near(np.array(got), np.array(want), z, "f32")
    base.near(np.array([-INF, 1.0]), np.array([-INF, 1.0]), z, "f32")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,columns,history,biases,masks", [
    (1, 1, 1, 1, 1), (4, 1025, 0, 0, 3), (9, 8191, 300, 20, 2), (5, 20011, 3001, 5000, 4), (6, 8193, 0, 0, 1), (40, 70, 9, 5, 40)])
def test_adjusted_rows_place_by_place(capi, dtype, rows, columns, history, biases, masks):  # noqa: F811
    rng = np.random.default_rng(rows * 1000033 + columns)
    x = with_odd_values(rng, rng.normal(0, 4, (rows, columns)))
    kw = some_rules(rng, rows, columns, history, biases, masks)
    for pad, out_pad, lead, in_place in ((0, 0, 0, False), (3, 5, 1, False), (7, 0, 3, True)):
        run_adjust(capi, x, dtype, pad, out_pad, lead, in_place, **kw)


DEGREES = [0, 1, 255, 256, 257, 300, 511, 512, 513, 768, 769, 1000, 1023, 1024, 1025, 1300, 5000]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust_by_a_graph_with_rows_of_every_length(capi, dtype, in_place):  # noqa: F811
    # a workgroup has up to four neighbours a thread in its table; rows of more than 1,024 are done tile by tile
    rng = np.random.default_rng(17)
    V, n = 9001, len(DEGREES)
    xadj = np.concatenate([[0], np.cumsum(DEGREES), np.full(V - n, sum(DEGREES))]).astype(np.uint32)
    adjncy = np.concatenate([rng.permutation(V)[:d] if i % 2 else rng.integers(0, V, d) for i, d in enumerate(DEGREES)]).astype(np.uint32)  # none sorted, half with repetitions
    g = capi.Graph.upload(xadj, adjncy, None)
    states = np.concatenate([rng.permutation(n), [V, INVALID, V - 1]]).astype(np.uint32)
    rows = len(states)
    for columns, stride in ((V, 1), (V - 333, 9), (V + 777, 1)):
        x = with_odd_values(rng, rng.normal(0, 4, (rows, columns)))
        for rules in ((0, 0, 0), (81, 0, 0), (300, 40, 3), (0, 2500, 2)):
            for pad, lead in ((0, 0), (3, 1)):
                run_adjust(capi, x, dtype, pad, 2 * pad, lead, in_place, g=g, stride_of=stride, xadj=xadj, adjncy=adjncy, states=states, **some_rules(rng, rows, columns, *rules))
    g.free()


# ------------------------------------------------------------------------------------------------ draw
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_draw_from_rows_without_columns(capi, dtype):  # noqa: F811
    tokens, logprobs, kept = dev(capi, np.full(3, 777), np.uint32), dev(capi, np.full(3, 5.0), np.float32), dev(capi, np.full(3, 777), np.uint32)
    capi.logits_draw(None, base.code(capi, dtype), 3, 0, None, tokens, logprobs=logprobs, kept=kept)
    assert tokens.to_host().tolist() == [INVALID] * 3 and logprobs.to_host().tolist() == [-INF] * 3 and kept.to_host().tolist() == [0] * 3


@pytest.mark.parametrize("dtype,largest", [("f32", float(np.finfo(np.float32).max)), ("f16", 65504.0), ("bf16", 3.3895313892515355e38)])
@pytest.mark.parametrize("columns", [70, 5000, 40007])
def test_draw_counts_infinity_as_the_largest_number_of_the_type(capi, orc, monkeypatch, dtype, largest, columns):  # noqa: F811
    monkeypatch.setattr(so, "BIG", largest)
    rng = np.random.default_rng(columns)
    x = (rng.normal(0, 0.2, (6, columns)) * largest).clip(-largest, largest).astype(np.float32)
    x[:, [3, 50]], x[:, [7, 20]] = INF, largest
    x[4:, 3::2] = INF
    for t in (largest, largest / 50, 1e-3):
        run_draw(capi, orc, x, dtype, pad=1, t=np.full(6, t), u=rng.random(6), workspace=True)
        run_draw(capi, orc, x, dtype, t=np.full(6, t), top_k=np.array([0, 3, 40, columns // 2, 700, 1]), top_p=np.full(6, 0.9), min_p=np.full(6, 0.01), u=rng.random(6), workspace=True)


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


@pytest.mark.parametrize("E,groups,kept,top2", [(64, 1, 1, False), (300, 1, 1, False), (64, 4, 2, True), (512, 4, 2, True)])
def test_route_of_scores_that_are_equal_in_64_bits(capi, E, groups, kept, top2):  # noqa: F811
    # sigmoids of 40 and more are 1: by the logits themselves where nothing is added to a score, by their sums else
    x = np.full((2, E), -3.0, np.float32)
    x[0, [9, 20, 31]] = [40.0, 60.0, 50.0]
    x[1, [9, 20, 31]] = [50.0, 40.0, 60.0]
    ids = run_route(capi, x, "f32", 3, sigmoid=True, groups=groups, kept=kept, top2=top2)
    assert ids.tolist() == ([[20, 31, 9], [31, 9, 20]] if not top2 else [[9, 20, 31]] * 2)
    for b in (np.zeros(E, np.float32), np.full(E, 0.25, np.float32)):
        assert run_route(capi, x, "f32", 3, sigmoid=True, bias=b, groups=groups, kept=kept, top2=top2).tolist() == [[9, 20, 31]] * 2


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups,kept", [(24, 1, 1), (100, 1, 1), (256, 8, 3), (203, 1, 1), (288, 32, 21), (700, 1, 1), (1024, 4, 2)])
def test_route_past_pairs_of_equal_experts(capi, sigmoid, E, groups, kept):  # noqa: F811
    # scores that fp32 cannot tell apart and fp64 can: the last that is chosen and the first that is not are often the same, and a better one stands behind
    rng = np.random.default_rng(E * 13 + groups)
    if sigmoid:
        x = rng.choice(np.float32([24, 24.5, 26, 30, 17, 2]), (90, E), p=[0.3, 0.2, 0.02, 0.01, 0.37, 0.1])
    else:
        x = np.float32(1.0) + rng.choice(np.float32([0, 1, 2, 3, -2.0 ** 22]), (90, E), p=[0.6, 0.05, 0.03, 0.02, 0.3]) * np.float32(2.0 ** -23)
    x[80:] = x[80:, :1]  # all of a row the same
    x[:, :(groups - kept) * (E // groups)] = -9.0  # groups that are worth less, beyond doubt
    for k in (1, 2, 3, 8, 13, 16):
        for b in (np.zeros(E, np.float32), np.full(E, 0.25, np.float32)):
            run_route(capi, x, "f32", k, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=k % 2 == 1)
