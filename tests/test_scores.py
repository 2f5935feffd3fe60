"""Choices from rows of scores: the checks of arguments, which end before any GPU is touched."""
import ctypes as C

import numpy as np
import pytest

import scores_oracle as so

ARG, LIMIT = -1, -5


@pytest.fixture(scope="module")
def capi():
    from skywalker_amd import capi as _capi
    _capi.lib()
    return _capi


class Fake:
    """An address that no call gets as far as using."""

    def __init__(self, address=4096):
        self.ptr = address


def refused(capi, code, word, call, *args, **kw):
    with pytest.raises(capi.SkyError) as e:
        call(*args, **kw)
    assert e.value.code == code and word in str(e.value), str(e.value)


def test_rules_structs_have_the_headers_layout(capi):
    # 19 fields; pointers and 64-bit words are 8 bytes, the two pairs of 32-bit words share 8
    assert C.sizeof(capi.LogitsRules) == 8 * 18
    assert capi.LogitsRules.history_lengths.offset == 24 and capi.LogitsRules.allowed_rows.offset == 8 * 17
    assert C.sizeof(capi.DrawRules) == 32
    assert C.sizeof(capi.RouteRules) == 40 and capi.RouteRules.scale.offset == 24 and capi.RouteRules.bias.offset == 32


def test_adjust_refusals(capi):
    x, y = Fake(), Fake(8192)
    adjust, rules = capi.logits_adjust, capi.LogitsRules
    refused(capi, ARG, "dtype", adjust, x, 3, 1, 8, None, y)
    refused(capi, ARG, "null", adjust, None, capi.F32, 1, 8, None, y)
    refused(capi, ARG, "null", adjust, x, capi.F32, 1, 8, None, None)
    refused(capi, ARG, "stride", adjust, x, capi.F32, 1, 8, None, y, row_stride=7)
    refused(capi, ARG, "stride", adjust, x, capi.F32, 1, 8, None, y, out_stride=7)
    refused(capi, ARG, "in place", adjust, x, capi.F32, 2, 8, None, x, out_stride=9)
    refused(capi, ARG, "aligned", adjust, Fake(4098), capi.F32, 1, 8, None, y)
    refused(capi, ARG, "aligned", adjust, Fake(4097), capi.BF16, 1, 8, None, y)
    refused(capi, LIMIT, "2^31", adjust, x, capi.F32, 1 << 31, 8, None, y)
    refused(capi, LIMIT, "2^31", adjust, x, capi.F32, 1, 1 << 31, None, y)
    refused(capi, ARG, "history", adjust, x, capi.F32, 1, 8, rules(repetition=Fake()), y)
    refused(capi, ARG, "history", adjust, x, capi.F32, 1, 8, rules(history_columns=3), y)
    refused(capi, ARG, "history_stride", adjust, x, capi.F32, 1, 8, rules(history=Fake(), history_columns=3, history_stride=2), y)
    refused(capi, ARG, "biases", adjust, x, capi.F32, 1, 8, rules(bias_ids=Fake(), bias_values=Fake(), bias_count=3), y)
    refused(capi, ARG, "biases", adjust, x, capi.F32, 1, 8, rules(bias_offsets=Fake(), bias_ids=Fake(), bias_count=3), y)
    refused(capi, ARG, "allowed", adjust, x, capi.F32, 1, 8, rules(allowed=Fake()), y)
    refused(capi, ARG, "mask rows", adjust, x, capi.F32, 3, 8, rules(allowed=Fake(), allowed_rows=2), y)
    refused(capi, ARG, "mask rows", adjust, x, capi.F32, 3, 8, rules(allowed_row=Fake()), y)
    refused(capi, ARG, "allowed_stride", adjust, x, capi.F32, 1, 65, rules(allowed=Fake(), allowed_rows=1, allowed_stride=2), y)
    refused(capi, ARG, "states", adjust, x, capi.F32, 1, 8, rules(states=Fake()), y)
    refused(capi, ARG, "aligned", adjust, x, capi.F32, 1, 8, rules(history=Fake(4097), history_columns=1), y)


def test_draw_refusals(capi):
    x, t = Fake(), Fake(8192)
    draw = capi.logits_draw
    refused(capi, ARG, "dtype", draw, x, -1, 1, 8, None, t)
    refused(capi, ARG, "null", draw, None, capi.F16, 1, 8, None, t)
    refused(capi, ARG, "tokens", draw, x, capi.F16, 1, 8, None, None)
    refused(capi, ARG, "stride", draw, x, capi.F16, 1, 8, None, t, row_stride=1)
    refused(capi, ARG, "aligned", draw, x, capi.F16, 1, 8, None, t, uniforms=Fake(4100))
    refused(capi, ARG, "aligned", draw, x, capi.F16, 1, 8, capi.DrawRules(top_k=Fake(4097)), t)
    refused(capi, ARG, "aligned", draw, x, capi.F16, 1, 8, None, t, workspace=Fake(4100), workspace_bytes=1 << 40)
    refused(capi, LIMIT, "2^31", draw, x, capi.F16, 1, 1 << 31, None, t)
    refused(capi, LIMIT, "too large", draw, x, capi.F16, 1 << 30, 8, None, t, row_stride=1 << 40)
    assert capi.lib().sky_logits_draw_workspace(0, 1, 1, None) == ARG
    need = capi.logits_draw_workspace(capi.F32, 3, 100000)
    refused(capi, ARG, "too small", draw, x, capi.F32, 3, 100000, None, t, workspace=Fake(4096), workspace_bytes=need - 1)


def test_route_refusals(capi):
    x, i, w = Fake(), Fake(8192), Fake(16384)
    rules = capi.RouteRules

    def both(code, word, rows, experts, r):
        refused(capi, code, word, capi.route_topk, x, capi.F32, rows, experts, r, i, w)
        refused(capi, code, word, capi.route_topk_backward, x, capi.F32, rows, experts, r, i, w, Fake(32768))

    both(ARG, "rules", 1, 8, None)
    both(ARG, "no experts", 1, 0, rules(1))
    both(ARG, "k must", 1, 8, rules(0))
    both(ARG, "k must", 1, 8, rules(9))
    both(ARG, "groups must", 1, 8, rules(1, groups=3))
    both(ARG, "groups must", 1, 8, rules(1, groups=0))
    both(ARG, "groups_kept", 1, 8, rules(1, groups=4, groups_kept=0))
    both(ARG, "groups_kept", 1, 8, rules(1, groups=4, groups_kept=5))
    both(ARG, "fewer than k", 1, 8, rules(5, groups=4, groups_kept=2))
    both(ARG, "finite", 1, 8, rules(1, scale=float("nan")))
    both(LIMIT, "1024", 1, 1025, rules(1))
    both(LIMIT, "1024", 1, 128, rules(65))
    both(LIMIT, "1024", 1, 130, rules(1, groups=65))
    both(ARG, "aligned", 1, 8, rules(1, bias=Fake(4097)))
    refused(capi, ARG, "null", capi.route_topk, x, capi.F32, 1, 8, rules(1), None, w)
    refused(capi, ARG, "null", capi.route_topk, x, capi.F32, 1, 8, rules(1), i, None)
    refused(capi, ARG, "null", capi.route_topk_backward, x, capi.F32, 1, 8, rules(1), i, None, Fake(32768))
    refused(capi, ARG, "null", capi.route_topk_backward, x, capi.F32, 1, 8, rules(1), i, w, None)


def test_sizes_beyond_a_launch_are_refused(capi):
    x, y = Fake(), Fake(8192)
    refused(capi, LIMIT, "2^30", capi.logits_adjust, x, capi.BF16, 1, (1 << 30) + 1, None, y)
    refused(capi, LIMIT, "threads", capi.logits_adjust, x, capi.BF16, 1 << 23, 8192, None, y)
    refused(capi, LIMIT, "threads", capi.logits_adjust, x, capi.BF16, 1 << 26, 50, None, y)
    refused(capi, LIMIT, "2^26", capi.logits_draw, x, capi.F16, 1, (1 << 26) + 1, None, y)
    refused(capi, LIMIT, "2^25", capi.route_topk, x, capi.F32, (1 << 25) + 1, 8, capi.RouteRules(1), y, Fake(16384))
    refused(capi, LIMIT, "2^25", capi.route_topk_backward, x, capi.F32, (1 << 25) + 1, 8, capi.RouteRules(1), y, Fake(16384), Fake(32768))


def test_no_rows_are_no_work(capi):
    # no GPU is asked for, and no pointer needed
    capi.logits_adjust(None, capi.F32, 0, 8, None, None)
    capi.logits_adjust(Fake(), capi.F32, 3, 0, None, Fake(8192))
    capi.logits_draw(None, capi.BF16, 0, 8, None, None)
    capi.route_topk(None, capi.F32, 0, 8, capi.RouteRules(2), None, None)
    capi.route_topk_backward(None, capi.F32, 0, 8, capi.RouteRules(2), None, None, None)


# ------------------------------------------------------------------------------------------------ the oracle against itself
def test_oracle_draws_with_the_probabilities_of_the_softmax():
    rng = np.random.default_rng(0)
    x = rng.normal(size=7)
    p = np.exp(x / 0.7) / np.exp(x / 0.7).sum()
    n = 200000
    got = np.bincount([so.draw(x, t=0.7, u=(i + 0.5) / n)[0] for i in range(n)], minlength=7) / n
    assert np.abs(got - p).max() < 2 / n * 7
    tok, logp, kept = so.draw(x, t=0.7, u=0.3)
    assert kept == 7 and abs(np.exp(logp) - p[tok]) < 1e-12


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renormalise", [False, True])
def test_oracle_gradient_is_the_slope_of_the_weights(sigmoid, renormalise):
    rng = np.random.default_rng(1)
    x, dw = rng.normal(size=(3, 9)), rng.normal(size=(3, 4))
    ids, _, _ = so.route(x, 4, sigmoid=sigmoid, renormalise=renormalise, scale=1.5)

    def loss(v):
        s = so.scores(v, sigmoid)
        w = so.shares(v, ids, sigmoid) if renormalise else np.take_along_axis(s, ids.astype(np.int64), 1)
        return (1.5 * w * dw).sum()

    got = so.route_backward(x, ids, dw, sigmoid, renormalise, 1.5)
    h = 1e-5
    for r in range(3):
        for e in range(9):
            a, b = x.copy(), x.copy()
            a[r, e] += h
            b[r, e] -= h
            assert abs((loss(a) - loss(b)) / (2 * h) - got[r, e]) < 1e-8  # the step's error is h^2 / 6 of the third derivative
