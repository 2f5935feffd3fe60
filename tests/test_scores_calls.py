"""Choices from rows of scores: what the Python calls hand on and keep, without a GPU."""
import weakref

import pytest


@pytest.fixture(scope="module")
def capi():
    from skywalker_amd import capi as _capi
    _capi.lib()
    return _capi


class Array:
    def __init__(self, address=4096):
        self.ptr = address


@pytest.mark.parametrize("make", [
    lambda c, a: c.LogitsRules(repetition=a, history=a, history_columns=3), lambda c, a: c.DrawRules(top_k=a), lambda c, a: c.RouteRules(2, bias=a)],
    ids=["logits", "draw", "route"])
def test_rules_keep_their_arrays_as_long_as_they_live_and_no_longer(capi, make):
    a = Array()
    alive, rules = weakref.ref(a), make(capi, a)
    del a
    assert alive() is not None
    del rules
    assert alive() is None
