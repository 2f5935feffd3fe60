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


@pytest.fixture
def draws(capi, monkeypatch):
    """The workspaces and their sizes that draws hand to the library, which is not called."""
    seen = []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        @staticmethod
        def sky_logits_draw(*args):
            seen.append(args[-3:-1])
            return 0

    real = capi.lib()
    monkeypatch.setattr(capi, "_lib", Library())
    return seen


class Sized(Array):
    def __init__(self, nbytes):
        super().__init__(8192)
        self.nbytes = nbytes


def test_a_workspace_made_for_fewer_rows_is_refused(capi):
    columns = 40000
    few, many = capi.logits_draw_workspace(capi.F32, 8, columns), capi.logits_draw_workspace(capi.F32, 40, columns)
    assert 0 < few < many
    with pytest.raises(capi.SkyError) as e:
        capi.logits_draw(Array(), capi.F32, 40, columns, None, Array(16384), workspace=Sized(few))
    assert e.value.code == -1 and "too small" in str(e.value)


def test_draws_hand_on_the_size_that_the_workspace_has(capi, draws):
    def draw(rows, **kw):
        capi.logits_draw(Array(), capi.F32, rows, 40000, None, Array(16384), **kw)
        return draws.pop()

    need = capi.logits_draw_workspace(capi.F32, 8, 40000)
    assert draw(8, workspace=Sized(need)) == (8192, need)
    assert draw(8, workspace=Sized(5 * need)) == (8192, 5 * need)
    assert draw(8, workspace=Sized(5 * need), workspace_bytes=need) == (8192, need)
    assert draw(8, workspace=Array(8192), workspace_bytes=need) == (8192, need)
    assert draw(8) == (None, 0)


def test_a_workspace_of_unknown_size_is_not_written_to(capi, draws):
    with pytest.warns(RuntimeWarning, match="workspace_bytes"):
        capi.logits_draw(Array(), capi.F32, 8, 40000, None, Array(16384), workspace=Array(8192))
    assert draws.pop() == (None, 0)
