"""Choices from rows of scores on the GPU: settings at their borders, against the definitions in 64 bits (scores_oracle)."""
import ctypes

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


@pytest.mark.parametrize("by_graph", [False, True])
def test_adjust_takes_a_prefix_of_the_paths_as_history(capi, by_graph):  # noqa: F811
    # what of a row of paths lies behind history_columns does not count, whatever it is
    rng = np.random.default_rng(23)
    rows, V, have, stride = 20, 3000, 31, 81
    paths = rng.integers(0, 40, (rows, stride)).astype(np.uint32)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    xadj, adjncy = (np.arange(V + 1) * 20).astype(np.uint32), rng.integers(0, 60, V * 20, dtype=np.uint32)
    g = capi.Graph.upload(xadj, adjncy, None) if by_graph else None
    column = dev(capi, paths, np.uint32)
    rep, frequency = rng.uniform(1, 1.5, rows).astype(np.float32), rng.uniform(0, 1, rows).astype(np.float32)

    class Last:
        ptr = column.ptr.value + 4 * (have - 1)

    m, out = Matrix(capi, x, "f32"), Matrix(capi, x, "f32", 3)
    rules = capi.LogitsRules(history=column, history_columns=have, history_stride=stride, repetition=dev(capi, rep, np.float32), frequency=dev(capi, frequency, np.float32),
                             graph=g, states=Last if by_graph else None, states_stride=stride if by_graph else 0)
    capi.logits_adjust(m, capi.F32, rows, V, rules, out, out_stride=out.stride)
    held = dict(xadj=xadj, adjncy=adjncy, states=paths[:, have - 1]) if by_graph else {}
    want, error = so.adjust(m.values, history=paths[:, :have], rep=rep, frequency=frequency, **held)
    base.near(out.read(), want, error, "f32")
    if g:
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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_draw_from_the_longest_rows(capi, dtype):  # noqa: F811
    # 2^26 columns of one value, and of one in three: the units of 2^26 weights stay below 2^62
    n = 1 << 26
    bits = np.zeros(n, so.storage(dtype))
    need = capi.logits_draw_workspace(base.code(capi, dtype), 1, n)
    tokens, logprobs, kept = capi.DeviceArray(1, np.uint32), capi.DeviceArray(1, np.float32), capi.DeviceArray(1, np.uint32)
    for third in (False, True):
        if third:
            bits[:] = so.to_bits(np.full(1, -INF, np.float32), dtype)[0]
            bits[1::3] = 0
        there = np.count_nonzero(bits == 0)
        m = capi.DeviceArray.from_host(bits)
        for ws in [None] + ([capi.DeviceArray(need, np.uint8)] if need else []):
            for u, k in ((0.0, 0), (0.3, 0), (1 - 2.0 ** -53, 0), (0.5, 20000001)):
                at = dev(capi, [u], np.float64)
                capi.logits_draw(m, base.code(capi, dtype), 1, n, capi.DrawRules(top_k=dev(capi, [k], np.uint32)), tokens, uniforms=at, logprobs=logprobs, kept=kept, workspace=ws)
                stay = min(k or there, there)
                rank = int(u * stay)
                assert (int(tokens.to_host()[0]), int(kept.to_host()[0])) == (3 * rank + 1 if third else rank, stay)
                assert abs(float(logprobs.to_host()[0]) + np.log(stay)) < 1e-6 * np.log(stay)


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


@pytest.mark.parametrize("E,k", [(40, 30), (256, 64), (300, 64), (1000, 20)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_backward_of_ids_whose_experts_are_closed(capi, sigmoid, E, k):  # noqa: F811
    rng = np.random.default_rng(E + k)
    rows = 21
    x = rng.normal(0, 2, (rows, E)).astype(np.float32)
    x = np.where(rng.random(x.shape) < 0.4, rng.choice(np.float32([-INF, np.nan]), x.shape), x).astype(np.float32)
    x[5] = -INF
    ids = np.stack([rng.permutation(E)[:k] for _ in range(rows)]).astype(np.uint32)
    ids[rng.random(ids.shape) < 0.1] = INVALID
    dw = rng.normal(size=(rows, k)).astype(np.float32)
    for renormalise in (False, True):
        m, dx = Matrix(capi, x, "f32", 3), Matrix(capi, np.full(x.shape, 9.0), "f32", 1)
        capi.route_topk_backward(m, capi.F32, rows, E, capi.RouteRules(k, sigmoid=sigmoid, renormalise=renormalise), dev(capi, ids, np.uint32), dev(capi, dw, np.float32), dx,
                                 row_stride=m.stride, dlogits_stride=dx.stride)
        want = so.route_backward(m.values, ids, dw, sigmoid, renormalise, 1.0)
        # as in run_route: exponentials, sums of up to 1,024 and 64 in fp32, over the size of all of the row's gradients
        base.near(dx.read(), want, np.abs(dw).sum(1, keepdims=True) * (40 + 2 * 10) * 2.0 ** -24 + np.zeros_like(want), "f32")


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
class FarRows:
    """Rows so far apart that the last ones' elements have numbers above 2^32, in memory that nothing else is read from."""

    def __init__(self, capi, values, dtype, stride):
        bits, self.values = so.to_bits(values, dtype)
        self.capi, self.dtype, self.stride, self.bits = capi, dtype, stride, bits
        self.dev = capi.DeviceArray((len(bits) - 1) * stride + bits.shape[1], bits.dtype)
        self.ptr = self.dev.ptr.value
        for r in range(len(bits)):
            self._put(r)

    def _put(self, r):
        row = np.ascontiguousarray(self.bits[r])
        assert self.capi.lib().sky_memcpy_h2d(ctypes.c_void_p(self.ptr + r * self.stride * row.itemsize), row.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(row.nbytes)) == 0

    def read(self):
        out = np.empty_like(self.bits)
        for r in range(len(out)):
            row = np.empty(out.shape[1], out.dtype)
            assert self.capi.lib().sky_memcpy_d2h(row.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(self.ptr + r * self.stride * row.itemsize), ctypes.c_size_t(row.nbytes)) == 0
            out[r] = row
        return so.from_bits(out, self.dtype)


@pytest.mark.parametrize("columns", [100, 40000])
def test_rows_that_begin_beyond_32_bits(capi, orc, columns):  # noqa: F811
    rng = np.random.default_rng(29)
    rows, stride = 4, (1 << 31) - 1
    x = rng.normal(0, 3, (rows, columns)).astype(np.float32)
    m, out = FarRows(capi, x, "bf16", stride), FarRows(capi, np.zeros_like(x), "bf16", stride)
    kw = some_rules(rng, rows, columns, 9, 5, 2)
    rules = capi.LogitsRules(history=dev(capi, kw["history"], np.uint32), history_columns=9, repetition=dev(capi, kw["rep"], np.float32),
                             allowed=dev(capi, kw["masks"], np.uint32), allowed_rows=2, allowed_stride=kw["masks"].shape[1], allowed_row=dev(capi, kw["mask_row"], np.uint32))
    capi.logits_adjust(m, capi.BF16, rows, columns, rules, out, row_stride=stride, out_stride=stride)
    want, error = so.adjust(m.values, history=kw["history"], rep=kw["rep"], masks=kw["masks"], mask_row=kw["mask_row"])
    base.near(out.read(), want, error, "bf16")
    tokens, u = capi.DeviceArray(rows, np.uint32), rng.random(rows)
    capi.logits_draw(m, capi.BF16, rows, columns, None, tokens, uniforms=dev(capi, u, np.float64), row_stride=stride)
    assert tokens.to_host().tolist() == [so.draw(m.values[r], u=float(u[r]))[0] for r in range(rows)]
    if columns <= 1024:
        ids, w = capi.DeviceArray(rows * 5, np.uint32), capi.DeviceArray(rows * 5, np.float32)
        for r in (capi.RouteRules(5, sigmoid=True, renormalise=False), capi.RouteRules(5)):
            capi.route_topk(m, capi.BF16, rows, columns, r, ids, w, row_stride=stride)
            chosen = ids.to_host().reshape(rows, 5)
            assert np.array_equal(chosen, so.route(m.values, 5)[0])
            capi.route_topk_backward(m, capi.BF16, rows, columns, r, ids, w, out, row_stride=stride, dlogits_stride=stride)
            dw = w.to_host().reshape(rows, 5)
            want = so.route_backward(m.values, chosen, dw, bool(r.sigmoid), bool(r.renormalise))
            base.near(out.read(), want, np.full(want.shape, 5 * 60 * 2.0 ** -24), "bf16")


# ------------------------------------------------------------------------------------------------ the largest calls
@pytest.mark.parametrize("by_graph", [False, True])
def test_adjust_of_the_widest_row(capi, by_graph):  # noqa: F811
    n, one = 1 << 30, 0x3C003C00  # 1.0 in both halves
    x, out = capi.DeviceArray(n // 2, np.uint32, fill=one), capi.DeviceArray(n // 2, np.uint32, fill=0)
    V = 9000  # a graph's neighbours are among its vertices
    ids = np.array([0, 7, 4095, 4096, 5000, V - 9, V - 1] if by_graph else [0, 7, 4095, 4096, n // 2, n - 9, n - 1], np.uint32)
    xadj = np.full(V + 1, len(ids), np.uint32)
    xadj[0] = 0
    g = capi.Graph.upload(xadj, ids, None) if by_graph else None
    rules = capi.LogitsRules(history=dev(capi, ids[1::2], np.uint32), history_columns=3, presence=dev(capi, [0.5], np.float32), bias_offsets=dev(capi, [0, len(ids)], np.uint32),
                             bias_ids=dev(capi, ids, np.uint32), bias_values=dev(capi, np.arange(len(ids)) + 1.0, np.float32), bias_count=len(ids),
                             graph=g, states=dev(capi, [0], np.uint32) if by_graph else None)
    capi.logits_adjust(x, capi.F16, 1, n, rules, out)
    want = 2.0 + np.arange(len(ids)) - 0.5 * (np.arange(len(ids)) % 2)
    for at in ids.tolist() + [n // 2, n - 1]:
        lo = min(max(at - 40, 0), n - 80)
        near = np.empty(80, np.float16)
        assert capi.lib().sky_memcpy_d2h(near.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(out.ptr.value + 2 * lo), ctypes.c_size_t(160)) == 0
        here = {int(i) - lo: v for i, v in zip(ids, want) if lo <= i < lo + 80}
        assert near.tolist() == [here.get(i, -INF if by_graph else 1.0) for i in range(80)], at
    if g:
        g.free()


def test_adjust_and_route_of_the_most_rows(capi):  # noqa: F811
    rows = 1 << 25
    x = np.random.default_rng(41).integers(-1000, 1000, (rows, 2)).astype(np.float16)
    m, y = capi.DeviceArray.from_host(x), capi.DeviceArray(rows * 2, np.float16)
    capi.logits_adjust(m, capi.F16, rows, 2, capi.LogitsRules(allowed=dev(capi, [1, 2, 3], np.uint32), allowed_rows=3, allowed_row=dev(capi, np.arange(rows) % 3, np.uint32)), y)
    want = x.copy()
    want[0::3, 1] = want[1::3, 0] = -INF
    assert np.array_equal(y.to_host().reshape(rows, 2), want)
    ids, w, counts = capi.DeviceArray(rows, np.uint32), capi.DeviceArray(rows, np.float32), capi.DeviceArray(2, np.uint32)
    capi.route_topk(y, capi.F16, rows, 2, capi.RouteRules(1), ids, w, counts=counts)
    chosen = (want[:, 1] > want[:, 0]).astype(np.uint32)
    assert np.array_equal(ids.to_host(), chosen) and counts.to_host().tolist() == np.bincount(chosen, minlength=2).tolist()
    assert (w.to_host() == 1.0).all()
    capi.route_topk_backward(y, capi.F16, rows, 2, capi.RouteRules(1, sigmoid=True, renormalise=False), ids, w, m)
    z = want.astype(np.float32).max(1)
    s = 1.0 / (1.0 + np.exp(-np.abs(z)))
    got, at = m.to_host().reshape(rows, 2), np.arange(rows)
    assert (got[at, 1 - chosen] == 0).all()
    # three exponentials' worth of fp32 roundings, one to 16 bits
    assert (np.abs(got[at, chosen].astype(np.float64) - s * (1.0 - s)) <= s * (1.0 - s) * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -23).all()


# ------------------------------------------------------------------------------------------------ memory
def test_no_path_of_the_calls_allocates(capi):  # noqa: F811
    rng = np.random.default_rng(19)
    g = capi.Graph.upload(np.array([0, 1, 2], np.uint32), np.array([1, 0], np.uint32), None)
    parts, long, r_in = Matrix(capi, rng.normal(0, 3, (24, 40003)), "f32"), Matrix(capi, rng.normal(0, 3, (300, 21000)), "bf16"), Matrix(capi, rng.normal(0, 2, (50, 300)), "f32")
    need = capi.logits_draw_workspace(capi.F32, 24, 40003)
    assert need > 0
    ws, tokens = capi.DeviceArray(need, np.uint8), capi.DeviceArray(300, np.uint32)
    ids, w, counts, dx = capi.DeviceArray(200, np.uint32), capi.DeviceArray(200, np.float32), capi.DeviceArray(300, np.uint32), capi.DeviceArray(50 * 300, np.float32)
    top_p = capi.DrawRules(top_p=dev(capi, np.full(300, 0.9), np.float32))
    held = capi.LogitsRules(graph=g, states=dev(capi, np.arange(24) % 2, np.uint32))

    def all_calls():
        capi.logits_draw(parts, capi.F32, 24, 40003, top_p, tokens, seed=1, workspace=ws)
        capi.logits_draw(long, capi.BF16, 300, 21000, top_p, tokens, seed=1)
        capi.route_topk(r_in, capi.F32, 50, 300, capi.RouteRules(4), ids, w, counts=counts)
        capi.route_topk_backward(r_in, capi.F32, 50, 300, capi.RouteRules(4), ids, w, dx)
        capi.route_topk(r_in, capi.F32, 50, 200, capi.RouteRules(4), ids, w, counts=counts, row_stride=300)
        capi.logits_adjust(parts, capi.F32, 24, 40003, held, parts)
        capi.synchronize()

    all_calls()
    before, _ = capi.mem_info()
    for _ in range(3):
        all_calls()
    assert capi.mem_info()[0] == before
    g.free()


# ------------------------------------------------------------------------------------------------ together
def test_walk_in_place_with_the_paths_so_far_as_history(capi, orc):  # noqa: F811
    rng = np.random.default_rng(31)
    xadj, adjncy = orc.rmat_csr(11, 10, 5)
    V, N, steps, seed = 2048, 60, 5, 77
    g = capi.Graph.upload(xadj, adjncy, None)
    paths = dev(capi, rng.integers(0, V, (N, steps + 1)), np.uint32)  # columns that are not drawn yet hold anything
    rep, t = rng.uniform(1.0, 1.4, N).astype(np.float32), rng.uniform(0.5, 1.5, N).astype(np.float32)
    d_rep, draw = dev(capi, rep, np.float32), capi.DrawRules(temperature=dev(capi, t, np.float32))
    device = [Matrix(capi, rng.normal(0, 2, (N, V)).astype(np.float32), "bf16", 1, 1) for _ in range(steps)]
    hip = base.Hip()
    side = hip.stream()
    capi.synchronize()

    class Column:
        def __init__(self, at):
            self.ptr = paths.ptr.value + 4 * at

    for i in range(steps):
        rules = capi.LogitsRules(history=paths, history_columns=i + 1, history_stride=steps + 1, repetition=d_rep, graph=g, states=Column(i), states_stride=steps + 1)
        capi.logits_adjust(device[i], capi.BF16, N, V, rules, device[i], row_stride=V + 1, out_stride=V + 1, stream=side)
        capi.logits_draw(device[i], capi.BF16, N, V, draw, Column(i + 1), seed=seed, step=i, tokens_stride=steps + 1, row_stride=V + 1, stream=side)
    capi.synchronize()
    got = paths.to_host((N, steps + 1))
    for i in range(steps):
        want, error = so.adjust(device[i].values, history=got[:, :i + 1], rep=rep, xadj=xadj, adjncy=adjncy, states=got[:, i])
        now = device[i].read()
        base.near(now, want, error, "bf16")
        for r in range(N):
            tok = so.draw(now[r], float(t[r]), u=so.philox_uniform(orc, seed, r, i))[0]
            assert got[r, i + 1] == (INVALID if tok is None else tok)
    hip.hipStreamDestroy(side)
    g.free()


def test_other_paths_in_a_graph(capi):  # noqa: F811
    # rows held to a graph, long 16-bit rows by two kernels, more than 256 experts
    rng = np.random.default_rng(37)
    rows, columns, E = 270, 21000, 400
    degs = rng.integers(0, 1500, columns) * (rng.random(columns) < 0.05)
    xadj = np.concatenate([[0], np.cumsum(degs)]).astype(np.uint32)
    g = capi.Graph.upload(xadj, rng.integers(0, columns, int(xadj[-1]), dtype=np.uint32), None)
    x, r_in = Matrix(capi, rng.normal(0, 3, (rows, columns)), "bf16"), Matrix(capi, rng.normal(0, 2, (rows, E)), "bf16")
    held = capi.LogitsRules(graph=g, states=dev(capi, rng.choice(np.append(np.flatnonzero(degs), INVALID), rows), np.uint32))
    draw = capi.DrawRules(top_p=dev(capi, np.full(rows, 0.8), np.float32), temperature=dev(capi, rng.choice([0.0, 0.5, 1.0], rows), np.float32))
    route = capi.RouteRules(6, bias=dev(capi, rng.uniform(-0.1, 0.1, E), np.float32))

    def outputs():
        z = lambda n, d: dev(capi, np.zeros(n), d)  # noqa: E731
        return dict(y=z(rows * columns, np.uint16), some=z(rows, np.uint32), all=z(rows, np.uint32), lp=z(rows, np.float32), ids=z(rows * 6, np.uint32), w=z(rows * 6, np.float32), counts=z(E, np.uint32),
                    dx=z(rows * E, np.uint16))

    def step(o, s):
        capi.logits_draw(x, capi.BF16, rows, columns, draw, o["all"], seed=3, step=1, logprobs=o["lp"], stream=s)
        capi.logits_adjust(x, capi.BF16, rows, columns, held, o["y"], stream=s)
        capi.logits_draw(o["y"], capi.BF16, rows, columns, draw, o["some"], seed=3, step=2, stream=s)
        capi.route_topk(r_in, capi.BF16, rows, E, route, o["ids"], o["w"], counts=o["counts"], stream=s)
        capi.route_topk_backward(r_in, capi.BF16, rows, E, route, o["ids"], o["w"], o["dx"], stream=s)

    hip, eager, captured = base.Hip(), outputs(), outputs()
    side, graph, ready = hip.stream(), ctypes.c_void_p(), ctypes.c_void_p()
    capi.synchronize()
    step(eager, None)
    capi.synchronize()
    hip.hipStreamBeginCapture(side, 0)
    step(captured, side)
    hip.hipStreamEndCapture(side, ctypes.byref(graph))
    hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0))
    for _ in range(4):
        for m in (x, r_in):
            fresh = so.to_bits(rng.normal(0, 2, m.rows * m.columns).astype(np.float32), "bf16")[0]
            hip.hipMemcpy(m.dev.ptr, fresh.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(fresh.nbytes), 1)
        capi.synchronize()
        hip.hipGraphLaunch(ready, side)
        capi.synchronize()
        step(eager, None)
        capi.synchronize()
        for name in eager:
            assert np.array_equal(eager[name].to_host(), captured[name].to_host()), name
        assert (eager["some"].to_host() == INVALID).any() and (eager["some"].to_host() != INVALID).any()
    hip.hipGraphExecDestroy(ready)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(side)
    g.free()
