"""Choices from rows of scores on the GPU against their definitions in 64 bits (scores_oracle)."""
import ctypes

import numpy as np
import pytest

import scores_oracle as so

pytestmark = pytest.mark.gpu
INVALID = 0xFFFFFFFF
INF = np.inf


@pytest.fixture(scope="module")
def capi():
    from skywalker_amd import capi as _capi
    return _capi


def code(capi, dtype):
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[dtype]


class Matrix:
    """Rows in device memory with `pad` elements between them, `lead` in front and guards that nothing may touch."""

    def __init__(self, capi, values, dtype, pad=0, lead=0):
        bits, self.values = so.to_bits(values, dtype)
        self.rows, self.columns = values.shape
        self.stride, self.lead, self.dtype, self.pad = self.columns + pad, lead, dtype, pad
        self.host = np.full(lead + self.rows * self.stride + 64, 0x1234 if dtype != "f32" else 7.25, so.storage(dtype))
        if dtype == "f16":
            self.host[:] = np.float16(7.25)
        self._view(self.host)[:, :self.columns] = bits
        self.dev = capi.DeviceArray.from_host(self.host)
        self.ptr = self.dev.ptr.value + lead * self.host.itemsize

    def _view(self, flat):
        return flat[self.lead:self.lead + self.rows * self.stride].reshape(self.rows, self.stride)

    def read(self):
        """Values as float64; what lies around them is checked to be as it was."""
        flat = self.dev.to_host()
        got = so.from_bits(self._view(flat)[:, :self.columns], self.dtype)
        same = flat.copy()
        self._view(same)[:, :self.columns] = self._view(self.host)[:, :self.columns]
        assert np.array_equal(same.view(np.uint8), self.host.view(np.uint8)), "memory around the rows was written"
        return got


def near(got, want, error, dtype):
    """got is want, rounded to its type, of a value that is off by at most `error`."""
    gone = ~np.isfinite(want)
    assert np.array_equal(got[gone], want[gone]) or (np.isnan(want[gone]) == np.isnan(got[gone])).all()
    w, g, e = want[~gone], got[~gone], error[~gone]
    bound = e + (np.abs(w) + e) * so.HALF_STEP[dtype] + so.TINY[dtype]
    assert (np.abs(g - w) <= bound).all(), np.max(np.abs(g - w) / bound)


# ------------------------------------------------------------------------------------------------ adjust
def dev(capi, a, dtype):
    return None if a is None else capi.DeviceArray.from_host(np.ascontiguousarray(a, dtype))


def run_adjust(capi, x, dtype, pad=0, out_pad=0, lead=0, in_place=False, g=None, stride_of=1, **kw):
    rows, columns = x.shape
    m = Matrix(capi, x, dtype, pad, lead)
    out = m if in_place else Matrix(capi, np.full(x.shape, 99.0), dtype, out_pad, (lead * 3) % 7)
    h = kw.get("history")
    masks, states = kw.get("masks"), kw.get("states")
    if states is not None:
        spread = np.full((rows, stride_of), 12345, np.uint32)
        spread[:, 0] = states
        states = spread
    rules = capi.LogitsRules(
        history=dev(capi, h, np.uint32), history_columns=0 if h is None else h.shape[1],
        history_lengths=dev(capi, kw.get("lengths"), np.uint32), history_first=dev(capi, kw.get("first"), np.uint32),
        repetition=dev(capi, kw.get("rep"), np.float32), presence=dev(capi, kw.get("presence"), np.float32),
        frequency=dev(capi, kw.get("frequency"), np.float32), bias_offsets=dev(capi, kw.get("offsets"), np.uint32),
        bias_ids=dev(capi, kw.get("ids"), np.uint32), bias_values=dev(capi, kw.get("values"), np.float32),
        bias_count=0 if kw.get("ids") is None else len(kw["ids"]), allowed=dev(capi, masks, np.uint32),
        allowed_rows=0 if masks is None else masks.shape[0], allowed_stride=0 if masks is None else masks.shape[1],
        allowed_row=dev(capi, kw.get("mask_row"), np.uint32), graph=g, states=dev(capi, states, np.uint32), states_stride=stride_of if states is not None else 0)
    capi.logits_adjust(m, code(capi, dtype), rows, columns, rules, out, row_stride=m.stride, out_stride=out.stride)
    capi.synchronize()
    if not in_place:
        m.read()
    want, error = so.adjust(m.values, **kw)
    near(out.read(), want, error, dtype)
    return out


def some_rules(rng, rows, columns, history=0, biases=0, masks=0):
    kw = {}
    if history:
        kw["history"] = np.where(rng.random((rows, history)) < 0.1, INVALID, (columns * rng.random((rows, history)) ** 3).astype(np.uint32)).astype(np.uint32)
        kw["lengths"] = rng.integers(0, history + 3, rows)
        kw["first"] = rng.integers(0, history + 1, rows)
        kw["rep"], kw["presence"], kw["frequency"] = rng.uniform(0.8, 1.6, rows).astype(np.float32), rng.uniform(-1, 1, rows).astype(np.float32), rng.uniform(0, 0.5, rows).astype(np.float32)
    if biases:
        n = rng.integers(0, biases + 1, rows)
        kw["offsets"] = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
        kw["ids"] = np.concatenate([np.sort(rng.integers(0, columns + 2, k)) for k in n] + [[1]]).astype(np.uint32)
        kw["values"] = rng.uniform(-8, 8, kw["ids"].size).astype(np.float32)
    if masks:
        words = (columns + 31) // 32
        kw["masks"] = rng.integers(0, 1 << 32, (masks, words + 1), dtype=np.uint32) & rng.integers(0, 1 << 32, (masks, words + 1), dtype=np.uint32)
        kw["mask_row"] = rng.choice(np.append(np.arange(masks + 1), INVALID), rows).astype(np.uint32)
    return kw


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,columns,history,biases,masks", [
    (1, 1, 1, 1, 1), (3, 7, 0, 0, 0), (2, 64, 5, 0, 0), (5, 1000, 0, 40, 0), (4, 1025, 0, 0, 3), (3, 8191, 300, 20, 2), (2, 8200, 81, 0, 0),
    (2, 20011, 3001, 5000, 4), (7, 4096, 1, 0, 0), (2, 8193, 0, 0, 1)])
def test_adjust_follows_its_formula(capi, dtype, rows, columns, history, biases, masks):
    rng = np.random.default_rng(rows * 1000003 + columns)
    x = rng.normal(0, 4, (rows, columns)).astype(np.float32)
    kw = some_rules(rng, rows, columns, history, biases, masks)
    for pad, out_pad, lead in ((0, 0, 0), (3, 5, 1), (8, 1, 3)):
        run_adjust(capi, x, dtype, pad, out_pad, lead, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_adjust_in_place(capi, dtype):
    rng = np.random.default_rng(5)
    for columns, pad, lead in ((1000, 0, 0), (9001, 7, 3)):
        x = rng.normal(0, 4, (6, columns)).astype(np.float32)
        run_adjust(capi, x, dtype, pad, lead=lead, in_place=True, **some_rules(rng, 6, columns, 50, 30, 3))


def test_adjust_without_rules_copies(capi):
    x = np.array([[1.5, -0.0, INF, -INF, np.nan, 3e38]], np.float32)
    m, out = Matrix(capi, x, "f32"), Matrix(capi, np.zeros((1, 6)), "f32")
    capi.logits_adjust(m, capi.F32, 1, 6, None, out)
    assert np.array_equal(out.read().astype(np.float32).view(np.uint32)[:, :4], x.view(np.uint32)[:, :4]) and np.isnan(out.read()[0, 4])


def test_adjust_masks_take_out_whatever_is_there(capi):
    x = np.array([[np.nan, INF, -INF, np.finfo(np.float32).min, 1.0, np.nan]], np.float32)
    out = run_adjust(capi, np.nan_to_num(x, nan=INF, posinf=INF), "f32", masks=np.array([[0b010000]], np.uint32))
    assert out.read()[0].tolist() == [-INF, -INF, -INF, -INF, 1.0, -INF]
    m, out = Matrix(capi, x, "f32"), Matrix(capi, np.zeros((1, 6)), "f32")
    capi.logits_adjust(m, capi.F32, 1, 6, capi.LogitsRules(allowed=dev(capi, [0b010000], np.uint32), allowed_rows=1), out)
    assert out.read()[0].tolist() == [-INF, -INF, -INF, -INF, 1.0, -INF]


def test_adjust_one_mask_row_serves_all_rows_and_equal_biases_add_up(capi):
    rng = np.random.default_rng(6)
    x = rng.normal(0, 2, (3, 70)).astype(np.float32)
    run_adjust(capi, x, "f32", masks=rng.integers(0, 1 << 32, (1, 3), dtype=np.uint32))
    run_adjust(capi, x, "f32", masks=rng.integers(0, 1 << 32, (3, 3), dtype=np.uint32))
    run_adjust(capi, x, "f32", offsets=np.array([0, 4, 4, 90]), ids=np.array([5, 5, 5, 80, 0, 0, 69]), values=np.array([1, 2, 4, 100, 3, -1, 2.0]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_adjust_by_a_graph(capi, dtype):
    rng = np.random.default_rng(7)
    V = 9000
    degs = np.where(rng.random(V) < 0.3, 0, rng.integers(1, 40, V))
    degs[17] = 5000
    xadj = np.concatenate([[0], np.cumsum(degs)]).astype(np.uint32)
    adjncy = rng.integers(0, V, xadj[-1], dtype=np.uint32)  # unsorted, with repetitions
    g = capi.Graph.upload(xadj, adjncy, None)
    states = np.array([17, 0, V, INVALID, 3, V - 1, 17], np.uint32)
    for columns, stride in ((V, 1), (V - 333, 9), (V + 777, 1)):
        x = rng.normal(0, 4, (7, columns)).astype(np.float32)
        kw = some_rules(rng, 7, columns, 81)
        run_adjust(capi, x, dtype, 1, 3, 1, g=g, stride_of=stride, xadj=xadj, adjncy=adjncy, states=states, **kw)
        run_adjust(capi, x, dtype, g=g, stride_of=stride, xadj=xadj, adjncy=adjncy, states=states, **some_rules(rng, 7, columns, 0, 9, 2))
    g.free()


def test_adjust_wants_the_graphs_device(capi):
    xadj, adjncy = np.array([0, 1, 2], np.uint32), np.array([1, 0], np.uint32)
    g = capi.Graph.upload(xadj, adjncy, None)
    x = Matrix(capi, np.zeros((1, 2)), "f32")
    rules = capi.LogitsRules(graph=g, states=dev(capi, [0], np.uint32))
    capi.logits_adjust(x, capi.F32, 1, 2, rules, x)
    assert x.read()[0].tolist() == [-INF, 0.0]
    g.free()


# ------------------------------------------------------------------------------------------------ draw
def run_draw(capi, orc, x, dtype, pad=0, lead=0, t=None, top_k=None, top_p=None, min_p=None, u=None, seed=0, first=0, step=0, stride=1,
             workspace=False):
    rows, columns = x.shape
    m = Matrix(capi, x, dtype, pad, lead)
    rules = capi.DrawRules(temperature=dev(capi, t, np.float32), top_k=dev(capi, top_k, np.uint32), top_p=dev(capi, top_p, np.float32),
                           min_p=dev(capi, min_p, np.float32))
    tokens = dev(capi, np.full(rows * stride + 1, 777), np.uint32)
    logprobs, kept = dev(capi, np.full(rows + 1, 5.0), np.float32), dev(capi, np.full(rows + 1, 777), np.uint32)
    need = capi.logits_draw_workspace(code(capi, dtype), rows, columns)
    results = []
    for ws in ([None, dev(capi, np.full(need + 16, 255), np.uint8)] if workspace else [None]):  # nothing need be in it
        capi.logits_draw(m, code(capi, dtype), rows, columns, rules, tokens, uniforms=dev(capi, u, np.float64), seed=seed, first_walker=first,
                         step=step, logprobs=logprobs, kept=kept, row_stride=m.stride, tokens_stride=stride, workspace=ws)
        capi.synchronize()
        assert ws is None or (ws.to_host()[need:] == 255).all()
        results.append((tokens.to_host(), logprobs.to_host(), kept.to_host()))
    for tok, lp, kp in results:
        assert (tok[rows * stride:] == 777).all() and lp[rows] == 5.0 and kp[rows] == 777
        if stride > 1:
            assert (tok[:rows * stride].reshape(rows, stride)[:, 1:] == 777).all()
        for r in range(rows):
            uu = float(u[r]) if u is not None else so.philox_uniform(orc, seed, first + r, step)
            want = so.draw(m.values[r], 1.0 if t is None else float(np.float32(t[r])), 0 if top_k is None else int(top_k[r]),
                           1.0 if top_p is None else float(np.float32(top_p[r])), 0.0 if min_p is None else float(np.float32(min_p[r])), uu)
            got = int(tok[r * stride])
            assert (got, int(kp[r])) == (INVALID if want[0] is None else want[0], want[2]), (r, got, kp[r], want)
            # one rounding to fp32 of a number that is off by the weights' units (below 2^-40 of the mass)
            assert lp[r] == want[1] or abs(lp[r] - want[1]) <= 2.0 ** -24 * abs(want[1]) + 1e-9, (r, lp[r], want)
    m.read()
    return results[0]


SIZES = [(3, 1), (2, 2), (4, 63), (4, 1000), (3, 2048), (3, 2049), (2, 8191), (2, 40007), (1, 140001)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,columns", SIZES)
def test_draw_follows_its_definition(capi, orc, dtype, rows, columns):
    rng = np.random.default_rng(columns)
    x = rng.normal(0, 3, (rows, columns)).astype(np.float32)
    for n, (t, k, p, m) in enumerate([(1, 0, 1, 0), (0.7, 0, 0.9, 0), (1.3, 50, 1, 0), (0.8, 40, 0.95, 0), (1, 0, 1, 0.02), (2, 0, 0.99, 0.01),
                                      (0, 0, 1, 0), (1, 3000, 0.8, 0), (5, 2500, 1, 0), (0.05, 0, 0.5, 0.5), (1e30, 0, 0.3, 0), (3, 7000, 0.999, 1e-4)]):
        full = lambda v: np.full(rows, v)  # noqa: E731
        run_draw(capi, orc, x, dtype, pad=n % 4, lead=n % 3, t=full(t), top_k=full(k), top_p=full(p), min_p=full(m), u=rng.random(rows), workspace=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("columns", [5, 3000, 70001])
def test_draw_from_rows_of_equal_and_repeated_values(capi, orc, dtype, columns):
    rng = np.random.default_rng(columns + 1)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    rows = [np.zeros(columns), np.full(columns, low), np.where(np.arange(columns) % 3 == 0, 1.0, -1.0), rng.integers(-2, 3, columns) * 0.5,
            np.where(np.arange(columns) == columns - 1, 4.0, low), np.where(rng.random(columns) < 0.5, low, 2.0), np.where(np.arange(columns) % 2 == 0, -0.0, 0.0)]
    x = np.stack(rows).astype(np.float32)
    n = len(rows)
    for k, p, m in ((0, 1, 0), (0, 0.5, 0), (columns // 2 + 1, 1, 0), (3, 1, 0), (columns // 2, 0.7, 0), (0, 1, 1.0), (columns, 0.9, 0.3), (columns - 1, 1, 0)):
        for t in (1.0, 0.0):
            run_draw(capi, orc, x, dtype, t=np.full(n, t), top_k=np.full(n, k), top_p=np.full(n, p), min_p=np.full(n, m), u=rng.random(n), workspace=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("columns", [9, 5000])
def test_draw_from_rows_with_little_or_nothing_to_draw(capi, orc, dtype, columns):
    rng = np.random.default_rng(8)
    x = rng.normal(0, 3, (6, columns)).astype(np.float32)
    x[0] = -INF
    x[1] = np.nan
    x[2] = -INF
    x[2, columns // 2] = -7.0
    x[3, rng.random(columns) < 0.9] = -INF
    x[3, 1] = np.nan
    x[4, 3] = INF
    x[5, [2, 7]] = INF
    for t in (None, np.full(6, 0.0), np.full(6, np.nan), np.full(6, np.inf)):
        run_draw(capi, orc, x, dtype, t=t if t is None or not np.isnan(t[0]) else t, u=rng.random(6), workspace=True)
        run_draw(capi, orc, x, dtype, t=t, top_p=np.full(6, 0.9), top_k=np.full(6, 4), u=rng.random(6), workspace=True)


def test_draw_extremes_of_its_settings(capi, orc):
    rng = np.random.default_rng(9)
    x = rng.normal(0, 3, (12, 6000)).astype(np.float32)
    one = np.ones(12)
    for kw in (dict(u=0 * one), dict(u=one - 2.0 ** -53), dict(u=rng.random(12), top_p=0 * one), dict(u=rng.random(12), top_p=-one),
               dict(u=rng.random(12), top_p=np.nan * one), dict(u=rng.random(12), min_p=2 * one), dict(u=rng.random(12), min_p=np.nan * one),
               dict(u=rng.random(12), top_k=np.full(12, 4000000000)), dict(u=rng.random(12), top_k=one), dict(u=one - 2.0 ** -53, top_k=9 * one),
               dict(u=rng.random(12), t=-one), dict(u=rng.random(12), min_p=1e-30 * one), dict(u=rng.random(12), t=np.full(12, 1e-30)),
               dict(u=rng.random(12), min_p=np.full(12, 1e-25), t=np.full(12, 0.1), top_k=np.full(12, 5900))):
        run_draw(capi, orc, x, "f32", workspace=True, **kw)
        run_draw(capi, orc, x, "bf16", workspace=True, **kw)


def test_draw_by_philox_and_into_a_column(capi, orc):
    rng = np.random.default_rng(10)
    x = rng.normal(0, 3, (33, 700)).astype(np.float32)
    run_draw(capi, orc, x, "bf16", seed=(5 << 32) + 3, first=4294967290, step=17, stride=6)
    run_draw(capi, orc, x, "bf16", seed=1, first=0, step=0)
    from helpers import chi_square_p
    N, row = 20000, rng.normal(0, 1.5, 40).astype(np.float32)
    m = Matrix(capi, np.tile(row, (N, 1)), "f32")
    tokens = capi.DeviceArray(N, np.uint32)
    capi.logits_draw(m, capi.F32, N, 40, None, tokens, seed=99)
    p = np.exp(row.astype(np.float64))
    assert chi_square_p(np.bincount(tokens.to_host(), minlength=40), p / p.sum()) > 0.01


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_draw_of_many_rows(capi, orc, dtype):
    rng = np.random.default_rng(11)
    x = rng.normal(0, 2, (700, 3001)).astype(np.float32)
    x[rng.random(700) < 0.1] = -INF
    run_draw(capi, orc, x, dtype, pad=5, t=rng.uniform(0.3, 2, 700), top_k=rng.integers(0, 4000, 700), top_p=rng.uniform(0.3, 1.2, 700),
             min_p=rng.choice([0.0, 0.01], 700), u=rng.random(700), workspace=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("columns", [700, 5000, 40007])
def test_draw_by_a_min_p_above_one_leaves_the_first_entry(capi, orc, dtype, columns):
    rng = np.random.default_rng(columns)
    x = rng.integers(-3, 4, (4, columns)).astype(np.float32)  # many are as large as the largest
    for m in (1.0, 1.5):
        for p in (1.0, 0.9):
            run_draw(capi, orc, x, dtype, min_p=np.full(4, m), top_p=np.full(4, p), u=rng.random(4))


@pytest.mark.parametrize("dtype,columns", [("f32", 33001), ("f16", 20611), ("bf16", 20611)])
def test_draw_of_many_long_rows(capi, orc, dtype, columns):
    # more rows than CUs, some of which most entries are missing from, some to be drawn from few entries, some from all
    rng = np.random.default_rng(columns)
    n = 270
    x = rng.normal(0, 2, (n, columns)).astype(np.float32)
    x[::5][rng.random(x[::5].shape) < 0.995] = -INF
    x[1::9, 3000:] = -INF  # as full as can be where the kernel looks first, empty behind
    x[2::9, :3000] = -INF
    x[7] = -INF
    run_draw(capi, orc, x, dtype, pad=1, t=rng.choice([0.0, 0.4, 1.0, 2.0], n), top_k=rng.choice([0, 0, 20, 200, 700], n),
             top_p=rng.choice([1.0, 0.9, 0.5], n), min_p=rng.choice([0.0, 0.0, 0.02], n), u=rng.random(n))


@pytest.mark.parametrize("rows,columns", [(1, 131072), (61, 40011), (64, 33000)])
def test_draw_of_a_few_long_rows_with_a_workspace(capi, orc, rows, columns):
    assert capi.logits_draw_workspace(capi.F32, rows, columns) > 0 and capi.logits_draw_workspace(capi.F32, 65, columns) == 0
    assert capi.logits_draw_workspace(capi.BF16, rows, columns) == 0 and capi.logits_draw_workspace(capi.F32, rows, 32768) == 0
    rng = np.random.default_rng(columns)
    for n in range(3):
        x = rng.normal(0, 3, (rows, columns)).astype(np.float32)
        x[3::8] = rng.integers(-9, 10, x[3::8].shape)  # bins of one value, more than a list holds
        x[4::8] = np.where(rng.random(x[4::8].shape) < 0.97, -INF, x[4::8])
        x[5::8] = np.round(x[5::8] * 64) / 64
        x[6::8, : columns // 2] = -INF
        x[7::16] *= np.float32(1e-6)
        if rows > 9:
            x[9] = -INF
        k = rng.choice([0, 0, 0, 1, 50, 128, 129, 3000], rows)
        run_draw(capi, orc, x, "f32", pad=n, lead=n, t=rng.choice([0.0, 0.3, 1.0, 2.0, 50.0], rows, p=[0.1, 0.2, 0.4, 0.2, 0.1]), top_k=k if n else 0 * k,
                 top_p=rng.choice([1.0, 0.97, 0.6, 1e-6, 0.0], rows), min_p=rng.choice([0.0, 0.0, 0.02, 0.5, 1e-12], rows),
                 u=rng.choice([0.0, 1 - 2.0 ** -53], rows) if n == 2 else rng.random(rows), workspace=True)


def test_draw_of_more_rows_than_a_launch_has(capi):
    rows = (1 << 21) + 5
    x = np.random.default_rng(13).normal(0, 2, (rows, 2)).astype(np.float16)
    m, tokens, kept = dev(capi, x, np.float16), capi.DeviceArray(rows, np.uint32), capi.DeviceArray(rows, np.uint32)
    capi.logits_draw(m, capi.F16, rows, 2, capi.DrawRules(temperature=dev(capi, np.zeros(rows), np.float32)), tokens, kept=kept)
    assert np.array_equal(tokens.to_host(), (x[:, 1] > x[:, 0]).astype(np.uint32)) and (kept.to_host() == 1).all()
    capi.logits_draw(m, capi.F16, rows, 2, None, tokens, seed=5, first_walker=7)
    last, end = dev(capi, x[-9:], np.float16), capi.DeviceArray(9, np.uint32)
    capi.logits_draw(last, capi.F16, 9, 2, None, end, seed=5, first_walker=7 + rows - 9)
    assert np.array_equal(tokens.to_host()[-9:], end.to_host())


# ------------------------------------------------------------------------------------------------ route
def run_route(capi, x, dtype, k, pad=0, lead=0, counts=True, **kw):
    rows, E = x.shape
    m = Matrix(capi, x, dtype, pad, lead)
    names = dict(sigmoid="sigmoid", groups="groups", kept="groups_kept", top2="group_top2", renormalise="renormalise", scale="scale")
    rules = capi.RouteRules(k, bias=dev(capi, kw.get("bias"), np.float32), **{names[a]: b for a, b in kw.items() if a in names})
    ids, w = dev(capi, np.full(rows * k + 1, 777), np.uint32), dev(capi, np.full(rows * k + 1, 5.0), np.float32)
    c = dev(capi, np.full(E + 1, 777), np.uint32) if counts else None
    capi.route_topk(m, code(capi, dtype), rows, E, rules, ids, w, counts=c, row_stride=m.stride)
    capi.synchronize()
    want_ids, want_w, want_c = so.route(m.values, k, **kw)
    gi, gw = ids.to_host(), w.to_host()
    assert gi[rows * k] == 777 and gw[rows * k] == 5.0
    assert np.array_equal(gi[:-1].reshape(rows, k), want_ids)
    # scores in fp64, one rounding to fp32
    assert (np.abs(gw[:-1].reshape(rows, k) - want_w) <= np.abs(want_w) * (2.0 ** -24 + 1e-12) + 1e-45).all()
    if counts:
        assert np.array_equal(c.to_host()[:E], want_c) and c.to_host()[E] == 777
    # the gradient, into rows of another stride
    dw = np.random.default_rng(E).normal(size=(rows, k)).astype(np.float32)
    dx = Matrix(capi, np.full((rows, E), 9.0), dtype, (pad * 3) % 5, lead)
    capi.route_topk_backward(m, code(capi, dtype), rows, E, rules, ids, dev(capi, dw, np.float32), dx, row_stride=m.stride, dlogits_stride=dx.stride)
    capi.synchronize()
    want = so.route_backward(m.values, want_ids, dw, kw.get("sigmoid", False), kw.get("renormalise", True), kw.get("scale", 1.0))
    # fp32: exponentials to 2 units of 2^-23 and of differences that are off by 2^-24 of the logits' size, sums over up to 1,024 experts
    # and 64 chosen (13 + 7 additions deep at most, here taken as 24), products
    span = np.where(np.isfinite(m.values), np.abs(m.values), 0).max(initial=0.0)
    size = np.abs(kw.get("scale", 1.0) * dw).sum(1, keepdims=True)
    s = so.scores(m.values, kw.get("sigmoid", False))
    chosen = np.zeros((rows, E))
    for r in range(rows):
        ok = want_ids[r] < E
        chosen[r, want_ids[r][ok].astype(int)] = 1.0
    reach = np.maximum(chosen, s if not kw.get("sigmoid", False) else 0.0) * size
    near(dx.read(), want, reach * (40 + 2 * min(span, 200.0)) * 2.0 ** -24 + 1e-37, dtype)
    return want_ids


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,E,k", [(1, 1, 1), (5, 8, 2), (3, 64, 64), (9, 100, 6), (130, 65, 3), (7, 256, 8), (7, 203, 14), (5, 203, 13), (6, 203, 12), (3, 256, 16), (4, 500, 16), (3, 1024, 33)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_follows_its_definition(capi, dtype, rows, E, k, sigmoid):
    rng = np.random.default_rng(E * 7 + k)
    x = rng.normal(0, 2, (rows, E)).astype(np.float32)
    bias = rng.uniform(-0.2, 0.2, E).astype(np.float32)
    for n, (b, renorm, scale) in enumerate([(None, True, 1.0), (None, False, 1.0), (bias, True, 2.5), (bias, False, -0.5)]):
        run_route(capi, x, dtype, k, pad=n, lead=n % 2, counts=n != 1, sigmoid=sigmoid, bias=b, renormalise=renorm, scale=scale)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups,kept,k", [(256, 8, 4, 8), (64, 64, 5, 5), (60, 4, 1, 15), (96, 2, 2, 7), (1000, 50, 3, 20), (66, 3, 2, 44)])
def test_route_by_groups(capi, sigmoid, E, groups, kept, k):
    rng = np.random.default_rng(E + groups)
    x = rng.normal(0, 2, (37, E)).astype(np.float32)
    x[3, : E // groups] = -INF
    x[4, E // groups:] = -INF
    bias = rng.uniform(-0.2, 0.2, E).astype(np.float32)
    for top2 in (False, True):
        for b in (None, bias):
            run_route(capi, x, "bf16", k, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=top2)
            run_route(capi, x, "f32", k, pad=3, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=top2, renormalise=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_with_ties_closed_experts_and_extremes(capi, dtype, sigmoid):
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    x = np.zeros((9, 70), np.float32)
    x[1, 10:20] = 1.0
    x[2] = -INF
    x[3] = np.nan
    x[4, 3:] = -INF
    x[5] = low
    x[6, 5], x[6, 6] = INF, np.nan
    x[7] = -200.0
    x[7, 69] = -201.0
    x[8] = np.arange(70) % 7
    for renorm in (True, False):
        ids = run_route(capi, x, dtype, 6, sigmoid=sigmoid, renormalise=renorm)
        assert ids[0].tolist() == [0, 1, 2, 3, 4, 5] and ids[2].tolist() == [INVALID] * 6 and ids[4].tolist() == [0, 1, 2] + [INVALID] * 3
        run_route(capi, x, dtype, 6, sigmoid=sigmoid, renormalise=renorm, bias=np.zeros(70, np.float32))


@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_of_equal_groups_and_equal_choices(capi, sigmoid):
    # experts whose scores and biases differ in different last bits, groups that are worth the same, rows of one value
    x = np.zeros((40, 256), np.float32)
    x[1:20] = np.float32(2.0) + np.random.default_rng(3).integers(-2, 3, (19, 256)) * np.float32(2.0 ** -22)
    x[20:] = np.random.default_rng(4).integers(-3, 4, (20, 256))
    bias = (np.random.default_rng(5).integers(-2, 3, 256) * 2.0 ** -24).astype(np.float32)
    for top2 in (False, True):
        for b in (None, bias, np.zeros(256, np.float32)):
            for groups, kept, k in ((8, 3, 7), (1, 1, 16), (16, 5, 16), (32, 20, 9), (8, 4, 33)):
                run_route(capi, x, "f32", k, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=top2)
                run_route(capi, x[:, :96], "bf16", min(k, 15), sigmoid=sigmoid, bias=None if b is None else b[:96], groups=groups, kept=max(kept, -(-min(k, 15) // (96 // groups))), top2=top2, renormalise=False)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups,kept,k", [(24, 1, 1, 5), (256, 8, 3, 8), (256, 32, 9, 8), (600, 1, 1, 20)])
def test_route_by_biases_that_are_no_finite_numbers(capi, sigmoid, E, groups, kept, k):
    # -inf and NaN close an expert, +inf puts it first
    rng = np.random.default_rng(E + groups)
    x = rng.normal(0, 2, (19, E)).astype(np.float32)
    bias = rng.uniform(-0.2, 0.2, E).astype(np.float32)
    for odd in ((-INF,), (np.nan,), (INF,), (-INF, np.nan, INF)):
        b = bias.copy()
        b[rng.permutation(E)[: E // 3]] = np.resize(np.array(odd, np.float32), E // 3)
        for top2 in (False, True):
            run_route(capi, x, "f32", k, sigmoid=sigmoid, bias=b, groups=groups, kept=kept, top2=top2)


def test_route_of_a_long_batch(capi):
    rng = np.random.default_rng(12)
    run_route(capi, rng.normal(0, 2, (20011, 32)).astype(np.float32), "bf16", 4)


def test_route_without_rows_clears_the_counts(capi):
    c = dev(capi, np.full(9, 777), np.uint32)
    capi.route_topk(None, capi.F32, 0, 8, capi.RouteRules(2), None, None, counts=c)
    capi.synchronize()
    assert c.to_host().tolist() == [0] * 8 + [777]


def test_route_backward_passes_over_ids_that_are_no_experts_and_adds_equal_ones(capi):
    x = Matrix(capi, np.array([[0.5, -1.0, 2.0, 0.0]]), "f32")
    ids = np.array([[2, 9, 2]], np.uint32)
    dw = np.array([[1.0, 5.0, 0.25]], np.float32)
    dx = Matrix(capi, np.zeros((1, 4)), "f32")
    capi.route_topk_backward(x, capi.F32, 1, 4, capi.RouteRules(3, sigmoid=True, renormalise=False), dev(capi, ids, np.uint32), dev(capi, dw, np.float32), dx)
    s = 1 / (1 + np.exp(-2.0))
    near(dx.read(), np.array([[0, 0, 1.25 * s * (1 - s), 0]]), np.full((1, 4), 1e-6), "f32")


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def test_walk_by_a_models_scores(capi, orc):
    """Paths drawn step by step: the graph says where a walker may go, what it has visited counts against itself."""
    rng = np.random.default_rng(13)
    xadj, adjncy = orc.rmat_csr(10, 8, 3)
    V, N, steps, seed = 1024, 50, 6, 21
    g = capi.Graph.upload(xadj, adjncy, None)
    paths = np.full((N, steps + 1), INVALID, np.uint32)
    paths[:, 0] = rng.integers(0, V, N)
    d_paths = dev(capi, paths, np.uint32)
    rep, presence, frequency = np.full(N, 1.2, np.float32), np.full(N, 0.4, np.float32), np.full(N, 0.1, np.float32)
    t, p = np.full(N, 0.9, np.float32), np.full(N, 0.95, np.float32)

    class Column:
        def __init__(self, at):
            self.ptr = d_paths.ptr.value + 4 * at

    draw = capi.DrawRules(temperature=dev(capi, t, np.float32), top_p=dev(capi, p, np.float32))
    scores = [rng.normal(0, 2, (N, V)).astype(np.float32) for _ in range(steps)]
    device = [Matrix(capi, s, "bf16") for s in scores]
    arrays = [dev(capi, a, np.float32) for a in (rep, presence, frequency)]
    ready = Matrix(capi, np.zeros((N, V)), "bf16")
    for i in range(steps):
        rules = capi.LogitsRules(history=d_paths, history_columns=steps + 1, repetition=arrays[0], presence=arrays[1], frequency=arrays[2],
                                 graph=g, states=Column(i), states_stride=steps + 1)
        capi.logits_adjust(device[i], capi.BF16, N, V, rules, ready)
        capi.logits_draw(ready, capi.BF16, N, V, draw, Column(i + 1), seed=seed, step=i, tokens_stride=steps + 1)
    capi.synchronize()
    got = d_paths.to_host((N, steps + 1))
    for i in range(steps):
        # bf16 of a sum that may be rounded either way in fp32: the oracle's next step starts from the GPU's path so far
        want, error = so.adjust(device[i].values, history=np.where(np.arange(steps + 1) <= i, got, INVALID).astype(np.uint32), rep=rep,
                                presence=presence, frequency=frequency, xadj=xadj, adjncy=adjncy, states=got[:, i])
        _, rounded = so.to_bits(want.astype(np.float32), "bf16")
        for r in range(N):
            tok = so.draw(rounded[r], float(t[r]), 0, float(p[r]), 0.0, so.philox_uniform(orc, seed, r, i))[0]
            assert got[r, i + 1] == (INVALID if tok is None else tok)
            if tok is not None:
                assert tok in adjncy[xadj[got[r, i]]:xadj[got[r, i] + 1]]
    assert (got[:, 1] != INVALID).sum() > N // 4
    g.free()


class Hip:
    """Streams and graphs of the HIP runtime that the library runs on."""

    def __init__(self):
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
        self.lib = ctypes.CDLL(path)

    def __getattr__(self, name):
        f = getattr(self.lib, name)

        def call(*args):
            assert f(*args) == 0, name
        return call

    def stream(self):
        s = ctypes.c_void_p()
        self.hipStreamCreateWithFlags(ctypes.byref(s), 1)  # of its own: does not wait for the null stream
        return s


@pytest.mark.parametrize("columns", [5003, 40003])  # a workgroup a row, and rows in parts
def test_scores_on_a_stream_and_in_a_graph(capi, columns):
    rng = np.random.default_rng(14)
    rows, E = 24, 100
    hip = Hip()
    x, r_in = Matrix(capi, rng.normal(0, 3, (rows, columns)), "f32"), Matrix(capi, rng.normal(0, 2, (rows, E)), "f32")
    rules = capi.LogitsRules(history=dev(capi, rng.integers(0, columns, (rows, 90)), np.uint32), history_columns=90,
                             repetition=dev(capi, np.full(rows, 1.3), np.float32), presence=dev(capi, np.full(rows, 0.5), np.float32))
    draw = capi.DrawRules(top_p=dev(capi, np.full(rows, 0.8), np.float32))
    route = capi.RouteRules(5, sigmoid=True, bias=dev(capi, rng.uniform(-0.1, 0.1, E), np.float32))
    u = dev(capi, rng.random(rows), np.float64)
    need = capi.logits_draw_workspace(capi.F32, rows, columns)

    def outputs():
        z = lambda n, d: capi.DeviceArray.from_host(np.zeros(n, d))  # noqa: E731
        return dict(y=z(rows * columns, np.float32), tok=z(rows, np.uint32), lp=z(rows, np.float32), kept=z(rows, np.uint32), ids=z(rows * 5, np.uint32),
                    w=z(rows * 5, np.float32), counts=z(E, np.uint32), dx=z(rows * E, np.float32), ws=z(max(need, 16), np.uint8))

    def step(o, s):
        capi.logits_adjust(x, capi.F32, rows, columns, rules, o["y"], stream=s)
        capi.logits_draw(o["y"], capi.F32, rows, columns, draw, o["tok"], uniforms=u, logprobs=o["lp"], kept=o["kept"], workspace=o["ws"], stream=s)
        capi.route_topk(r_in, capi.F32, rows, E, route, o["ids"], o["w"], counts=o["counts"], stream=s)
        capi.route_topk_backward(r_in, capi.F32, rows, E, route, o["ids"], o["w"], o["dx"], stream=s)

    def same(a, b):
        for name in a:
            if name != "ws":
                assert np.array_equal(a[name].to_host(), b[name].to_host()), name

    eager, other, captured, again = outputs(), outputs(), outputs(), outputs()
    capi.synchronize()
    step(eager, None)
    side, side2 = hip.stream(), hip.stream()
    step(other, side)
    capi.synchronize()
    same(eager, other)
    graphs = []
    for o in (captured, again):  # each with a workspace of its own
        graph, ready = ctypes.c_void_p(), ctypes.c_void_p()
        hip.hipStreamBeginCapture(side, 0)
        step(o, side)
        hip.hipStreamEndCapture(side, ctypes.byref(graph))
        hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0))
        graphs.append((graph, ready))
    for n in range(4):
        fresh = rng.normal(0, 3, rows * columns).astype(np.float32)
        hip.hipMemcpy(x.dev.ptr, fresh.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(fresh.nbytes), 1)
        capi.synchronize()
        hip.hipGraphLaunch(graphs[0][1], side)
        hip.hipGraphLaunch(graphs[1][1], side2)  # at the same time
        step(eager, None)
        capi.synchronize()
        same(eager, captured)
        same(eager, again)
    for graph, ready in graphs:
        hip.hipGraphExecDestroy(ready)
        hip.hipGraphDestroy(graph)
    for s in (side, side2):
        hip.hipStreamDestroy(s)


def test_scores_calls_allocate_nothing(capi):
    x = Matrix(capi, np.zeros((300, 20000)), "f32")
    tokens, ids, w = capi.DeviceArray(300, np.uint32), capi.DeviceArray(600, np.uint32), capi.DeviceArray(600, np.float32)
    need = capi.logits_draw_workspace(capi.F32, 300, 20000)
    ws = capi.DeviceArray(max(need, 16), np.uint8)

    def all_calls():
        capi.logits_adjust(x, capi.F32, 300, 20000, None, x)
        capi.logits_draw(x, capi.F32, 300, 20000, None, tokens, seed=1, workspace=ws)
        capi.route_topk(x, capi.F32, 300, 64, capi.RouteRules(2), ids, w, row_stride=20000)
        capi.synchronize()

    all_calls()
    before, _ = capi.mem_info()
    for _ in range(3):
        all_calls()
    assert capi.mem_info()[0] == before
