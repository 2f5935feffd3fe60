"""Choices from rows of a model's scores, sized as their users size them, for timing and checking each operator by itself.

Models of sequences are trained on the walks and samples that the library draws; what such a model answers with is a row of
scores per walker, over the vertices (or tokens) that may come next or over the experts that may work on it.

  adjust          a row of logits made ready for the draw: repeated vertices made less likely, biases, and what the grammar (a table
                  of bit masks by state, or a graph: the neighbours of the vertex a walker stands on) does not allow taken out
  draw            one entry of every row by chance: temperature, top-k, top-p, min-p
  route           the k best experts of every row with their weights: softmax or sigmoid scores, a bias for balance, groups
  route_backward  the gradient of the weights with respect to the logits

`own` false computes them with elementary torch operations, `own` true through skywalker_amd.capi.  Where a whole number hangs on
a comparison (the entry drawn, the experts chosen) the plain form computes in 64 bits.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST_ENTRIES = 1 << 28  # of a row matrix


def _adjust(name, rows, columns, dtype, history=0, biases=0, masks=0, graph=False, pad=0):
    return dict(name=name, kind="adjust", rows=rows, columns=columns, dtype=dtype, history=history, biases=biases, masks=masks,
                graph=graph, pad=pad)


def _draw(name, rows, columns, dtype, temperature, top_k, top_p, min_p, allowed=1.0, pad=0):
    return dict(name=name, kind="draw", rows=rows, columns=columns, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, allowed=allowed, pad=pad)


def _route(name, kind, rows, experts, dtype, k, scores, bias=False, groups=1, groups_kept=1, group_top2=False, renormalise=True,
           scale=1.0):
    return dict(name=name, kind=kind, rows=rows, experts=experts, dtype=dtype, k=k, scores=scores, bias=bias, groups=groups,
                groups_kept=groups_kept, group_top2=group_top2, renormalise=renormalise, scale=scale)


def listed():
    return [
        # one walker of a small graph (c1: 65,536 vertices, walks of 80 steps): a step is all launches and waits
        _adjust("adjust_one", 1, 65536, "bf16", history=81),
        # a serving batch: long histories, a list of biases each, grammar states with their masks; no size a round number
        _adjust("adjust_grammar", 61, 100003, "bf16", history=2047, biases=300, masks=32, pad=5),
        # c1's 4,096 walkers, each held to the edges of the graph, repeated vertices penalised
        _adjust("adjust_graph", 4096, 65536, "f16", history=81, graph=True),
        # the draw that follows adjust_one, by the usual filters
        _draw("draw_one", 1, 65536, "bf16", 0.8, 50, 0.95, 0.0),
        # an ordinary serving batch by probability mass
        _draw("draw_batch", 256, 131072, "bf16", 0.7, 0, 0.9, 0.0),
        # scores in fp32, rows padded, every filter at once, another setting in each row (some greedy, some rows with nothing allowed)
        _draw("draw_mixed", 40, 100003, "f32", -1.0, 40, 0.9, 0.05, pad=3),
        # the draw of 4,096 walkers from what adjust_graph leaves: a few neighbours of 65,536 vertices
        _draw("draw_walkers", 4096, 65536, "f16", 1.0, 0, 1.0, 0.0, allowed=0.0003),
        # routing while decoding: a handful of tokens
        _route("route_decode", "route", 8, 64, "bf16", 2, "softmax"),
        # routing of a long batch: sigmoid scores, a bias for balance, 4 of 8 groups by their two best
        _route("route_batch", "route", 32768, 256, "bf16", 8, "sigmoid", bias=True, groups=8, groups_kept=4, group_top2=True, scale=2.5),
        # ragged: experts that do not fill wavefronts, weights not renormalised
        _route("route_ragged", "route", 10007, 100, "f32", 6, "softmax", renormalise=False),
        # their gradients: only the chosen entries; every entry of a long batch
        _route("route_backward_small", "route_backward", 1024, 64, "bf16", 2, "softmax"),
        _route("route_backward_dense", "route_backward", 32768, 256, "f32", 8, "softmax", bias=True, renormalise=False),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["adjust", "draw", "route", "route_backward"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind in ("adjust", "draw"):
        columns = _log(rng, 1000, 200000)
        rows = _log(rng, 1, max(1, min(2000, (1 << 26) // columns)))
        pad = rng.choice([0, 0, 1, 3, 8, 64])
        if kind == "adjust":
            grammar = rng.choice(["none", "masks", "graph"])
            return _adjust(None, rows, columns, dtype, history=rng.choice([0, _log(rng, 1, 8000)]), biases=rng.choice([0, _log(rng, 1, 500)]),
                           masks=_log(rng, 1, 64) if grammar == "masks" else 0, graph=grammar == "graph", pad=pad)
        return _draw(None, rows, columns, dtype, rng.choice([-1.0, 0.3, 0.7, 1.0, 1.5]), rng.choice([0, 0, _log(rng, 1, 1000)]),
                     rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), rng.choice([0.0, 0.0, 0.02, 0.1]), allowed=rng.choice([1.0, 1.0, 0.3, 0.001]),
                     pad=pad)
    groups = rng.choice([1, 1, 2, 4, 8])
    experts = groups * max(2, _log(rng, 8, 512) // groups)
    kept = rng.randint(max(1, groups // 2), groups)
    k = rng.randint(1, min(16, kept * (experts // groups)))
    return _route(None, kind, _log(rng, 1, min(65536, (1 << 23) // experts)), experts, dtype, k, rng.choice(["softmax", "sigmoid"]),
                  bias=rng.random() < 0.5, groups=groups, groups_kept=kept, group_top2=groups > 1 and rng.random() < 0.5,
                  renormalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))


# ------------------------------------------------------------------------------------------------ inputs
def _logits(gen, rows, columns, dtype, pad):
    """Scores as a model gives them: normal, a row's scale its own, a handful of entries that stand out; in rows of `columns + pad`."""
    x = torch.randn((rows, columns + pad), generator=gen, device="cuda")
    x *= 1.0 + 2.0 * torch.rand((rows, 1), generator=gen, device="cuda")
    best = torch.randint(0, columns, (rows, 8), generator=gen, device="cuda")
    x.scatter_add_(1, best, 6.0 * torch.rand((rows, 8), generator=gen, device="cuda"))
    return x.to(DTYPES[dtype])


def _csr(gen, vertices):
    """Rows of 0 to some hundred sorted neighbours, no two of a row alike."""
    degree = (torch.empty(vertices, device="cuda").log_normal_(2.0, 1.0, generator=gen)).long().clamp(max=vertices // 2)
    source = torch.repeat_interleave(torch.arange(vertices, device="cuda"), degree)
    target = torch.randint(0, vertices, (source.numel(),), generator=gen, device="cuda")
    edges = torch.unique(source * vertices + target)
    xadj = torch.zeros(vertices + 1, dtype=torch.int64, device="cuda")
    xadj[1:] = torch.cumsum(torch.bincount(edges // vertices, minlength=vertices), 0)
    return xadj, edges % vertices


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] in ("adjust", "draw"):
        rows, columns = case["rows"], case["columns"]
        s["logits"] = _logits(gen, rows, columns, case["dtype"], case["pad"])

    def uniform(shape, lo, hi):
        return lo + (hi - lo) * torch.rand(shape, generator=gen, device="cuda")

    def whole(shape, lo, hi):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    if case["kind"] == "adjust":
        if case["history"]:
            # visited vertices, some of them often; every row as long as its walk came, the slots after that as they were filled
            h = (columns * torch.rand((rows, case["history"]), generator=gen, device="cuda") ** 3).int().clamp(max=columns - 1)
            s["history_lengths"] = whole((rows,), 0, case["history"] + 1)
            h[torch.arange(case["history"], device="cuda")[None, :] >= s["history_lengths"][:, None]] = -1
            s["history"] = h
            s["history_first"] = (s["history_lengths"] * uniform((rows,), 0.0, 0.5)).int()
            s["repetition"], s["presence"], s["frequency"] = uniform((rows,), 1.0, 1.5), uniform((rows,), 0.0, 1.0), uniform((rows,), 0.0, 0.5)
        if case["biases"]:
            n = whole((rows,), 0, min(case["biases"], columns) + 1).long()
            row = torch.repeat_interleave(torch.arange(rows, device="cuda"), n)
            pairs = torch.unique(row * columns + torch.randint(0, columns, (row.numel(),), generator=gen, device="cuda"))
            s["bias_offsets"] = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
            s["bias_offsets"][1:] = torch.cumsum(torch.bincount(pairs // columns, minlength=rows), 0)
            s["bias_ids"], s["bias_values"] = (pairs % columns).int(), uniform((pairs.numel(),), -8.0, 8.0)
        if case["masks"]:
            words = (columns + 31) // 32
            dense = torch.rand((case["masks"], words, 32), generator=gen, device="cuda") < uniform((case["masks"], 1, 1), 0.0, 0.6) ** 2
            bits = (dense.long() << torch.arange(32, device="cuda")).sum(-1)
            s["allowed"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
            s["allowed_row"] = whole((rows,), -1, case["masks"])  # -1: a row that no grammar holds
        if case["graph"]:
            s["xadj"], s["adjncy"] = _csr(gen, columns)
            s["states"] = whole((rows,), 0, columns)
    elif case["kind"] == "draw":
        if case["allowed"] < 1.0:
            x = s["logits"]
            keep = torch.rand(x.shape, generator=gen, device="cuda") < case["allowed"] * uniform((rows, 1), 0.0, 2.0)
            s["logits"] = torch.where(keep, x, torch.full((), -math.inf, dtype=x.dtype, device="cuda"))
        s["uniforms"] = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
        if case["temperature"] < 0:  # every row its own settings
            s["temperature"] = uniform((rows,), 0.2, 1.5)
            s["temperature"][::7] = 0.0
            s["logits"][5::11] = -math.inf
            s["top_k"] = whole((rows,), 0, max(2, 2 * case["top_k"]))
            s["top_p"], s["min_p"] = uniform((rows,), case["top_p"] / 2, case["top_p"]), uniform((rows,), 0.0, case["min_p"])
        else:
            s["temperature"] = torch.full((rows,), case["temperature"], device="cuda")
            s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
            s["top_p"], s["min_p"] = torch.full((rows,), case["top_p"], device="cuda"), torch.full((rows,), case["min_p"], device="cuda")
    else:
        rows, experts, k = case["rows"], case["experts"], case["k"]
        s["logits"] = (2.0 * torch.randn((rows, experts), generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
        s["bias"] = uniform((experts,), -0.1, 0.1) if case["bias"] else None
        if case["kind"] == "route_backward":
            s["ids"] = _plain_route(s)["ids"]
            s["dweights"] = torch.randn((rows, k), generator=gen, device="cuda")
    return s


class _Buffer:
    """A torch tensor where capi takes one of its own arrays: anything with the address under `ptr`, and the size of a workspace."""

    def __init__(self, tensor):
        self.tensor, self.ptr, self.nbytes = tensor, ctypes.c_void_p(tensor.data_ptr()), tensor.nbytes


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    from skywalker_amd import capi
    s["capi"], s["dtype"] = capi, {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[case["dtype"]]

    def buffer(name):
        return _Buffer(s[name]) if s.get(name) is not None else None

    def empty(shape, dtype):
        return _Buffer(torch.empty(shape, dtype=dtype, device="cuda"))

    s["in"] = buffer("logits")
    rows = case["rows"]
    if case["kind"] == "adjust":
        if case["graph"]:
            s["g"] = capi.Graph.upload(s["xadj"].cpu().numpy(), s["adjncy"].cpu().numpy(), None)
        s["rules"] = capi.LogitsRules(
            history=buffer("history"), history_columns=case["history"], history_lengths=buffer("history_lengths"),
            history_first=buffer("history_first"), repetition=buffer("repetition"), presence=buffer("presence"), frequency=buffer("frequency"),
            bias_offsets=buffer("bias_offsets"), bias_ids=buffer("bias_ids"), bias_values=buffer("bias_values"),
            bias_count=s["bias_ids"].numel() if case["biases"] else 0,
            allowed=buffer("allowed"), allowed_rows=case["masks"], allowed_row=buffer("allowed_row"),
            graph=s.get("g"), states=buffer("states"))
        s["out"] = empty((rows, case["columns"]), DTYPES[case["dtype"]])
    elif case["kind"] == "draw":
        s["rules"] = capi.DrawRules(temperature=buffer("temperature"), top_k=buffer("top_k"), top_p=buffer("top_p"), min_p=buffer("min_p"))
        s["u"] = buffer("uniforms")
        s["tokens"], s["logprobs"], s["kept"] = empty(rows, torch.int32), empty(rows, torch.float32), empty(rows, torch.int32)
        n = capi.logits_draw_workspace(s["dtype"], rows, case["columns"])
        s["workspace"] = empty(n, torch.uint8) if n else None
    else:
        s["rules"] = capi.RouteRules(k=case["k"], sigmoid=case["scores"] == "sigmoid", bias=buffer("bias"), groups=case["groups"],
                                     groups_kept=case["groups_kept"], group_top2=case["group_top2"], renormalise=case["renormalise"],
                                     scale=case["scale"])
        if case["kind"] == "route":
            s["ids"], s["weights"] = empty((rows, case["k"]), torch.int32), empty((rows, case["k"]), torch.float32)
            s["counts"] = empty(case["experts"], torch.int32)
        else:
            s["ids_in"], s["dw"] = buffer("ids"), buffer("dweights")
            s["dlogits"] = empty((rows, case["experts"]), DTYPES[case["dtype"]])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_adjust(s):
    case = s["case"]
    rows, columns = case["rows"], case["columns"]
    x = s["logits"][:, :columns].float()
    if case["history"]:
        h, position = s["history"].long(), torch.arange(case["history"], device="cuda")[None, :]
        there = (position < s["history_lengths"][:, None]) & (h >= 0) & (h < columns)
        h = torch.where(there, h, torch.zeros_like(h))
        counted = there & (position >= s["history_first"][:, None])
        seen = torch.zeros((rows, columns), device="cuda").scatter_add_(1, h, there.float()) > 0
        count = torch.zeros((rows, columns), device="cuda").scatter_add_(1, h, counted.float())
        rep = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = torch.where(count > 0, x - (s["presence"][:, None] + s["frequency"][:, None] * count), x)
    if case["biases"]:
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), s["bias_offsets"].diff().long())
        x = x.index_put((row, s["bias_ids"].long()), s["bias_values"], accumulate=True)
    if case["masks"]:
        column = torch.arange(columns, device="cuda")
        state = s["allowed_row"].long()
        bits = ((s["allowed"][:, column // 32] >> (column % 32).int()) & 1).bool()
        x = torch.where(bits[state.clamp(min=0)] | (state < 0)[:, None], x, torch.full_like(x, -math.inf))
    if case["graph"]:
        state = s["states"].long()
        begin, degree = s["xadj"][state], s["xadj"][state + 1] - s["xadj"][state]
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), degree)
        first = torch.cumsum(degree, 0) - degree
        slot = torch.arange(row.numel(), device="cuda") - first[row] + begin[row]
        can = torch.zeros((rows, columns), dtype=torch.bool, device="cuda")
        can[row, s["adjncy"][slot]] = True
        x = torch.where(can, x, torch.full_like(x, -math.inf))
    return x.to(s["logits"].dtype)


def _plain_draw(s):
    case = s["case"]
    rows, columns = case["rows"], case["columns"]
    parts = []
    step = max(1, (1 << 26) // columns)
    for lo in range(0, rows, step):  # 64-bit copies of a part of the rows at a time
        part = slice(lo, min(rows, lo + step))
        x = s["logits"][part, :columns].float()
        x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).clamp(max=torch.finfo(torch.float32).max)
        z, order = torch.sort(x, dim=1, descending=True, stable=True)
        allowed = z > -math.inf
        t = s["temperature"][part, None].double()
        d = torch.where(allowed, z.double() - z[:, :1].double(), torch.full_like(z, -math.inf, dtype=torch.float64))
        w = torch.exp(d / torch.where(t > 0, t, torch.ones_like(t)))
        rank = torch.arange(columns, device="cuda")[None, :]
        top_k = s["top_k"][part, None]
        keep = allowed & ((top_k <= 0) | (rank < top_k))
        cum = torch.cumsum(torch.where(keep, w, torch.zeros_like(w)), 1)
        top_p = s["top_p"][part, None].double()
        keep &= (top_p >= 1) | (cum - w < top_p * cum[:, -1:]) | (rank == 0)
        keep &= (w >= s["min_p"][part, None].double()) | (rank == 0)
        keep &= (t > 0) | (rank == 0)
        kept = keep.sum(1)
        mass = torch.where(keep, w, torch.zeros_like(w))
        cum = torch.cumsum(mass, 1)
        at = (cum <= s["uniforms"][part, None] * cum[:, -1:]).sum(1)
        at = torch.minimum(at, kept - 1).clamp(min=0)[:, None]
        token = torch.where(kept > 0, torch.gather(order, 1, at)[:, 0], torch.full_like(kept, -1))
        logprob = torch.where(kept > 0, torch.log(torch.gather(w, 1, at)[:, 0] / cum[:, -1]), torch.full_like(cum[:, 0], -math.inf))
        parts.append((token.int(), logprob.float(), kept.int()))
    token, logprob, kept = [torch.cat(p) for p in zip(*parts)]
    return {"tokens": token, "logprobs": logprob, "kept": kept}


def _plain_scores(s):
    x = s["logits"].double()
    return torch.sigmoid(x) if s["case"]["scores"] == "sigmoid" else torch.softmax(x, 1)


def _plain_route(s):
    case = s["case"]
    rows, experts, groups, k = case["rows"], case["experts"], case["groups"], case["k"]
    score = _plain_scores(s)
    choice = score + s["bias"].double() if case["bias"] else score
    if groups > 1:
        by_group = choice.view(rows, groups, experts // groups)
        best = by_group.topk(min(2, experts // groups), dim=2).values
        of_group = best.sum(2) if case["group_top2"] else best[:, :, 0]
        _, order = torch.sort(of_group, dim=1, descending=True, stable=True)
        kept = torch.zeros((rows, groups), dtype=torch.bool, device="cuda").scatter_(1, order[:, :case["groups_kept"]], True)
        choice = torch.where(kept[:, :, None], by_group, torch.full_like(by_group, -math.inf)).view(rows, experts)
    _, order = torch.sort(choice, dim=1, descending=True, stable=True)
    ids = order[:, :k]
    w = torch.gather(score, 1, ids)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return {"ids": ids.int(), "weights": (w * case["scale"]).float(),
            "counts": torch.bincount(ids.reshape(-1), minlength=experts).int()}


def _plain_route_backward(s):
    case = s["case"]
    score, ids = _plain_scores(s).float(), s["ids"].long()
    chosen = torch.gather(score, 1, ids)
    g = s["dweights"] * case["scale"]
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True)
        g = (g - (g * chosen).sum(1, keepdim=True) / total) / total
    dscore = torch.zeros_like(score).scatter_add_(1, ids, g)
    if case["scores"] == "sigmoid":
        dx = dscore * score * (1 - score)
    else:
        dx = score * (dscore - (dscore * score).sum(1, keepdim=True))
    return dx.to(s["logits"].dtype)


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if not own:
        return {"adjust": _plain_adjust, "draw": _plain_draw, "route": _plain_route, "route_backward": _plain_route_backward}[kind](s)
    capi, rows = s["capi"], case["rows"]
    if kind == "adjust":
        capi.logits_adjust(s["in"], s["dtype"], rows, case["columns"], s["rules"], s["out"], row_stride=case["columns"] + case["pad"])
        return s["out"].tensor
    if kind == "draw":
        capi.logits_draw(s["in"], s["dtype"], rows, case["columns"], s["rules"], s["tokens"], uniforms=s["u"], logprobs=s["logprobs"],
                         kept=s["kept"], row_stride=case["columns"] + case["pad"], workspace=s["workspace"])
        return {"tokens": s["tokens"].tensor, "logprobs": s["logprobs"].tensor, "kept": s["kept"].tensor}
    if kind == "route":
        capi.route_topk(s["in"], s["dtype"], rows, case["experts"], s["rules"], s["ids"], s["weights"], counts=s["counts"])
        return {"ids": s["ids"].tensor, "weights": s["weights"].tensor, "counts": s["counts"].tensor}
    capi.route_topk_backward(s["in"], s["dtype"], rows, case["experts"], s["rules"], s["ids_in"], s["dw"], s["dlogits"])
    return s["dlogits"].tensor


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_adjust(case, a):
    rows, columns = case["rows"], case["columns"]
    out = a["logits"][:, :columns].astype(np.float64)
    for r in range(rows):
        x = out[r]
        if case["history"]:
            h = a["history"][r, :a["history_lengths"][r]]
            seen = np.unique(h)
            rep = float(a["repetition"][r])
            x[seen] = np.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
            tokens, counts = np.unique(h[a["history_first"][r]:], return_counts=True)
            x[tokens] -= float(a["presence"][r]) + float(a["frequency"][r]) * counts
        if case["biases"]:
            mine = slice(a["bias_offsets"][r], a["bias_offsets"][r + 1])
            np.add.at(x, a["bias_ids"][mine], a["bias_values"][mine].astype(np.float64))
        if case["masks"] and a["allowed_row"][r] >= 0:
            bits = np.unpackbits(a["allowed"][a["allowed_row"][r]].view(np.uint8), bitorder="little")[:columns]
            x[bits == 0] = -np.inf
        if case["graph"]:
            v = a["states"][r]
            gone = np.ones(columns, bool)
            gone[a["adjncy"][a["xadj"][v]:a["xadj"][v + 1]]] = False
            x[gone] = -np.inf
    return out


def _exact_draw(case, a):
    rows, columns = case["rows"], case["columns"]
    tokens, logprobs, kept = np.full(rows, -1, np.int32), np.full(rows, -np.inf), np.zeros(rows, np.int32)
    for r in range(rows):
        x = a["logits"][r, :columns].astype(np.float64)
        there = np.flatnonzero(x > -np.inf)
        if there.size == 0:
            continue
        order = there[np.argsort(-x[there], kind="stable")]
        z, t = x[order], float(a["temperature"][r])
        if t <= 0:
            tokens[r], logprobs[r], kept[r] = order[0], 0.0, 1
            continue
        w = np.exp((z - z[0]) / t)
        n = w.size
        if a["top_k"][r] > 0:
            n = min(n, int(a["top_k"][r]))
        cum = np.cumsum(w[:n])
        if a["top_p"][r] < 1:
            n = min(n, 1 + int(np.searchsorted(cum, float(a["top_p"][r]) * cum[-1])))
        n = max(1, min(n, int(np.count_nonzero(w >= float(a["min_p"][r])))))
        at = min(n - 1, int(np.searchsorted(cum[:n], a["uniforms"][r] * cum[n - 1], side="right")))
        tokens[r], logprobs[r], kept[r] = order[at], math.log(w[at] / cum[n - 1]) if w[at] > 0 else (z[at] - z[0]) / t - math.log(cum[n - 1]), n
    return {"tokens": tokens, "logprobs": logprobs, "kept": kept}


def _exact_scores(case, x):
    if case["scores"] == "sigmoid":
        return 1.0 / (1.0 + np.exp(-x))
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def _exact_route(case, a):
    rows, experts, groups, k = case["rows"], case["experts"], case["groups"], case["k"]
    score = _exact_scores(case, a["logits"].astype(np.float64))
    choice = score + (a["bias"].astype(np.float64) if case["bias"] else 0.0)
    if groups > 1:
        ranked = -np.sort(-choice.reshape(rows, groups, -1), axis=2)
        of_group = ranked[:, :, :2].sum(2) if case["group_top2"] else ranked[:, :, 0]
        out = np.argsort(-of_group, axis=1, kind="stable")[:, case["groups_kept"]:]
        closed = np.zeros((rows, groups), bool)
        np.put_along_axis(closed, out, True, 1)
        choice = np.where(np.repeat(closed, experts // groups, axis=1), -np.inf, choice)
    ids = np.argsort(-choice, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(score, ids, 1)
    if case["renormalise"]:
        w = w / w.sum(1, keepdims=True)
    return {"ids": ids.astype(np.int32), "weights": w * case["scale"], "counts": np.bincount(ids.ravel(), minlength=experts).astype(np.int32)}


def _exact_route_backward(case, a):
    score, ids, g = _exact_scores(case, a["logits"].astype(np.float64)), a["ids"].astype(np.int64), a["dweights"].astype(np.float64) * case["scale"]
    chosen = np.take_along_axis(score, ids, 1)
    out = np.zeros_like(score)
    if case["renormalise"]:
        share = chosen / chosen.sum(1, keepdims=True)
        away = share * (g - (g * share).sum(1, keepdims=True))
        np.put_along_axis(out, ids, away * (1.0 - chosen) if case["scores"] == "sigmoid" else away, 1)
    elif case["scores"] == "sigmoid":
        np.put_along_axis(out, ids, g * chosen * (1.0 - chosen), 1)
    else:
        np.put_along_axis(out, ids, g * chosen, 1)
        out -= score * (g * chosen).sum(1, keepdims=True)
    return out


def exact(case, seed):
    entries = case["rows"] * case.get("columns", case.get("experts", 0))
    if entries > (1 << 26 if case["kind"] != "draw" else 1 << 25):
        return None
    a = {}
    for name, value in _inputs(case, seed).items():
        if isinstance(value, torch.Tensor):
            a[name] = (value.float() if value.is_floating_point() and value.dtype != torch.float64 else value).cpu().numpy()
    return {"adjust": _exact_adjust, "draw": _exact_draw, "route": _exact_route, "route_backward": _exact_route_backward}[case["kind"]](case, a)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    rows, b = case["rows"], BYTES[case["dtype"]]
    if case["kind"] == "adjust":
        n = rows * case["columns"]
        # the mean row of _csr holds 11.7 neighbours; a mask lets 0.12 of a row through and one row in masks + 1 has none
        read = 12 * rows if case["graph"] else n * (0.12 + 0.88 / (case["masks"] + 1)) if case["masks"] else n
        total = read * b + n * b + rows * (case["history"] // 2 * 4 + 20)
        total += rows * case["biases"] * 4 + (min(rows, case["masks"]) * case["columns"] / 8 if case["masks"] else 0)
        return {"bytes": total + (rows * 12 * 4 if case["graph"] else 0), "flops": 0}
    if case["kind"] == "draw":
        n = rows * case["columns"]
        # a difference, a quotient, an exponential (16) and a sum for every entry that may be drawn
        return {"bytes": n * b + rows * 36, "flops": 19 * n * case["allowed"]}
    n, k = rows * case["experts"], case["k"]
    if case["kind"] == "route":
        return {"bytes": n * b + 8 * rows * k + 4 * case["experts"], "flops": 18 * n}
    return {"bytes": 2 * n * b + 8 * rows * k, "flops": 20 * n}
