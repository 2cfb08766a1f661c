"""Sparse rows of ids against dense matrices: the operators a memory layer or an embedding trains and serves with.

    lookup               out[r] = scale * sum over row r's ids of weight * table[id]
    lookup_grad          the gradients of that sum: to the table (by sorted ids) and to the weights
    winners              dense scores -> the k winning ids of every row with their weights
                         (softmax or sigmoid, a bias for balance, groups, renormalised weights)
    winners_grad         the gradient of the weights to the scores

`run` computes them in elementary torch operations, or by the calls a user makes of this package where `own` is set.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # an embedding read for the one token that a server decodes, scaled as a transformer scales its embedding
        dict(name="lookup_one_token", op="lookup", rows=1, row_len=1, ids=32768, dim=2048, table="bf16", out="bf16",
             weights=False, dist="zipf", pad=False, id_bits=64, scale=45.25),
        # the tokens of one training step in a large vocabulary; short sequences are padded with -1
        dict(name="lookup_tokens", op="lookup", rows=16384, row_len=1, ids=131072, dim=4096, table="bf16", out="bf16",
             weights=False, dist="zipf", pad=True, id_bits=64, scale=1.0),
        # sparse codes of 16 384 ids with 2 % active and payloads in [0,1), each decoded to a dense vector
        dict(name="lookup_codes_16k", op="lookup", rows=4096, row_len=328, ids=16384, dim=1024, table="bf16", out="bf16",
             weights=True, dist="distinct", pad=False, id_bits=32, scale=1.0),
        # ragged rows, some of them empty, of a 2048-wide code; an odd dimension in fp32
        dict(name="lookup_ragged_odd", op="lookup", rows=5003, row_len=-64, ids=2048, dim=1001, table="f32", out="f32",
             weights=False, dist="uniform", pad=False, id_bits=32, scale=0.5),
        # the table's gradient of a few tokens, as one short sequence brings
        dict(name="grad_few_tokens", op="lookup_grad", rows=37, row_len=1, ids=2048, dim=512, table="f32", grad="f16",
             weights=False, dist="zipf", pad=False, id_bits=64, scale=22.5),
        # the embedding's gradient of one training step: few ids hold many tokens, most ids hold none
        dict(name="grad_tokens", op="lookup_grad", rows=16384, row_len=1, ids=65536, dim=2048, table="bf16", grad="bf16",
             weights=False, dist="zipf", pad=True, id_bits=64, scale=1.0),
        # a memory layer's step: 40 of 2048 slots a row; gradients to the slots' values and to the weights
        dict(name="grad_codes", op="lookup_grad", rows=8192, row_len=40, ids=2048, dim=512, table="bf16", grad="bf16",
             weights=True, dist="distinct", pad=False, id_bits=32, scale=1.0),
        # one token routed to experts in groups
        dict(name="winners_one_token", op="winners", rows=1, ids=256, k=8, scores="f32", score="sigmoid", bias=True,
             groups=8, top_groups=4, group_top=2, renormalise=True, masked=0.0, scale=2.0),
        # the tokens of one training step routed to experts in groups
        dict(name="winners_grouped", op="winners", rows=16384, ids=256, k=8, scores="f32", score="sigmoid", bias=True,
             groups=8, top_groups=4, group_top=2, renormalise=True, masked=0.0, scale=2.0),
        # 40 winners of 2048 a row: dense activations made into sparse codes; some ids are masked out by -inf
        dict(name="winners_codes_2k", op="winners", rows=8192, ids=2048, k=40, scores="bf16", score="softmax", bias=False,
             groups=1, top_groups=1, group_top=1, renormalise=True, masked=0.1, scale=1.0),
        # the scores' gradient of a routed training step; every score takes part in the softmax
        dict(name="winners_grad_experts", op="winners_grad", rows=16384, ids=128, k=6, scores="f32", score="softmax",
             renormalise=False, masked=0.0, scale=1.0),
        # the scores' gradient of sparse codes of an odd width
        dict(name="winners_grad_codes", op="winners_grad", rows=4099, ids=2047, k=40, scores="bf16", score="sigmoid",
             renormalise=True, masked=0.1, scale=1.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup", "lookup_grad", "lookup_grad", "winners", "winners", "winners_grad"])
    if op in ("lookup", "lookup_grad"):
        kind = rng.choice(["tokens", "codes", "ragged"])
        dim = _log_int(rng, 64, 4096) | rng.choice([0, 0, 1])
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        if kind == "tokens":
            rows, row_len, ids, dist = _log_int(rng, 1, 16384), 1, _log_int(rng, 500, 65536), "zipf"
        elif kind == "codes":
            ids = _log_int(rng, 256, 16384)
            row_len = max(1, ids * rng.choice([1, 2, 2, 5]) // 100)
            rows, dist = _log_int(rng, 1, min(4096, 60_000_000 // ids)), "distinct"
        else:
            ids, row_len, rows, dist = _log_int(rng, 256, 16384), -_log_int(rng, 2, 200), _log_int(rng, 16, 4096), "uniform"
        elems = rows * max(1, abs(row_len) if row_len > 0 else -row_len // 2)
        if op == "lookup":
            dim = min(dim, max(64, 1_300_000_000 // elems))
        else:
            dim = min(dim, max(64, 160_000_000 // elems), max(64, 134_000_000 // ids))
        c = dict(op=op, rows=rows, row_len=row_len, ids=ids, dim=dim, table=rng.choice(["bf16", "f16", "f32"]),
                 weights=dist != "zipf" and rng.random() < 0.6, dist=dist, pad=dist == "zipf" and rng.random() < 0.5,
                 id_bits=rng.choice([32, 64]), scale=rng.choice([1.0, 0.5, math.sqrt(dim)]))
        if op == "lookup":
            c["out"] = rng.choice([c["table"], "f32"])
        else:
            c["grad"] = rng.choice([c["table"], "f32"])
        return c
    ids = _log_int(rng, 8, 4096)
    rows = _log_int(rng, 1, min(16384, 16_000_000 // ids))
    score = rng.choice(["softmax", "sigmoid"])
    c = dict(op=op, rows=rows, ids=ids, k=_log_int(rng, 1, max(1, min(64, ids // 4))), scores=rng.choice(["f32", "bf16", "f16"]),
             score=score, renormalise=rng.random() < 0.6, masked=rng.choice([0.0, 0.1, 0.5]), scale=rng.choice([1.0, 2.5]))
    if op == "winners":
        groups = rng.choice([1, 1, 4, 8]) if ids >= 32 else 1
        c["ids"] = ids = ids // groups * groups
        top = 1 if groups == 1 else rng.choice([groups // 2, groups - 1])
        c.update(bias=rng.random() < 0.5, groups=groups, top_groups=top, group_top=rng.choice([1, 2]))
        c["k"] = max(1, min(c["k"], ids // groups * top // 2))
    return c


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _rows(case, g):
    """ids (and offsets where rows are ragged) of a case."""
    n, m, v = case["rows"], case["row_len"], case["ids"]
    kind = torch.int64 if case["id_bits"] == 64 else torch.int32
    offsets = None
    if m < 0:
        lens = torch.randint(0, -m + 1, (n,), generator=g, device="cuda")
        offsets = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = lens.cumsum(0)
        ids = torch.randint(0, v, (int(offsets[-1]),), generator=g, device="cuda")
    elif case["dist"] == "distinct":
        ids = torch.rand(n, v, generator=g, device="cuda").topk(m, dim=1).indices.sort(dim=1).values
    else:
        # a token's chance falls with one over its rank, as words' do
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(v + 1)).floor().long() - 1).clamp(0, v - 1)
        if case["pad"]:
            # the last eighth of every 512 tokens is padding
            ids = torch.where(torch.arange(n, device="cuda") % 512 >= 448, -1, ids)
    return ids.to(kind), offsets


def _scores(case, g):
    s = torch.randn(case["rows"], case["ids"], generator=g, device="cuda") * 2
    if case["masked"]:
        s = torch.where(torch.rand(s.shape, generator=g, device="cuda") < case["masked"], float("-inf"), s)
    return s.to(_TYPES[case["scores"]])


def prepare(case, seed):
    g = _generator(seed)
    st = {"case": case}
    if case["op"] in ("lookup", "lookup_grad"):
        st["ids"], st["offsets"] = _rows(case, g)
        st["weights"] = torch.rand(st["ids"].shape, generator=g, device="cuda") if case["weights"] else None
        st["table"] = (torch.randn(case["ids"], case["dim"], generator=g, device="cuda") * 0.5).to(_TYPES[case["table"]])
        if case["op"] == "lookup_grad":
            st["grad"] = torch.randn(case["rows"], case["dim"], generator=g, device="cuda").to(_TYPES[case["grad"]])
    else:
        st["scores"] = _scores(case, g)
        if case["op"] == "winners":
            st["bias"] = torch.rand(case["ids"], generator=g, device="cuda") * 0.1 if case["bias"] else None
        else:
            # the ids that the forward pass chose: the k largest scores, ascending, -1 where the row has fewer
            top = st["scores"].float().topk(case["k"], dim=1)
            ids = torch.where(top.values > float("-inf"), top.indices, case["ids"]).sort(dim=1).values
            st["ids"] = torch.where(ids < case["ids"], ids, -1).int()
            st["grad"] = torch.randn(case["rows"], case["k"], generator=g, device="cuda")
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------


def _flat(st):
    """ids as indexes (what lies outside the table points at one row more) and the row of each."""
    c, ids = st["case"], st["ids"].long()
    n = ids.numel()
    if st["offsets"] is not None:
        row = torch.repeat_interleave(torch.arange(c["rows"], device=ids.device), st["offsets"].diff(), output_size=n)
    else:
        row = torch.arange(c["rows"], device=ids.device).repeat_interleave(n // c["rows"], output_size=n)
    ids = ids.reshape(-1)
    return torch.where((ids >= 0) & (ids < c["ids"]), ids, c["ids"]), row


def _plain_lookup(st):
    c = st["case"]
    ids, row = _flat(st)
    if c["row_len"] == 1:
        out = st["table"][ids.clamp(max=c["ids"] - 1)].float()
        if st["weights"] is not None:
            out = out * st["weights"].reshape(-1, 1)
        out = torch.where((ids < c["ids"])[:, None], out, 0.0)
    else:
        terms = st["table"][ids.clamp(max=c["ids"] - 1)].float()
        if st["weights"] is not None:
            terms *= st["weights"].reshape(-1, 1)
        if st["offsets"] is None:
            out = terms.view(c["rows"], c["row_len"], c["dim"]).sum(1)
        else:
            out = torch.zeros(c["rows"], c["dim"], device="cuda").index_add_(0, row, terms)
    return (out * c["scale"]).to(_TYPES[c["out"]])


def _plain_lookup_grad(st):
    c = st["case"]
    ids, row = _flat(st)
    terms = st["grad"][row].float()
    weighed = terms if st["weights"] is None else terms * st["weights"].reshape(-1, 1)
    table = torch.zeros(c["ids"] + 1, c["dim"], device="cuda").index_add_(0, ids, weighed)[:-1] * c["scale"]
    if st["weights"] is None:
        return {"table": table}
    of = (terms * st["table"][ids.clamp(max=c["ids"] - 1)].float()).sum(1) * c["scale"]
    return {"table": table, "weights": torch.where(ids < c["ids"], of, 0.0).view(st["ids"].shape)}


def _shares(x, live, score):
    """softmax over a row's live scores, or sigmoid."""
    if score == "sigmoid":
        return torch.where(live, 1 / (1 + torch.exp(-x)), 0.0)
    m = torch.where(live, x, float("-inf")).amax(1, keepdim=True)
    e = torch.where(live, torch.exp(torch.where(x == m, 0.0, x - m)), 0.0)
    return e / e.sum(1, keepdim=True).clamp(min=1e-300 if x.dtype == torch.float64 else 1e-37)


def _logits(x, score):
    """what a softmax over the winners gives the renormalised weights of: the scores, or the logarithms of their sigmoids."""
    return torch.clamp(x, max=0) - torch.log1p(torch.exp(-x.abs())) if score == "sigmoid" else x


def _plain_winners(st):
    c = st["case"]
    x = st["scores"].double()  # in 64 bits: which of two close keys is larger decides between ids
    live = x > float("-inf")
    share = _shares(x, live, c["score"])
    # without a bias and sums of two the order of the shares is that of the scores
    key = share if st["bias"] is None else share + st["bias"].double()
    key = torch.where(live, key if st["bias"] is not None or (c["groups"] > 1 and c["group_top"] > 1) else x, float("-inf"))
    if c["groups"] > 1:
        best = key.view(c["rows"], c["groups"], -1).sort(dim=2, descending=True).values
        of = best[:, :, 0]
        if c["group_top"] > 1 and best.shape[2] > 1:
            of = of + torch.where(best[:, :, 1] > float("-inf"), best[:, :, 1], 0.0)
        first = of.sort(dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        inside = torch.zeros_like(of, dtype=torch.bool).scatter(1, first, True)
        key = torch.where(inside.repeat_interleave(c["ids"] // c["groups"], dim=1), key, float("-inf"))
    order = key.sort(dim=1, descending=True, stable=True)
    ids = torch.where(order.values[:, : c["k"]] > float("-inf"), order.indices[:, : c["k"]], c["ids"]).sort(dim=1).values
    there = ids < c["ids"]
    at = ids.clamp(max=c["ids"] - 1)
    if c["renormalise"]:
        w = _shares(_logits(x.gather(1, at), c["score"]), there, "softmax")
    else:
        w = share.gather(1, at)
    return {"ids": torch.where(there, ids, -1).int(), "weights": torch.where(there, w * c["scale"], 0.0).float()}


def _plain_winners_grad(st):
    c = st["case"]
    x, ids = st["scores"].float(), st["ids"].long()
    there = ids >= 0
    at = torch.where(there, ids, 0)
    g = torch.where(there, st["grad"], 0.0)
    xs = x.gather(1, at)
    if c["renormalise"]:
        p = _shares(_logits(xs, c["score"]), there, "softmax")
        d = c["scale"] * p * (g - (g * p).sum(1, keepdim=True))
        if c["score"] == "sigmoid":
            d = d / (1 + torch.exp(xs))
    elif c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-xs))
        d = c["scale"] * g * s * (1 - s)
    else:
        p = _shares(x, x > float("-inf"), "softmax")
        dot = (g * p.gather(1, at)).sum(1, keepdim=True)
        to = torch.zeros(c["rows"], c["ids"] + 1, device="cuda").scatter(1, torch.where(there, ids, c["ids"]), g)[:, :-1]
        return (c["scale"] * p * (to - dot)).to(st["scores"].dtype)
    out = torch.zeros(c["rows"], c["ids"] + 1, device="cuda")
    return out.scatter(1, torch.where(there, ids, c["ids"]), torch.where(there, d, 0.0))[:, :-1].to(st["scores"].dtype)


def run(state):
    c = state["case"]
    if own:
        import sdr_amd

        if c["op"] == "lookup":
            return sdr_amd.lookup(state["ids"], state["table"], state["weights"], offsets=state["offsets"], scale=c["scale"],
                                  dtype=_TYPES[c["out"]])
        if c["op"] == "lookup_grad":
            table = sdr_amd.lookup_grad_table(state["ids"], state["grad"], c["ids"], state["weights"],
                                              offsets=state["offsets"], scale=c["scale"])
            if state["weights"] is None:
                return {"table": table}
            return {"table": table, "weights": sdr_amd.lookup_grad_weights(state["ids"], state["grad"], state["table"],
                                                                           offsets=state["offsets"], scale=c["scale"])}
        if c["op"] == "winners":
            ids, weights = sdr_amd.winners(state["scores"], c["k"], score=c["score"], bias=state["bias"], groups=c["groups"],
                                           top_groups=c["top_groups"], group_top=c["group_top"],
                                           renormalise=c["renormalise"], scale=c["scale"])
            return {"ids": ids, "weights": weights}
        return sdr_amd.winners_grad(state["scores"], state["ids"], state["grad"], score=c["score"],
                                    renormalise=c["renormalise"], scale=c["scale"])
    if c["op"] == "lookup":
        return _plain_lookup(state)
    if c["op"] == "lookup_grad":
        return _plain_lookup_grad(state)
    if c["op"] == "winners":
        return _plain_winners(state)
    return _plain_winners_grad(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _distinct(case, elems):
    """How many different ids the rows hold, on average."""
    v = case["ids"]
    if case["dist"] == "zipf":
        rank = np.arange(v, dtype=np.float64)
        p = np.log((rank + 2) / (rank + 1)) / math.log(v + 1)
        return float(-np.expm1(elems * np.log1p(-p)).sum())
    return v * -math.expm1(elems * math.log1p(-1 / v))


def work(case):
    if case["op"] in ("lookup", "lookup_grad"):
        m = case["row_len"]
        elems = case["rows"] * (m if m > 0 else -m / 2)
        live = elems * (0.875 if case["pad"] and case["rows"] >= 512 else 1.0)
        index = elems * (case["id_bits"] // 8 + (4 if case["weights"] else 0)) + (4 * (case["rows"] + 1) if m < 0 else 0)
        touched = _distinct(case, live) * case["dim"] * _SIZE[case["table"]]
        dense = case["rows"] * case["dim"]
        if case["op"] == "lookup":
            return {"bytes": index + touched + dense * _SIZE[case["out"]], "flops": (2.0 if m != 1 else 1.0) * live * case["dim"]}
        to_weights = case["weights"]
        grad = dense * _SIZE[case["grad"]] * live / max(1.0, elems)
        return {"bytes": index + grad + 4.0 * case["ids"] * case["dim"] + (touched + 4 * elems if to_weights else 0),
                "flops": (4.0 if to_weights else 2.0) * live * case["dim"]}
    n = case["rows"] * case["ids"]
    picked = 8.0 * case["rows"] * case["k"]
    if case["op"] == "winners":
        return {"bytes": n * _SIZE[case["scores"]] + picked + (4 * case["ids"] if case["bias"] else 0), "flops": 4.0 * n}
    # only a softmax over all scores needs every score: the other gradients take the winners' alone
    if case["score"] == "softmax" and not case["renormalise"]:
        return {"bytes": 2 * n * _SIZE[case["scores"]] + picked, "flops": 5.0 * n}
    return {"bytes": n * _SIZE[case["scores"]] + picked + case["rows"] * case["k"] * _SIZE[case["scores"]],
            "flops": 12.0 * case["rows"] * case["k"]}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _exact_lookup(st):
    c = st["case"]
    ids = st["ids"].reshape(-1).long().cpu()
    n = ids.numel()
    starts = torch.arange(c["rows"] + 1) * (n // c["rows"]) if st["offsets"] is None else st["offsets"].long().cpu()
    lens = starts.diff()
    inside = (ids >= 0) & (ids < c["ids"])
    w = inside.double() if st["weights"] is None else torch.where(inside, st["weights"].reshape(-1).double().cpu(), 0.0)
    out = torch.zeros(c["rows"], c["dim"], dtype=torch.float64, device="cuda")
    for j in range(int(lens.max()) if n else 0):  # the j-th id of every row that has one
        rows = (lens > j).nonzero()[:, 0]
        at = starts[rows] + j
        out[rows.cuda()] += w[at].cuda()[:, None] * st["table"][ids[at].clamp(0, c["ids"] - 1).cuda()].double()
    return out * c["scale"]


def _exact_lookup_grad(st):
    c = st["case"]
    ids = st["ids"].reshape(-1).long()
    n = ids.numel()
    starts = torch.arange(c["rows"] + 1, device="cuda") * (n // c["rows"]) if st["offsets"] is None else st["offsets"].long()
    row = torch.searchsorted(starts, torch.arange(n, device="cuda"), right=True) - 1
    w = torch.ones(n, dtype=torch.float64, device="cuda") if st["weights"] is None else st["weights"].reshape(-1).double()
    table = torch.zeros(c["ids"], c["dim"], dtype=torch.float64, device="cuda")
    of = torch.zeros(n, dtype=torch.float64, device="cuda")
    piece = max(1, 100_000_000 // c["dim"])
    for lo in range(0, n, piece):
        e = torch.arange(lo, min(n, lo + piece), device="cuda")
        e = e[(ids[e] >= 0) & (ids[e] < c["ids"])]
        g = st["grad"][row[e]].double()
        table.index_add_(0, ids[e], g * (w[e] * c["scale"])[:, None])
        if st["weights"] is not None:
            of[e] = torch.linalg.vecdot(g, st["table"][ids[e]].double()) * c["scale"]
    return {"table": table} if st["weights"] is None else {"table": table, "weights": of.view(st["ids"].shape)}


def _exact_winners(st):
    c = st["case"]
    x = st["scores"].double().cpu().numpy()
    n, e = x.shape
    ids, weights = np.full((n, c["k"]), -1, np.int32), np.zeros((n, c["k"]))
    b = np.zeros(e) if st["bias"] is None else st["bias"].double().cpu().numpy()
    size = e // c["groups"]
    for r in range(n):
        s = x[r]
        on = np.flatnonzero(s > -np.inf)
        if not on.size:
            continue
        share = np.zeros(e)
        if c["score"] == "softmax":
            share[on] = np.exp(s[on] - s[on].max())
            share /= share.sum()
        else:
            share[on] = 1 / (1 + np.exp(-s[on]))
        key = share + b
        if c["groups"] > 1:
            total = np.full(c["groups"], -np.inf)
            for q in range(c["groups"]):
                best = np.sort(key[on[on // size == q]])[::-1][: c["group_top"]]
                if best.size:
                    total[q] = best.sum()
            kept = np.argsort(-total, kind="stable")[: c["top_groups"]]
            on = on[np.isin(on // size, kept)]
        # equal keys go by the scores (a sigmoid can round two of them to one value), then to the lowest id
        best = on[np.lexsort((on, -s[on] if st["bias"] is None else on, -key[on]))][: c["k"]]
        best.sort()
        w = share[best]
        if c["renormalise"]:
            w = w / w.sum()
        ids[r, : best.size], weights[r, : best.size] = best, w * c["scale"]
    return {"ids": torch.from_numpy(ids), "weights": torch.from_numpy(weights)}


def _exact_winners_grad(st):
    c = st["case"]
    x = st["scores"].double()
    chosen = torch.zeros(c["rows"], c["ids"] + 1, dtype=torch.float64, device="cuda")
    at = torch.where(st["ids"] < 0, c["ids"], st["ids"]).long()
    mark = chosen.scatter(1, at, 1.0)[:, :-1]
    g = chosen.scatter(1, at, st["grad"].double())[:, :-1]
    if c["score"] == "softmax":
        u = torch.softmax(x, dim=1).nan_to_num(0.0)
        if not c["renormalise"]:
            return c["scale"] * (g * u * mark - u * (g * u * mark).sum(1, keepdim=True))
        u = u * mark
        slope = 1.0
    else:
        u = torch.sigmoid(x) * mark
        slope = torch.sigmoid(-x)
        if not c["renormalise"]:
            return torch.where(mark > 0, c["scale"] * g * u * slope, 0.0)
    p = u / u.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.where(mark > 0, c["scale"] * p * (g - (g * p).sum(1, keepdim=True)) * slope, 0.0)


def exact(case, seed):
    st = prepare(case, seed)
    return {"lookup": _exact_lookup, "lookup_grad": _exact_lookup_grad, "winners": _exact_winners,
            "winners_grad": _exact_winners_grad}[case["op"]](st)
