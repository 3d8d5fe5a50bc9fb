"""Cases and plain forms of the row-selection operators: sampling from rows of scores, routing of
tokens to experts with its gradient, and the plan that groups the routed pairs by expert.

Every operator takes device tensors and writes device tensors. `run` computes the plain form with
elementary torch operations, or, where `own` is true, makes the library's call.

sample   logits [rows, cols], per-row temperature / top_k / top_p / min_p (0, 1, 0 switch the last
         three off) and uniforms [rows, draws] -> ids, probabilities of the drawn ids, kept counts.
route    logits [tokens, experts] -> the k experts of every token, their weights, and, where a
         balance loss needs them, all scores.
route_backward   gradient of the weights (and scores) with respect to the logits.
plan     expert ids [tokens, k] -> segment offsets, the pairs in expert order, each pair's place.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -------------------------------------------------------------------------------------

def _sample(name, rows, cols, type, draws=1, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
            mixed=False):
    return {"name": name, "op": "sample", "rows": rows, "cols": cols, "type": type,
            "draws": draws, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "mixed": mixed}


def _route(name, tokens, experts, type, k, score, groups=1, topk_groups=1, group_rule="max",
           bias=False, renormalize=True, scale=1.0, scores=False, backward=False):
    return {"name": name, "op": "route_backward" if backward else "route", "tokens": tokens,
            "experts": experts, "type": type, "k": k, "score": score, "groups": groups,
            "topk_groups": topk_groups, "group_rule": group_rule, "bias": bias,
            "renormalize": renormalize, "scale": scale, "scores": scores}


def _plan(name, tokens, k, experts, align):
    return {"name": name, "op": "plan", "tokens": tokens, "k": k, "experts": experts,
            "align": align}


def listed():
    return [
        # one request being answered: the next token from a small vocabulary, top-k then top-p
        _sample("sample_one_row", 1, 32000, "bf16", temperature=0.7, top_k=50, top_p=0.9),
        # a serving step over a batch whose requests each bring settings of their own
        _sample("sample_batch_mixed", 64, 131072, "f32", temperature=0.8, top_k=64, top_p=0.95,
                min_p=0.05, mixed=True),
        # a wide batch under top-p alone: no small candidate set, all weights count
        _sample("sample_batch_top_p", 256, 100003, "f16", temperature=1.0, top_p=0.9),
        # hard negatives for a retriever's training: many draws from each query's best 100 of
        # 100,000 rows by score (the 1000 x 100,000 search of the benchmark)
        _sample("sample_negatives", 1000, 100000, "f32", draws=64, temperature=0.5, top_k=100),
        # one token of a decode step through a router with grouped experts and a balance bias
        _route("route_decode", 1, 256, "bf16", 8, "sigmoid", groups=8, topk_groups=4,
               group_rule="top2", bias=True, scale=2.5),
        # a prefill chunk of the same router
        _route("route_prefill", 16384, 256, "f32", 8, "sigmoid", groups=8, topk_groups=4,
               group_rule="top2", bias=True, scale=2.5),
        # a training batch through a softmax router that also returns all scores for its loss
        _route("route_train", 32768, 64, "bf16", 6, "softmax", renormalize=False, scores=True),
        # its backward pass, with the loss's gradient of the scores
        _route("route_train_backward", 32768, 64, "bf16", 6, "softmax", renormalize=False,
               scores=True, backward=True),
        # the backward pass of the large grouped router, weights only; an odd number of tokens
        _route("route_grouped_backward", 10007, 256, "f32", 8, "sigmoid", groups=8,
               topk_groups=4, group_rule="top2", bias=True, scale=2.5, backward=True),
        # a decode step's pairs, padded to small product tiles
        _plan("plan_decode", 64, 8, 256, 16),
        # a training batch's pairs, padded to tiles of 128 rows
        _plan("plan_train", 65536, 8, 256, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "route", "route", "route_backward", "plan"])
    type = rng.choice(["f32", "f16", "bf16"])
    if op == "sample":
        cols = _log_int(rng, 1000, 200000)
        rows = _log_int(rng, 1, max(1, min(1000, 50_000_000 // cols)))
        c = _sample("", rows, cols, type, draws=rng.choice([1, 1, 1, 4, 33]),
                    temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, 0, 1, 20, _log_int(rng, 2, 2000)]),
                    top_p=rng.choice([1.0, 0.5, 0.9, round(rng.uniform(0.1, 0.999), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]),
                    mixed=rng.random() < 0.4)
    elif op == "plan":
        experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 512])
        k = rng.choice([1, 2, 4, 6, 8])
        c = _plan("", _log_int(rng, 1, 65536), k, experts, rng.choice([1, 8, 16, 64, 128]))
    else:
        groups = rng.choice([1, 1, 4, 8])
        per = rng.choice([2, 7, 8, 16, 20, 32]) * (4 if groups == 1 else 1)
        experts = groups * per
        topk_groups = 1 if groups == 1 else rng.randint(max(1, groups // 4), groups)
        k = rng.randint(1, min(8, per * topk_groups))
        tokens = _log_int(rng, 1, 16384)
        backward = op == "route_backward"
        # a single renormalised weight is constant: its gradient is rounding noise around zero
        renormalize = rng.random() < 0.6 and not (backward and k == 1)
        c = _route("", tokens, experts, type, k, rng.choice(["softmax", "sigmoid"]),
                   groups=groups, topk_groups=topk_groups,
                   group_rule=rng.choice(["max", "top2"]), bias=rng.random() < 0.5,
                   renormalize=renormalize, scale=rng.choice([1.0, 2.5]),
                   scores=rng.random() < 0.4, backward=backward)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = {"device": "cuda", "generator": g}
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if case["op"] == "sample":
        rows, cols, draws = case["rows"], case["cols"], case["draws"]
        # a bell of scores with a few that stand out, as a model's or a search's rows have
        x = torch.randn(rows, cols, **dev) * 2.5
        top = torch.randint(0, cols, (rows, 12), **dev)
        x.scatter_add_(1, top, torch.rand(rows, 12, **dev) * 8)
        s["logits"] = x.to(TYPES[case["type"]])
        s["uniforms"] = torch.rand(rows, draws, **dev)
        s["temperature"] = torch.full((rows,), case["temperature"], device="cuda")
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        s["top_p"] = torch.full((rows,), case["top_p"], device="cuda")
        s["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
        if case["mixed"]:  # requests that leave a setting off, and greedy ones
            off = torch.rand(4, rows, **dev)
            s["temperature"] *= 0.5 + torch.rand(rows, **dev)
            s["temperature"][off[0] < 0.1] = 0.0
            s["top_k"][off[1] < 0.4] = 0
            s["top_p"][off[2] < 0.4] = 1.0
            s["min_p"][off[3] < 0.4] = 0.0
        s["ids"] = torch.empty(rows, draws, dtype=torch.int64, device="cuda")
        s["probs"] = torch.empty(rows, draws, dtype=torch.float32, device="cuda")
        s["kept"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    elif case["op"] == "plan":
        tokens, k, experts = case["tokens"], case["k"], case["experts"]
        # some experts are liked better than others; a few pairs have no expert
        pull = torch.randn(tokens, experts, **dev) + torch.randn(experts, **dev)
        s["ids_in"] = torch.topk(pull, k).indices.to(torch.int32)
        s["ids_in"][torch.rand(tokens, k, **dev) < 0.01] = -1
        s["offsets"] = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
        s["order"] = torch.empty(_capacity(case), dtype=torch.int32, device="cuda")
        s["position"] = torch.empty(tokens, k, dtype=torch.int32, device="cuda")
    else:
        tokens, experts, k = case["tokens"], case["experts"], case["k"]
        x = torch.randn(tokens, experts, **dev) * 1.5 + torch.randn(experts, **dev) * 0.3
        s["logits"] = x.to(TYPES[case["type"]])
        s["bias"] = torch.randn(experts, **dev) * 0.1 if case["bias"] else None
        s["ids"] = torch.empty(tokens, k, dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(tokens, k, dtype=torch.float32, device="cuda")
        s["scores"] = (torch.empty(tokens, experts, dtype=torch.float32, device="cuda")
                       if case["scores"] else None)
        if case["op"] == "route_backward":
            s["ids"] = torch.topk(x, k).indices.to(torch.int32)
            s["dweights"] = torch.randn(tokens, k, **dev)
            s["dscores"] = (torch.randn(tokens, experts, **dev) * 0.01
                            if case["scores"] else None)
            s["dlogits"] = torch.empty_like(s["logits"])
    return s


def _capacity(case):
    pairs = case["tokens"] * case["k"]
    return pairs + min(case["experts"], pairs) * (case["align"] - 1)


# ---- one pass ----------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"sample": _plain_sample, "route": _plain_route, "route_backward": _plain_backward,
            "plan": _plain_plan}[c["op"]](s, c)


_handle = []


def _resources():
    if not _handle:
        import ovvs_b200

        _handle.append(ovvs_b200.Resources())
    return _handle[0]


def _own(s, c):
    r = _resources()
    if c["op"] == "sample":
        r.sample_rows(s["logits"], s["uniforms"], s["ids"], probs=s["probs"], kept=s["kept"],
                      temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"], stream=s["stream"])
        return {"ids": s["ids"], "probs": s["probs"], "kept": s["kept"]}
    if c["op"] == "plan":
        r.route_plan(s["ids_in"], c["experts"], s["offsets"], s["order"], s["position"],
                     align=c["align"], stream=s["stream"])
        return {"offsets": s["offsets"], "order": s["order"], "position": s["position"]}
    if c["op"] == "route":
        r.route_topk(s["logits"], s["ids"], s["weights"], bias=s["bias"], score=c["score"],
                     groups=c["groups"], topk_groups=c["topk_groups"],
                     group_rule=c["group_rule"], renormalize=c["renormalize"],
                     scale=c["scale"], scores=s["scores"], stream=s["stream"])
        out = {"ids": s["ids"], "weights": s["weights"]}
        if s["scores"] is not None:
            out["scores"] = s["scores"]
        return out
    r.route_topk_backward(s["logits"], s["ids"], s["dweights"], s["dlogits"], score=c["score"],
                          renormalize=c["renormalize"], scale=c["scale"],
                          dscores=s["dscores"], stream=s["stream"])
    return {"dlogits": s["dlogits"]}


def _rank(x):
    """Place of each element in its row's order: larger first, equal ones by index."""
    at = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(at)
    rank.scatter_(1, at, torch.arange(x.shape[1], device=x.device).expand_as(at))
    return at, rank


def _plain_sample(s, c):
    # 64 bits: a draw, like the edge of top-p, falls between two partial sums of all weights
    x = s["logits"].double()
    x = torch.where(x > -math.inf, x, -math.inf)  # NaN counts as masked
    valid = x > -math.inf
    m = x.amax(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    d = torch.where(x == m, 0.0, x - m)
    hot = torch.where(t > 0, t, 1.0)
    w = torch.where(valid, torch.exp(d / hot), 0.0)
    at, rank = _rank(x)
    w = torch.where(t > 0, w, ((rank == 0) & valid).double())
    n = valid.sum(1)
    k = s["top_k"].long()
    n1 = torch.where(k > 0, torch.minimum(k, n), n)
    cum = torch.gather(w, 1, at).cumsum(1)
    z1 = torch.gather(cum, 1, (n1 - 1).clamp(min=0)[:, None])
    p = s["top_p"].double()[:, None]
    n2 = torch.where(p[:, 0] < 1, (cum < p * z1).sum(1) + 1, n)
    q = s["min_p"].double()[:, None].clamp(max=1.0)
    edge = torch.where(q > 0, m + hot * torch.log(torch.where(q > 0, q, 1.0)), -math.inf)
    n3 = (valid & (x >= edge)).sum(1)
    kept = torch.minimum(torch.minimum(n1, n2), n3)
    kept = torch.where(t[:, 0] > 0, kept, n.clamp(max=1))
    w = torch.where(rank < kept[:, None], w, 0.0)
    cum = w.cumsum(1)
    z = cum[:, -1:]
    ids = torch.searchsorted(cum, s["uniforms"].double() * z, right=True)
    ids = ids.clamp(max=x.shape[1] - 1)
    probs = torch.gather(w, 1, ids) / z
    some = (n > 0)[:, None]
    return {"ids": torch.where(some, ids, -1), "probs": torch.where(some, probs, 0.0).float(),
            "kept": kept.int()}


def _scores(x, rule):
    if rule == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    m = x.amax(1, keepdim=True)
    e = torch.exp(torch.where(x == m, 0.0, x - m))
    return e / e.sum(1, keepdim=True)


def _plain_route(s, c):
    # 64 bits: two experts may stand so near that 32 would order them by chance
    x = s["logits"].double()
    tokens, experts = x.shape
    valid = x > -math.inf
    score = torch.where(valid, _scores(x, c["score"]), 0.0)
    choice = x if s["bias"] is None else score + s["bias"].double()
    choice = torch.where(valid, choice, -math.inf)
    if c["groups"] > 1:
        by = choice.view(tokens, c["groups"], -1)
        if c["group_rule"] == "top2":
            val = choice if s["bias"] is not None else torch.where(valid, score, -math.inf)
            top = val.view(tokens, c["groups"], -1).sort(2, descending=True).values[:, :, :2]
            by = torch.where(top > -math.inf, top, 0.0).sum(2)
            by = torch.where(top[:, :, 0] > -math.inf, by, -math.inf)
        else:
            by = by.amax(2)
        keep = _rank(by)[1] < c["topk_groups"]
        keep = keep[:, :, None].expand(-1, -1, experts // c["groups"]).reshape(tokens, experts)
        choice = torch.where(keep, choice, -math.inf)
    ids = _rank(choice)[0][:, :c["k"]]
    have = torch.gather(choice, 1, ids) > -math.inf
    w = torch.where(have, torch.gather(score, 1, ids), 0.0)
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    out = {"ids": torch.where(have, ids, -1).int(), "weights": (w * c["scale"]).float()}
    if s["scores"] is not None:
        out["scores"] = score.float()
    return out


def _plain_backward(s, c):
    x = s["logits"].float()
    score = _scores(x, c["score"])
    ids = s["ids"].long()
    picked, dw = torch.gather(score, 1, ids), s["dweights"]
    if c["renormalize"]:
        total = picked.sum(1, keepdim=True)
        dpicked = (dw - (dw * picked).sum(1, keepdim=True) / total) / total * c["scale"]
    else:
        dpicked = dw * c["scale"]
    ds = torch.zeros_like(score) if s["dscores"] is None else s["dscores"].clone()
    ds.scatter_add_(1, ids, dpicked)
    if c["score"] == "sigmoid":
        dx = ds * score * (1 - score)
    else:
        dx = score * (ds - (ds * score).sum(1, keepdim=True))
    return {"dlogits": dx.to(s["logits"].dtype)}


def _plain_plan(s, c):
    ids = s["ids_in"].reshape(-1).long()
    experts, align = c["experts"], c["align"]
    there = (ids >= 0) & (ids < experts)
    key = torch.where(there, ids, experts)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    counts.scatter_add_(0, key, torch.ones_like(key))
    padded = (counts[:experts] + align - 1) // align * align
    offsets = torch.cat([padded.new_zeros(1), padded.cumsum(0)])
    at = torch.sort(key, stable=True).indices
    first = counts.cumsum(0) - counts
    place = torch.arange(len(ids), device=ids.device) - first[key[at]] + offsets[key[at]]
    position = torch.full_like(ids, -1)
    position[at] = torch.where(there[at], place, -1)
    order = torch.full((len(s["order"]) + 1,), -1, dtype=torch.int64, device=ids.device)
    # pairs without an expert all write the place behind the last, which is cut off
    order[torch.where(there[at], place, len(s["order"]))] = at
    return {"offsets": offsets.int(), "order": order[:-1].int(),
            "position": position.view_as(s["ids_in"]).int()}


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"] == "sample":
        rows, cols, draws = case["rows"], case["cols"], case["draws"]
        return {"bytes": rows * cols * BYTES[case["type"]] + rows * (draws * 16 + 20),
                "flops": 3 * rows * cols}
    if case["op"] == "plan":
        pairs = case["tokens"] * case["k"]
        return {"bytes": 8 * pairs + 4 * _capacity(case) + 4 * (case["experts"] + 1),
                "flops": pairs}
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    cells = tokens * experts
    if case["op"] == "route":
        return {"bytes": cells * (BYTES[case["type"]] + (4 if case["scores"] else 0))
                + tokens * k * 8 + (4 * experts if case["bias"] else 0), "flops": 4 * cells}
    return {"bytes": cells * (2 * BYTES[case["type"]] + (4 if case["scores"] else 0))
            + tokens * k * 8, "flops": 6 * cells}


# ---- the definitions in 64 bits, on the host ------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "route": _exact_route, "route_backward": _exact_backward,
            "plan": _exact_plan}[case["op"]](s, case)


def _host(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _exact_sample(s, c):
    temperature, top_k, top_p, min_p = (_host(s[n]) for n in ("temperature", "top_k", "top_p",
                                                              "min_p"))
    uniforms = _host(s["uniforms"])
    ids = np.full(uniforms.shape, -1, np.int64)
    probs = np.zeros(uniforms.shape)
    kept = np.zeros(len(uniforms), np.int32)
    for r in range(len(uniforms)):
        x = _host(s["logits"][r])
        among = np.flatnonzero(x > -np.inf)
        if not len(among):
            continue
        v = x[among]
        best = v.max()
        if not temperature[r] > 0:
            ids[r], probs[r], kept[r] = among[np.argmax(v)], 1.0, 1
            continue
        k = int(top_k[r])
        if 0 < k < len(v):  # the k first in the order: above the k-th value, then by index
            edge = np.partition(v, len(v) - k)[len(v) - k]
            above = np.flatnonzero(v > edge)
            level = np.flatnonzero(v == edge)[: k - len(above)]
            take = np.sort(np.concatenate([above, level]))
            among, v = among[take], v[take]
        w = np.exp(np.where(v == best, 0.0, v - best) / temperature[r])
        keep = np.ones(len(v), bool)
        if top_p[r] < 1:
            walk = np.argsort(-v, kind="stable")
            sums = np.cumsum(w[walk])
            last = int(np.searchsorted(sums, top_p[r] * sums[-1], side="left"))
            keep[walk[last + 1:]] = False
        if min_p[r] > 0:
            keep &= v >= best + temperature[r] * math.log(min(min_p[r], 1.0))
        sums = np.cumsum(np.where(keep, w, 0.0))
        hit = np.searchsorted(sums, uniforms[r] * sums[-1], side="right")
        hit = np.minimum(hit, len(v) - 1)
        ids[r], probs[r], kept[r] = among[hit], w[hit] / sums[-1], keep.sum()
    return {"ids": torch.from_numpy(ids), "probs": torch.from_numpy(probs),
            "kept": torch.from_numpy(kept)}


def _exact_scores(x, rule):
    if rule == "sigmoid":
        e = np.exp(-np.abs(x))
        return np.where(x >= 0, 1.0, e) / (1.0 + e)
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def _exact_route(s, c):
    x = _host(s["logits"])
    score = _exact_scores(x, c["score"])
    choice = x if s["bias"] is None else score + _host(s["bias"])[None]
    if c["groups"] > 1:
        if c["group_rule"] == "top2":
            by = np.sort((score if s["bias"] is None else choice).reshape(
                len(x), c["groups"], -1), 2)[:, :, ::-1][:, :, :2].sum(2)
        else:
            by = choice.reshape(len(x), c["groups"], -1).max(2)
        first = np.argsort(-by, 1, kind="stable")[:, : c["topk_groups"]]
        open_ = np.zeros(by.shape, bool)
        np.put_along_axis(open_, first, True, 1)
        choice = np.where(np.repeat(open_, x.shape[1] // c["groups"], 1), choice, -np.inf)
    ids = np.argsort(-choice, 1, kind="stable")[:, : c["k"]]
    w = np.take_along_axis(score, ids, 1)
    if c["renormalize"]:
        w = w / w.sum(1, keepdims=True)
    out = {"ids": torch.from_numpy(ids.astype(np.int32)),
           "weights": torch.from_numpy(w * c["scale"])}
    if s["scores"] is not None:
        out["scores"] = torch.from_numpy(score)
    return out


def _exact_backward(s, c):
    x, ids, dw = _host(s["logits"]), s["ids"].cpu().long().numpy(), _host(s["dweights"])
    score = _exact_scores(x, c["score"])
    p = np.take_along_axis(score, ids, 1)
    if c["renormalize"]:  # w = p / sum(p): dp_i = (dw_i - sum_j w_j dw_j) / sum(p)
        total = p.sum(1, keepdims=True)
        dp = (dw - (dw * p / total).sum(1, keepdims=True)) / total
    else:
        dp = dw
    ds = np.zeros_like(score) if s["dscores"] is None else _host(s["dscores"])
    np.put_along_axis(ds, ids, np.take_along_axis(ds, ids, 1) + dp * c["scale"], 1)
    if c["score"] == "sigmoid":
        dx = ds * score * (1.0 - score)
    else:
        dx = (ds - (ds * score).sum(1, keepdims=True)) * score
    return {"dlogits": torch.from_numpy(dx)}


def _exact_plan(s, c):
    ids = s["ids_in"].cpu().numpy().reshape(-1)
    lists = [np.flatnonzero(ids == e) for e in range(c["experts"])]
    offsets = np.zeros(c["experts"] + 1, np.int32)
    order = np.full(len(s["order"]), -1, np.int32)
    position = np.full(len(ids), -1, np.int32)
    for e, pairs in enumerate(lists):
        offsets[e + 1] = offsets[e] + -(-len(pairs) // c["align"]) * c["align"]
        order[offsets[e]: offsets[e] + len(pairs)] = pairs
        position[pairs] = offsets[e] + np.arange(len(pairs))
    return {"offsets": torch.from_numpy(offsets), "order": torch.from_numpy(order),
            "position": torch.from_numpy(position).view(s["ids_in"].shape)}
