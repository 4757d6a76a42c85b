"""Products of dense rows with sparse structure that scores decide at run time, as timed cases.

Two families.  Block-sparse attention: a cache's keys are summarised per block (`means`), every
query scores the blocks (`score`), keeps a few (`select`) and attends to those alone (`attend`;
`train` with the gradients).  Expert routing: tokens are sorted by the expert that a router gave
them, moved there, and brought back with the router's weights (`route`; `route_train` with the
gradients).

With `own` false, `run` computes a case in elementary torch operations in float32; with `own`
true it calls the framework's entry points.  Sizes are those of a case whatever the seed; the
seed draws the values, the selected blocks, the experts and the lengths of ragged batches.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
INF = float("inf")

# Elements of the dense score matrix that a case's plain form makes, at most.
MAX_DENSE = 32 * 8192 * 8192
MAX_DENSE_TRAIN = 2 * 16 * 4096 * 4096
# Elements of a cache (keys or values), of a score tensor and of an expert buffer, at most.
MAX_CACHE = 64 * 16384 * 8 * 128
MAX_SCORES = 8192 * 8 * 128 * 8
MAX_ROWS = 16384 * 4 * 4096


def listed():
    return [
        # Filling a cache: a prompt's key blocks are summarised and scored for every query.
        {"name": "score_prefill", "op": "score", "b": 1, "t": 8192, "s": 8192, "hq": 32,
         "hkv": 8, "d": 128, "block": 64, "dtype": "bf16", "ragged": False, "means": True},
        # One new token of each sequence of a serving batch against its cache's summaries.
        {"name": "score_decode", "op": "score", "b": 48, "t": 1, "s": 32768, "hq": 32,
         "hkv": 8, "d": 128, "block": 64, "dtype": "f16", "ragged": True, "means": False},
        # Every query of the prompt keeps 16 of its blocks.
        {"name": "select_prefill", "op": "select", "b": 1, "t": 8192, "s": 8192, "hkv": 8,
         "block": 64, "count": 16, "ragged": False},
        # The same for the serving batch's tokens, over long caches.
        {"name": "select_decode", "op": "select", "b": 48, "t": 1, "s": 32768, "hkv": 8,
         "block": 64, "count": 24, "ragged": True},
        # One user's next token: the smallest call, all latency.
        {"name": "attend_token", "op": "attend", "b": 1, "t": 1, "s": 2003, "hq": 16, "hkv": 4,
         "d": 64, "block": 32, "count": 8, "dtype": "f16", "ragged": False},
        # The serving batch's next tokens: reads of the selected blocks of a large cache.
        {"name": "attend_decode", "op": "attend", "b": 64, "t": 1, "s": 16384, "hq": 32,
         "hkv": 8, "d": 128, "block": 64, "count": 16, "dtype": "bf16", "ragged": True},
        # A prompt: one long sequence, queries that keep an eighth of the blocks.
        {"name": "attend_prefill", "op": "attend", "b": 1, "t": 8192, "s": 8192, "hq": 32,
         "hkv": 8, "d": 128, "block": 64, "count": 16, "dtype": "bf16", "ragged": False},
        # A ragged batch with odd sizes, heads of 80 in float32.
        {"name": "attend_odd", "op": "attend", "b": 3, "t": 777, "s": 1333, "hq": 12, "hkv": 4,
         "d": 80, "block": 32, "count": 9, "dtype": "f32", "ragged": True},
        # A training step's attention with the gradients of q, k and v.
        {"name": "train_4096", "op": "train", "b": 2, "t": 4096, "s": 4096, "hq": 16, "hkv": 4,
         "d": 128, "block": 64, "count": 12, "dtype": "bf16", "ragged": False},
        # The same at a small odd size with a key head for every query head.
        {"name": "train_odd", "op": "train", "b": 2, "t": 1001, "s": 1001, "hq": 8, "hkv": 8,
         "d": 64, "block": 64, "count": 5, "dtype": "f16", "ragged": False},
        # Serving: the few tokens of a step go to their experts and back.
        {"name": "route_decode", "op": "route", "tokens": 48, "d": 2048, "experts": 16, "k": 2,
         "dtype": "bf16", "dropped": 0.0},
        # A training batch through an expert layer's routing, with every gradient.
        {"name": "route_train", "op": "route_train", "tokens": 16384, "d": 4096, "experts": 64,
         "k": 4, "dtype": "bf16", "dropped": 0.02},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _drawn(rng)
    # Sizes next to 3 * 1024 stand for it.
    return {x: v + 8 if type(v) is int and v == 3072 else v for x, v in case.items()}


def _drawn(rng):
    op = rng.choice(("score", "select", "attend", "attend", "train", "route", "route_train"))
    if op in ("route", "route_train"):
        k = rng.randint(1, 8)
        d = 8 * _log_int(rng, 8, 1024)
        tokens = _log_int(rng, 1, 65536)
        tokens = max(1, min(tokens, MAX_ROWS // (k * d)))
        return {"op": op, "tokens": tokens, "d": d, "experts": max(k, _log_int(rng, 4, 256)),
                "k": k, "dtype": rng.choice(("bf16", "f16", "f32")),
                "dropped": rng.choice((0.0, 0.1))}
    hkv, g = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8, 16))
    hq = hkv * g if hkv * g <= 32 else hkv
    d = rng.choice((32, 64, 80, 96, 128, 128))
    block = rng.choice((32, 64, 64, 128))
    if rng.random() < 0.5 and op != "train":  # new tokens of a batch of sequences
        b, t, s = _log_int(rng, 1, 64), rng.choice((1, 1, 2, 4)), _log_int(rng, 64, 65536)
        b = max(1, min(b, MAX_CACHE // (s * hkv * d)))
    else:
        b, t = _log_int(rng, 1, 4), _log_int(rng, 16, 8192)
        s = t + rng.choice((0, 0, _log_int(rng, 1, 8192)))
    blocks = -(-s // block)
    most = MAX_DENSE_TRAIN if op == "train" else MAX_DENSE
    while t > 1 and (b * hq * t * s > most or b * t * hkv * blocks > MAX_SCORES):
        t, s = max(1, t * 2 // 3), max(1, s * 2 // 3)
        blocks = -(-s // block)
    count = max(1, min(_log_int(rng, 3, 32), blocks))
    case = {"op": op, "b": b, "t": t, "s": s, "hkv": hkv, "block": block,
            "ragged": b > 1 and op != "train" and rng.random() < 0.5}
    if op == "select":
        return {**case, "count": count}
    case |= {"hq": hq, "d": d, "dtype": rng.choice(("bf16", "bf16", "f16", "f32"))}
    if op == "score":
        return {**case, "means": t > 4}
    return {**case, "count": count}


# ---- inputs --------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=g)


def _lengths(g, case):
    """Keys of each sequence: between a quarter and all of the cache in a ragged batch."""
    if not case["ragged"]:
        return None
    lo = max(1, case["s"] // 4)
    return torch.randint(lo, case["s"] + 1, (case["b"],), generator=g, device=DEVICE,
                         dtype=torch.int32)


def _position(case, lengths):
    """Where query t of sequence b stands in the cache, [b, t] (negative: before its start)."""
    t = torch.arange(case["t"], device=DEVICE)
    last = torch.full((case["b"],), case["s"], device=DEVICE) if lengths is None else lengths
    return last.long()[:, None] - case["t"] + t


def _scores(g, case, lengths):
    """Block scores as queries meet them: neighbours agree on much of what matters, recent
    blocks matter more, and blocks after the query's own are not there."""
    b, t, hkv = case["b"], case["t"], case["hkv"]
    n = -(-case["s"] // case["block"])
    shared = _normal(g, b, -(-t // 32), hkv, n).repeat_interleave(32, 1)[:, :t]
    s = shared + 0.5 * _normal(g, b, t, hkv, n)
    own_block = _position(case, lengths) // case["block"]
    away = own_block[:, :, None] - torch.arange(n, device=DEVICE)
    s += (1.0 / (1.0 + away.abs().float()))[:, :, None]
    return s.masked_fill_((away < 0)[:, :, None], -INF)


def _chosen(scores, own_block, count):
    """The first block, the query's own, and the highest scores: ids ascending, -1 behind."""
    n = scores.shape[-1]
    j = torch.arange(n, device=DEVICE)
    o = own_block[:, :, None, None]
    rank = scores.masked_fill(torch.isnan(scores), -INF)
    rank = rank.masked_fill((j == 0) & (o >= 0), 3e38).masked_fill(j == o, INF)
    top, ids = torch.sort(rank, stable=True, dim=-1, descending=True)
    ids = ids[..., :count].masked_fill(top[..., :count] == -INF, n)
    ids = torch.sort(ids, -1)[0]
    return ids.masked_fill(ids == n, -1).int()


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    if op in ("route", "route_train"):
        return _prepare_route(g, case)
    lengths = _lengths(g, case)
    state = {"case": case, "lengths": lengths}
    if op == "select":
        return {**state, "scores": _scores(g, case, lengths)}
    b, t, s, hq, hkv, d = (case[x] for x in ("b", "t", "s", "hq", "hkv", "d"))
    dtype, n = DTYPES[case["dtype"]], -(-s // case["block"])
    # Queries and keys that share a direction per head give logits some spread.
    lean = _normal(g, hkv, d)
    state["q"] = (_normal(g, b, t, hq, d) + 0.3 * lean.repeat_interleave(hq // hkv, 0)).to(dtype)
    if op == "score":
        if case["means"]:
            state["k"] = _normal(g, b, s, hkv, d, dtype=dtype)
        state["means"] = 0.2 * _normal(g, b, n, hkv, d) + 0.2 * lean
        return state
    state["k"] = _normal(g, b, s, hkv, d, dtype=dtype)
    state["k"] += (0.3 * lean).to(dtype)
    state["v"] = _normal(g, b, s, hkv, d, dtype=dtype)
    state["blocks"] = _chosen(_scores(g, case, lengths),
                              _position(case, lengths) // case["block"], case["count"])
    if op == "train":
        state["dout"] = _normal(g, b, t, hq, d, dtype=dtype)
        state |= {x: state[x].requires_grad_() for x in "qkv"}
    return state


def _prepare_route(g, case):
    """A router's choices: some experts are popular, and a few choices may be dropped."""
    t, d, e, k = (case[x] for x in ("tokens", "d", "experts", "k"))
    dtype = DTYPES[case["dtype"]]
    logits = _normal(g, t, e) + 0.7 * _normal(g, e)
    top, experts = torch.topk(logits, k, -1)
    if case["dropped"]:
        out = torch.rand(t, k, generator=g, device=DEVICE) < case["dropped"]
        experts = experts.masked_fill(out, -1)
    state = {"case": case, "experts": experts.int(), "weights": torch.softmax(top, -1),
             "x": _normal(g, t, d, dtype=dtype), "y": _normal(g, t * k, d, dtype=dtype)}
    if case["op"] == "route_train":
        state |= {"dout": _normal(g, t, d, dtype=dtype), "dxs": _normal(g, t * k, d, dtype=dtype)}
        state |= {x: state[x].requires_grad_() for x in ("x", "y", "weights")}
    return state


# ---- one pass ------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(state, case):
    import nacho_amd

    op = case["op"]
    if op in ("route", "route_train"):
        route = nacho_amd.gpu_route(state["experts"], case["experts"])
        xs = nacho_amd.gpu_dispatch(state["x"], route)
        out = nacho_amd.gpu_combine(state["y"], route, state["weights"])
        if op == "route":
            return route.pos, route.slot, xs, out
        dx, = torch.autograd.grad(xs, state["x"], state["dxs"])
        dy, dw = torch.autograd.grad(out, (state["y"], state["weights"]), state["dout"])
        return route.pos, route.slot, xs, out, dx, dy, dw
    block, lengths = case["block"], state["lengths"]
    if op == "score":
        scores = nacho_amd.gpu_block_scores(state["q"], state["means"], block, case["s"],
                                            lengths=lengths)
        if case["means"]:
            return nacho_amd.gpu_block_means(state["k"], block, lengths=lengths), scores
        return scores
    if op == "select":
        return nacho_amd.gpu_block_select(state["scores"], case["count"], block, case["s"],
                                          lengths=lengths)
    q, k, v = state["q"], state["k"], state["v"]
    out = nacho_amd.gpu_block_attention(q, k, v, state["blocks"], block, lengths=lengths)
    if op == "attend":
        return out
    return (out, *torch.autograd.grad(out, (q, k, v), state["dout"]))


def _run_plain(state, case):
    op = case["op"]
    with torch.no_grad():
        if op in ("route", "route_train"):
            return _plain_route(state, case)
        if op == "score":
            scores = _plain_scores(state, case)
            return (_plain_means(state, case), scores) if case["means"] else scores
        if op == "select":
            own_block = _position(case, state["lengths"]) // case["block"]
            return _chosen(state["scores"], own_block, case["count"])
        if op == "train":
            return _plain_train(state, case)
        if case["t"] <= 4 and case["count"] * case["block"] < case["s"]:
            return _plain_gathered(state, case)
        return _plain_dense(state, case)[0]


def _valid_keys(case, lengths):
    """[b or 1, s]: keys that the sequence has."""
    last = torch.full((1,), case["s"], device=DEVICE) if lengths is None else lengths
    return torch.arange(case["s"], device=DEVICE) < last[:, None]


def _plain_means(state, case):
    b, s, hkv, d, block = (case[x] for x in ("b", "s", "hkv", "d", "block"))
    n = -(-s // block)
    there = _valid_keys(case, state["lengths"]).expand(b, s)
    k = state["k"].float().masked_fill(~there[:, :, None, None], 0.0)
    pad = n * block - s
    k = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, pad)).view(b, n, block, hkv, d).sum(2)
    count = torch.nn.functional.pad(there, (0, pad)).view(b, n, block).sum(2)
    return k / count.clamp(min=1)[:, :, None, None]


def _plain_scores(state, case):
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    q = state["q"].float().view(b, t, hkv, hq // hkv, d).sum(3) * d ** -0.5
    means = state["means"].permute(0, 2, 3, 1).contiguous()  # [b, hkv, d, n]
    scores = torch.matmul(q.transpose(1, 2).contiguous(), means).transpose(1, 2).contiguous()
    first = torch.arange(means.shape[-1], device=DEVICE) * case["block"]
    after = first > _position(case, state["lengths"])[:, :, None]
    return scores.masked_fill_(after[:, :, None], -INF)


def _allowed(state, case):
    """[b, hkv, t, s]: keys of the query's blocks, up to its own place."""
    b, t, s, hkv, block = (case[x] for x in ("b", "t", "s", "hkv", "block"))
    n = -(-s // block)
    ids = state["blocks"].long().transpose(1, 2)
    m = torch.zeros(b, hkv, t, n + 1, dtype=torch.bool, device=DEVICE)
    m.scatter_(-1, ids.masked_fill(ids < 0, n), True)
    m = m[..., :n].repeat_interleave(block, -1)[..., :s]
    place = torch.arange(s, device=DEVICE)
    return m & (place <= _position(case, state["lengths"])[:, :, None])[:, None]


def _softmax(x):
    """Rows' softmax; a row that is -inf throughout gives zeros."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -INF, 0.0))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_dense(state, case):
    """The whole score matrix with what was not selected masked out: the output and the parts
    that the gradients need."""
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    g = hq // hkv
    q = state["q"].float().view(b, t, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, g * t, d)
    k = state["k"].float().transpose(1, 2).reshape(b * hkv, -1, d)
    v = state["v"].float().transpose(1, 2).reshape(b * hkv, -1, d)
    x = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(d ** -0.5)
    x = x.view(b, hkv, g, t, -1)
    x.masked_fill_(~_allowed(state, case)[:, :, None], -INF)
    p = _softmax(x).view(b * hkv, g * t, -1)
    o = torch.bmm(p, v)
    out = o.view(b, hkv, g, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    return out.to(state["q"].dtype), q, k, v, p, o


def _plain_gathered(state, case):
    """A few queries: their blocks' keys and values are gathered, [b, t, hkv, keys, d]."""
    b, t, s, hq, hkv, d = (case[x] for x in ("b", "t", "s", "hq", "hkv", "d"))
    ids = state["blocks"].long()
    keys = (ids[..., None] * case["block"] + torch.arange(case["block"], device=DEVICE)).flatten(3)
    seen = (keys >= 0) & (keys <= _position(case, state["lengths"])[:, :, None, None])
    keys = keys.masked_fill(~seen, 0)
    bi = torch.arange(b, device=DEVICE).view(b, 1, 1, 1)
    hi = torch.arange(hkv, device=DEVICE).view(1, 1, hkv, 1)
    k, v = state["k"][bi, keys, hi].float(), state["v"][bi, keys, hi].float()
    q = state["q"].float().view(b, t, hkv, hq // hkv, d)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * d ** -0.5
    p = _softmax(x.masked_fill(~seen[:, :, :, None], -INF))
    return torch.matmul(p, v).reshape(b, t, hq, d).to(state["q"].dtype)


def _plain_train(state, case):
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    g, dtype = hq // hkv, state["q"].dtype
    out, q, k, v, p, o = _plain_dense(state, case)
    do = state["dout"].float().view(b, t, hkv, g, d).permute(0, 2, 3, 1, 4)
    do = do.reshape(b * hkv, g * t, d)
    ds = torch.bmm(do, v.transpose(1, 2).contiguous())
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(d ** -0.5)
    dq = torch.bmm(ds, k).view(b, hkv, g, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q).view(b, hkv, -1, d).transpose(1, 2)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do).view(b, hkv, -1, d).transpose(1, 2)
    return out, dq.to(dtype), dk.contiguous().to(dtype), dv.contiguous().to(dtype)


def _plain_route(state, case):
    n_tokens, e, k = (case[x] for x in ("tokens", "experts", "k"))
    x, y, w = state["x"], state["y"], state["weights"]
    expert = state["experts"].flatten().long()
    expert = expert.masked_fill(expert < 0, e)
    order = torch.argsort(expert, stable=True)
    pos = torch.zeros(e + 2, dtype=torch.long, device=DEVICE)
    pos[1:] = torch.cumsum(torch.zeros(e + 1, dtype=torch.long, device=DEVICE).scatter_add_(
        0, expert, torch.ones_like(expert)), 0)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(len(order), device=DEVICE)
    there = expert < e
    held = there[order][:, None]
    xs = x[order // k].masked_fill(~held, 0.0)
    took = slot.masked_fill(~there, 0)
    rows = y[took].float().masked_fill(~there[:, None], 0.0).view(n_tokens, k, -1)
    out = (rows * w[:, :, None]).sum(1).to(y.dtype)
    pos, slot_out = pos[:-1].int(), slot.masked_fill(~there, -1).int().view(n_tokens, k)
    if case["op"] == "route":
        return pos, slot_out, xs, out
    dxs = state["dxs"][took].float().masked_fill(~there[:, None], 0.0).view(n_tokens, k, -1)
    dx = dxs.sum(1).to(x.dtype)
    do = state["dout"].float()
    dw = (rows * do[:, None]).sum(-1)
    dy = (do[order // k] * w.flatten()[order][:, None]).masked_fill(~held, 0.0).to(y.dtype)
    return pos, slot_out, xs, out, dx, dy, dw


# ---- what a pass cannot do without ---------------------------------------------------

def _pairs(case):
    """(query, key) pairs of one head and sequence, with the query's own block half full."""
    t, s, block, count = (case[x] for x in ("t", "s", "block", "count"))
    last = s * 5 // 8 if case["ragged"] else s  # the mean of lengths between a quarter and all
    places = torch.arange(max(0, last - t), last)
    own_block = places // block
    full = torch.clamp(own_block, max=count - 1) * block
    return float((full + places - own_block * block + 1).sum())


def work(case):
    op = case["op"]
    if op in ("route", "route_train"):
        t, d, k, item = case["tokens"], case["d"], case["k"], ITEM[case["dtype"]]
        there = 1.0 - case["dropped"]
        ids = 4 * (2 * t * k + case["experts"] + 1)
        rows, tokens = item * t * k * d * there, item * t * d
        moved = ids + (tokens + item * t * k * d) + (rows + 4 * t * k + tokens)
        if op == "route":
            return {"bytes": moved, "flops": 2.0 * t * k * d * there}
        # dispatch's gradient reads the rows; combine's reads the tokens and y, writes dy and dw
        moved += (rows + tokens) + (tokens + item * t * k * d + 4 * t * k)
        return {"bytes": moved, "flops": 6.0 * t * k * d * there}
    b, t, s, hkv, block = (case[x] for x in ("b", "t", "s", "hkv", "block"))
    n = -(-s // block)
    if op == "select":
        return {"bytes": 4.0 * b * t * hkv * (n + case["count"]), "flops": 0.0}
    hq, d, item = case["hq"], case["d"], ITEM[case["dtype"]]
    if op == "score":
        bytes_ = item * b * t * hq * d + 4.0 * b * n * hkv * d + 4.0 * b * t * hkv * n
        flops = 2.0 * b * t * hkv * n * d
        if case["means"]:
            bytes_ += item * b * s * hkv * d + 4.0 * b * n * hkv * d
            flops += b * s * hkv * d
        return {"bytes": bytes_, "flops": flops}
    pairs = _pairs(case) * b * hq
    keys = min(s * (5 / 8 if case["ragged"] else 1), t * case["count"] * block)
    bytes_ = item * d * b * (2 * t * hq + 2 * keys * hkv) + 4.0 * b * t * hkv * case["count"]
    if op == "attend":
        return {"bytes": bytes_, "flops": 4.0 * d * pairs}
    # out and dout read, dq, dk, dv written
    bytes_ += item * d * b * (3 * t * hq + 2 * s * hkv + 2 * s * hkv)
    return {"bytes": bytes_, "flops": 14.0 * d * pairs}


# ---- the definition, in 64 bits ------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "select":
        return None
    if op in ("route", "route_train"):
        return _exact_route(state, case)
    if op == "score":
        return _exact_score(state, case)
    grads = op == "train"
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    g = hq // hkv
    wide = {x: state[x].detach().double() for x in ("q", "k", "v")}
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device=DEVICE)
    given = {x: torch.zeros_like(wide[x]) for x in wide}
    place = torch.arange(case["s"], device=DEVICE)
    last = state["lengths"].tolist() if state["lengths"] is not None else [case["s"]] * b
    step = max(1, (1 << 28) // (case["s"] * g))
    for i in range(b):
        for h in range(hkv):
            k, v = (wide[x][i, :, h].contiguous() for x in "kv")
            for t0 in range(0, t, step):
                rows = slice(t0, min(t, t0 + step))
                q = wide["q"][i, rows, h * g:h * g + g]
                at = last[i] - t + torch.arange(rows.start, rows.stop, device=DEVICE)
                ids = state["blocks"][i, rows, h]
                listed_ = torch.zeros(len(at), -(-case["s"] // case["block"]) + 1, device=DEVICE)
                listed_.scatter_(1, torch.where(ids < 0, listed_.shape[1] - 1, ids.long()), 1.0)
                listed_[:, -1] = 0.0
                see = (listed_[:, place // case["block"]] > 0) & (place <= at[:, None])
                x = (q @ k.T.contiguous()) / math.sqrt(d)
                x = torch.where(see[:, None], x, torch.full_like(x, -INF))
                lse = torch.logsumexp(x, -1, keepdim=True)
                p = torch.where(see[:, None], torch.exp(x - lse), torch.zeros_like(x))
                out[i, rows, h * g:h * g + g] = o = p @ v
                if grads:
                    do = state["dout"][i, rows, h * g:h * g + g].double()
                    ds = p * (do @ v.T.contiguous() - (do * o).sum(-1, keepdim=True))
                    ds = ds / math.sqrt(d)
                    given["q"][i, rows, h * g:h * g + g] = ds @ k
                    flat = ds.flatten(0, 1).T.contiguous()
                    given["k"][i, :, h] += flat @ q.flatten(0, 1)
                    given["v"][i, :, h] += p.flatten(0, 1).T.contiguous() @ do.flatten(0, 1)
    return (out, given["q"], given["k"], given["v"]) if grads else out


def _exact_score(state, case):
    b, s, hq, hkv, block = (case[x] for x in ("b", "s", "hq", "hkv", "block"))
    last = state["lengths"].tolist() if state["lengths"] is not None else [s] * b
    q, means = state["q"].double(), state["means"].double()
    scores = torch.full((b, case["t"], hkv, means.shape[1]), -INF, dtype=torch.float64,
                        device=DEVICE)
    at = torch.arange(case["t"], device=DEVICE) - case["t"]
    first = torch.arange(means.shape[1], device=DEVICE) * block
    for i in range(b):
        for h in range(hkv):
            heads = q[i, :, h * (hq // hkv):(h + 1) * (hq // hkv)].sum(1)
            x = heads @ means[i, :, h].T.contiguous() / math.sqrt(case["d"])
            scores[i, :, h] = torch.where(first <= (at + last[i])[:, None], x, -INF)
    if not case["means"]:
        return scores
    mean = torch.zeros(means.shape, dtype=torch.float64, device=DEVICE)
    for i in range(b):
        for j in range(-(-last[i] // block)):
            mean[i, j] = state["k"][i, j * block:min(last[i], (j + 1) * block)].double().mean(0)
    return mean, scores


def _exact_route(state, case):
    t, k, d = case["tokens"], case["k"], case["d"]
    expert = state["experts"].cpu().numpy().reshape(-1)
    there = expert >= 0
    entries = sorted(there.nonzero()[0].tolist(), key=lambda n: (expert[n], n))
    entries = torch.tensor(entries, dtype=torch.long, device=DEVICE)
    token, held = entries // k, len(entries)
    w = state["weights"].detach().double().flatten()[entries]
    y = state["y"].detach()[:held].double()

    def wide(rows, size):
        full = torch.zeros(size, d, dtype=torch.float64, device=DEVICE)
        full[:held] = rows
        return full

    xs = wide(state["x"].detach().double()[token], t * k)
    out = torch.zeros(t, d, dtype=torch.float64, device=DEVICE)
    out.index_add_(0, token, y * w[:, None])
    if case["op"] == "route":
        return None, None, xs, out
    dx = torch.zeros_like(out).index_add_(0, token, state["dxs"][:held].double())
    do = state["dout"].double()[token]
    dw = torch.zeros(t * k, dtype=torch.float64, device=DEVICE)
    dw[entries] = (do * y).sum(-1)
    return None, None, xs, out, dx, wide(do * w[:, None], t * k), dw.view(t, k)
