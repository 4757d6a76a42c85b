"""The ends of a language model's training step, as timed cases: words to rows (`embed`, and `embed_train`
with the gradient of the table), rows to a loss over the vocabulary (`loss`, and `loss_train` with
the gradients of the rows and of the table), and the gradients' common norm and their clipping
(`clip`).

With `own` false, `run` computes a case in elementary torch operations in float32; with `own`
true it calls the framework's entry points.  Sizes are those of a case whatever the seed; the
seed draws the values, the words, the targets and which tokens are left out.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}

# The most elements of a table and of a batch's rows, and tokens x words x width of a loss, that a
# drawn case has (float32 products are an eighth as fast).
MAX_TABLE = 131072 * 4096
MAX_ROWS = 65536 * 4096
MAX_PRODUCTS = 8192 * 131072 * 2048
MAX_GRADS = 1 << 30
# Elements that gradients' places in the flat buffer of clipped ones are multiples of.
PLACE = 64


def listed():
    return [
        # Serving: one step's new tokens of a batch of sequences.  All latency.
        {"name": "embed_step", "op": "embed", "tokens": 48, "words": 32768, "d": 2048,
         "dtype": "bf16", "scaled": False, "out": 0.0},
        # A batch of prompts, with the scaled rows that some models start from.
        {"name": "embed_prompts", "op": "embed", "tokens": 65536, "words": 131072, "d": 4096,
         "dtype": "bf16", "scaled": True, "out": 0.0},
        # A training batch's rows and the table's gradient: few of the words occur, some often.
        {"name": "embed_train", "op": "embed_train", "tokens": 16384, "words": 65537, "d": 2048,
         "dtype": "bf16", "scaled": True, "out": 0.05},
        # The same at odd sizes in float32: more tokens than words, rows between 16-byte pieces.
        {"name": "embed_train_odd", "op": "embed_train", "tokens": 30001, "words": 10007, "d": 333,
         "dtype": "f32", "scaled": False, "out": 0.1},
        # How likely one given token is: a single row against the whole table.
        {"name": "loss_token", "op": "loss", "tokens": 1, "words": 131072, "d": 4096,
         "dtype": "bf16", "reduction": "none", "scaled": False, "out": 0.0},
        # Scoring a text, token by token, with an odd vocabulary.
        {"name": "loss_text", "op": "loss", "tokens": 1000, "words": 50001, "d": 1024,
         "dtype": "f16", "reduction": "none", "scaled": True, "out": 0.0},
        # A training step's loss over a large vocabulary with both gradients: the largest.
        {"name": "loss_train", "op": "loss_train", "tokens": 8192, "words": 131072, "d": 2048,
         "dtype": "bf16", "reduction": "mean", "scaled": False, "out": 0.02},
        # Tuning on answers: half of the tokens are prompt or padding and have no target.
        {"name": "loss_train_answers", "op": "loss_train", "tokens": 3001, "words": 32003,
         "d": 776, "dtype": "f16", "reduction": "mean", "scaled": False, "out": 0.5},
        # A small model in float32, with a weight for each token's loss.
        {"name": "loss_train_f32", "op": "loss_train", "tokens": 2048, "words": 16384, "d": 1024,
         "dtype": "f32", "reduction": "none", "scaled": True, "out": 0.0},
        # The gradients of a small layer before a step: all latency.
        {"name": "clip_layer", "op": "clip", "tensors": 14, "elements": 200_000, "dtype": "f32",
         "out_dtype": "f32"},
        # A model's gradients in bfloat16, clipped into the float32 ones that an optimiser reads.
        {"name": "clip_model", "op": "clip", "tensors": 290, "elements": 1 << 30, "dtype": "bf16",
         "out_dtype": "f32"},
        # Many odd tensors, of one element to millions.
        {"name": "clip_odd", "op": "clip", "tensors": 611, "elements": 120_000_001,
         "dtype": "f16", "out_dtype": "f16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embed", "embed_train", "embed_train", "loss", "loss_train", "loss_train",
                     "clip"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "clip":
        tensors = _log_int(rng, 1, 1000)
        return {"op": op, "tensors": tensors, "dtype": dtype,
                "elements": max(tensors, _log_int(rng, 100, MAX_GRADS // (1 + (dtype == "f32")))),
                "out_dtype": rng.choice((dtype, "f32"))}
    d = _log_int(rng, 16, 8192)
    if rng.random() < 0.75:
        d = -(-d // 8) * 8
    words = _log_int(rng, 100, 262144)
    scaled = rng.random() < 0.5
    if op in ("embed", "embed_train"):
        words = min(words, MAX_TABLE // d)
        tokens = min(_log_int(rng, 1, 262144), MAX_ROWS // d)
        return {"op": op, "tokens": tokens, "words": words, "d": d, "dtype": dtype,
                "scaled": scaled, "out": rng.choice((0.0, 0.1))}
    words = min(words, MAX_TABLE // d)
    most = MAX_PRODUCTS // (8 if dtype == "f32" else 1)
    tokens = max(1, min(_log_int(rng, 1, 16384), most // (words * d)))
    return {"op": op, "tokens": tokens, "words": words, "d": d, "dtype": dtype, "scaled": scaled,
            "reduction": rng.choice(("mean", "sum", "none")),
            "out": rng.choice((0.0, 0.0, 0.1, 0.6))}


# ---- inputs --------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=g)


def _words(g, case):
    """Words as texts have them: the n-th most frequent has a share of about 1 / n.  A share `out`
    is -1: padding, or a target that does not count."""
    n, words = case["tokens"], case["words"]
    u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
    rank = torch.exp(u * math.log(words + 1.0)).long().sub_(1).clamp_(0, words - 1)
    ids = torch.randperm(words, generator=g, device=DEVICE)[rank]
    if case["out"]:
        left = torch.rand(n, generator=g, device=DEVICE) < case["out"]
        ids = ids.masked_fill(left, -1)
    return ids


def _scale(case):
    """A factor of the rows (their width's root) or of the logits (its inverse); 1 else."""
    if not case["scaled"]:
        return 1.0
    return math.sqrt(case["d"]) if case["op"].startswith("embed") else 1.0 / math.sqrt(case["d"])


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "clip":
        return _prepare_clip(g, case)
    dtype, n, words, d = DTYPES[case["dtype"]], case["tokens"], case["words"], case["d"]
    state = {"case": case, "scale": _scale(case), "ids": _words(g, case)}
    if op in ("embed", "embed_train"):
        state["table"] = _normal(g, words, d, dtype=dtype).mul_(0.02)
        if op == "embed_train":
            state["table"].requires_grad_()
            state["dout"] = _normal(g, n, d, dtype=dtype).mul_(1e-2)
        return state
    # Rows lean towards their targets: some are all but certain, some at a loss.
    wide = 1.0 if case["scaled"] else d ** -0.5
    state["table"] = _normal(g, words, d, dtype=dtype).mul_(wide)
    sure = 15.0 * torch.rand(n, 1, generator=g, device=DEVICE) / (wide * wide * d)
    if case["scaled"]:
        sure *= math.sqrt(d)
    toward = state["table"][state["ids"].clamp(min=0)].float()
    state["x"] = (_normal(g, n, d) + sure * toward).to(dtype)
    if op == "loss_train":
        state |= {"x": state["x"].requires_grad_(), "table": state["table"].requires_grad_()}
        if case["reduction"] == "none":
            state["dloss"] = torch.rand(n, generator=g, device=DEVICE) / n
        else:  # (float16 steps scale their loss)
            size = 1024.0 if case["dtype"] == "f16" else 1.0
            state["dloss"] = torch.full((), size, device=DEVICE)
        if case["reduction"] == "sum":
            state["dloss"] /= n
    return state


def _sizes(case):
    """Elements of each tensor: a few large ones, many small, together `elements`."""
    n = case["tensors"]
    share = [(1.0 + (7 * i + 3) % 11) ** 3 if i % 3 else 0.01 + 0.001 * i for i in range(n)]
    part = (case["elements"] - n) / sum(share)
    sizes = [1 + int(part * x) for x in share]
    sizes[-1] += case["elements"] - sum(sizes)
    return sizes


def _places(sizes):
    """Where each tensor starts in the flat buffer, and its length."""
    at, places = 0, []
    for n in sizes:
        places.append(at)
        at += -(-n // PLACE) * PLACE
    return places, at


def _prepare_clip(g, case):
    sizes = _sizes(case)
    places, total = _places(sizes)
    dtype = DTYPES[case["dtype"]]
    # Matrices and vectors; their layers' gradients differ in size.
    grads = [_normal(g, *((n // 64, 64) if n % 64 == 0 else (n,)), dtype=dtype)
             .mul_(10.0 ** (-(i % 4))) for i, n in enumerate(sizes)]
    flat = torch.zeros(total, dtype=DTYPES[case["out_dtype"]], device=DEVICE)
    outs = [flat[at:at + x.numel()].view(x.shape) for at, x in zip(places, grads)]
    return {"case": case, "grads": grads, "flat": flat, "outs": outs, "places": places,
            "max_norm": 1.0}


# ---- one pass ------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(state, case):
    import nacho_amd

    op = case["op"]
    if op == "clip":
        norm = nacho_amd.gpu_clip_grad_norm(state["grads"], state["max_norm"], out=state["outs"])
        return norm, state["flat"]
    ids, table, scale = state["ids"], state["table"], state["scale"]
    if op in ("embed", "embed_train"):
        rows = nacho_amd.gpu_embedding(ids, table, scale=scale)
        if op == "embed":
            return rows
        return rows, *torch.autograd.grad(rows, table, state["dout"])
    loss = nacho_amd.gpu_linear_cross_entropy(state["x"], table, ids, scale=scale,
                                              reduction=case["reduction"])
    if op == "loss":
        return loss
    return loss, *torch.autograd.grad(loss, (state["x"], table), state["dloss"])


def _run_plain(state, case):
    op = case["op"]
    with torch.no_grad():
        if op == "clip":
            return _plain_clip(state, case)
        if op in ("embed", "embed_train"):
            return _plain_embed(state, case)
        return _plain_loss(state, case)


def _plain_clip(state, case):
    squares = [x.float().square().sum(dtype=torch.float64) for x in state["grads"]]
    norm = torch.sqrt(torch.stack(squares).sum())
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    gap = [(-x.numel()) % PLACE for x in state["grads"]]
    dtype = state["flat"].dtype
    flat = torch.cat([torch.nn.functional.pad((x.float() * factor).to(dtype).flatten(), (0, n))
                      for x, n in zip(state["grads"], gap)])
    return norm.float(), flat


def _plain_embed(state, case):
    ids, table, scale = state["ids"], state["table"], state["scale"]
    there = ids >= 0
    at = ids.clamp(min=0)
    rows = (table[at].float() * scale).masked_fill_(~there[:, None], 0.0).to(table.dtype)
    if case["op"] == "embed":
        return rows
    given = (state["dout"].float() * scale).masked_fill_(~there[:, None], 0.0)
    grad = torch.zeros(table.shape, device=DEVICE).index_add_(0, at, given)
    return rows, grad.to(table.dtype)


def _plain_loss(state, case):
    ids, scale = state["ids"], state["scale"]
    x, table = state["x"].float(), state["table"].float()
    there = ids >= 0
    at = ids.clamp(min=0)[:, None]
    logits = torch.matmul(x, table.t()).mul_(scale)
    mine = logits.gather(1, at)[:, 0]
    top = logits.amax(1, keepdim=True)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    each = (torch.log(total[:, 0]) + (top[:, 0] - mine)).masked_fill(~there, 0.0)
    count = there.sum().clamp(min=1)
    if case["reduction"] == "none":
        loss = each
    else:
        loss = each.sum(dtype=torch.float64)
        loss = (loss / count if case["reduction"] == "mean" else loss).float()
    if case["op"] == "loss":
        return loss
    part = state["dloss"] / count if case["reduction"] == "mean" else state["dloss"]
    part = (part * scale).expand(len(ids)).masked_fill(~there, 0.0)[:, None]
    p.div_(total)
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p.mul_(part)
    dx = torch.matmul(p, table)
    dtable = torch.matmul(p.t(), x)
    return loss, dx.to(state["x"].dtype), dtable.to(state["table"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------

def _distinct(case):
    """Words that occur, on average: the n-th one's share is about 1 / (n log(words + 1))."""
    held = case["tokens"] * (1.0 - case["out"])
    n = torch.arange(1, case["words"] + 1, dtype=torch.float64)
    share = torch.log1p(1.0 / n) / math.log(case["words"] + 1.0)
    return float((1.0 - torch.exp(held * torch.log1p(-share.clamp(max=1 - 1e-12)))).sum())


def work(case):
    op = case["op"]
    if op == "clip":
        n = case["elements"]
        # (the norm needs every gradient before the first is scaled: they are read for it alone)
        return {"bytes": float(n) * (ITEM[case["dtype"]] + ITEM[case["out_dtype"]]),
                "flops": 3.0 * n}
    item, n, words, d = ITEM[case["dtype"]], case["tokens"], case["words"], case["d"]
    held = n * (1.0 - case["out"])
    if op in ("embed", "embed_train"):
        moved = 8.0 * n + item * d * (min(held, _distinct(case)) + n)
        if op == "embed":
            return {"bytes": moved, "flops": held * d}
        return {"bytes": moved + item * d * (held + words), "flops": 3.0 * held * d}
    moved = 8.0 * n + item * d * (held + float(words))
    flops = 2.0 * held * words * d
    if op == "loss":
        return {"bytes": moved + 4.0 * n, "flops": flops}
    # the logits, and the products that give dx and dtable
    return {"bytes": moved + item * d * (n + float(words)), "flops": 3.0 * flops}


# ---- the definition, in 64 bits ------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "clip":
            return _exact_clip(state)
        if case["op"].startswith("embed"):
            return _exact_embed(state, case)
        return _exact_loss(state, case)


def _exact_clip(state):
    total = sum(float(torch.dot(x.flatten().double(), x.flatten().double()))
                for x in state["grads"])
    factor = min(1.0, state["max_norm"] / (math.sqrt(total) + 1e-6))
    flat = torch.zeros(state["flat"].shape, dtype=torch.float64, device=DEVICE)
    for at, x in zip(state["places"], state["grads"]):
        flat[at:at + x.numel()] = x.flatten().double() * factor
    return torch.tensor(math.sqrt(total), dtype=torch.float64), flat


def _exact_embed(state, case):
    ids, table = state["ids"], state["table"].detach()
    held = torch.nonzero(ids >= 0)[:, 0]
    rows = torch.zeros(len(ids), case["d"], dtype=torch.float64, device=DEVICE)
    rows[held] = table[ids[held]].double() * state["scale"]
    if case["op"] == "embed":
        return rows
    grad = torch.zeros(table.shape, dtype=torch.float64, device=DEVICE)
    grad.index_add_(0, ids[held], state["dout"][held].double())
    return rows, grad * state["scale"]


def _exact_loss(state, case):
    ids, scale = state["ids"], state["scale"]
    n, words, d = case["tokens"], case["words"], case["d"]
    grads = case["op"] == "loss_train"
    x, table = state["x"].detach().double(), state["table"].detach().double()
    held = torch.nonzero(ids >= 0)[:, 0]
    each = torch.zeros(n, dtype=torch.float64, device=DEVICE)
    dx = torch.zeros_like(x)
    dtable = torch.zeros_like(table) if grads else None
    if grads:
        part = state["dloss"].double()
        if case["reduction"] == "mean":
            part = part / max(1, len(held))
        part = part.expand(n)
    step = max(1, (1 << 28) // words)
    for rows in held.split(step):
        z = (x[rows] @ table.T) * scale
        lse = torch.logsumexp(z, 1)
        each[rows] = lse - z[torch.arange(len(rows), device=DEVICE), ids[rows]]
        if grads:
            z -= lse[:, None]
            z.exp_()
            z[torch.arange(len(rows), device=DEVICE), ids[rows]] -= 1.0
            z *= part[rows][:, None] * scale
            dx[rows] = z @ table
            dtable += z.T @ x[rows]
    loss = each
    if case["reduction"] != "none":
        loss = each.sum()
        if case["reduction"] == "mean":
            loss = loss / max(1, len(held))
    return (loss, dx, dtable) if grads else loss
