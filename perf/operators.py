"""The two ends of a language model's training step: tokens to hidden states, logits to losses, and both gradients.

Kinds of case, each one call (or one forward and one backward call) of ``terapipe_b200.ops.functional``:

* ``embed``:       rows of the embedding table for a batch of tokens, scaled.
* ``embed_grad``:  the table's fp32 gradient, written whole (rows of absent tokens are zero).  With ``shards`` > 1 the
  table is one tensor-parallel rank's part of the vocabulary: other tokens contribute nothing.
* ``distill``:     loss against a teacher's top logits, alone or mixed with the labels' cross entropy.
* ``ce``:          cross entropy.

The last two in three forms: ``train`` (loss and gradient in one pass), ``eval`` (loss only), ``split`` (forward, then
backward with a gradient of every row's loss, as an autograd graph calls them).

Tokens are batch-first ``[batch, seq]`` and activations sequence-first, so ids and labels are transposed views.
"""
import math

import torch

own = False

_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_IDS = {"int32": torch.int32, "int64": torch.int64}
_IGNORE = -100


def _embed(name, kind, seq, batch, vocab, hidden, dtype, ids="int64", shards=1, padding=False):
    return {"name": name, "kind": kind, "seq": seq, "batch": batch, "vocab": vocab, "hidden": hidden,
            "dtype": dtype, "ids": ids, "shards": shards, "padding": padding}


def _loss(name, kind, form, seq, batch, vocab, dtype, top=0, temperature=1.0, teacher_weight=0.0, ids="int64",
          teacher="fp32", unused=0):
    return {"name": name, "kind": kind, "form": form, "seq": seq, "batch": batch, "vocab": vocab, "dtype": dtype,
            "top": top, "temperature": temperature, "teacher_weight": teacher_weight, "ids": ids, "teacher": teacher,
            "unused": unused}


def listed():
    return [
        # one token slice of a pipeline schedule enters the first stage of a 768-wide model: a latency
        _embed("embed slice", "embed", 128, 1, 50257, 768, "fp16"),
        # all tokens of a step of the 2048-wide model
        _embed("embed step", "embed", 2048, 8, 50257, 2048, "bf16", ids="int32"),
        # a slice's tokens against one of eight shards of the vocabulary
        _embed("embed grad shard", "embed_grad", 128, 2, 50304, 1024, "fp16", shards=8),
        # ragged batch of the 1600-wide model: an odd sequence length, an odd vocabulary
        _embed("embed grad ragged", "embed_grad", 1021, 5, 50257, 1600, "bf16", ids="int32", padding=True),
        # a step of the 2048-wide model
        _embed("embed grad step", "embed_grad", 2048, 8, 50304, 2048, "bf16"),
        # the largest batch of its latency table, with a large vocabulary
        _embed("embed grad large", "embed_grad", 2048, 72, 131072, 2048, "fp16", padding=True),
        # a handful of tokens (online distillation of a short answer): a latency
        _loss("distill few", "distill", "train", 7, 1, 32000, "bf16", top=16, temperature=2.0, teacher_weight=1.0),
        # one slice of a batch, mixed with the labels' term: two softmaxes of different temperature a row
        _loss("distill mixed", "distill", "train", 256, 4, 50257, "fp16", top=64, temperature=2.0, teacher_weight=0.5,
              ids="int32", teacher="fp16"),
        # a whole batch against a large vocabulary, the teacher's term alone
        _loss("distill large", "distill", "train", 2048, 4, 131072, "bf16", top=128, temperature=1.0,
              teacher_weight=1.0, ids="int32", teacher="bf16"),
        # fp32 logits as the matrix product can leave them, forward and backward as separate calls
        _loss("distill split fp32", "distill", "split", 409, 5, 32000, "fp32", top=33, temperature=3.0,
              teacher_weight=0.7),
        # a step's cross entropy; 47 columns of the vocabulary are padding, masked with -inf
        _loss("ce step", "ce", "train", 2048, 8, 50304, "bf16", unused=47),
        # evaluation of a small batch
        _loss("ce eval", "ce", "eval", 128, 1, 50257, "fp16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_MOST_LOGIT_BYTES = 2048 * 4 * 131072 * 2
_MOST_TABLE_BYTES = 131072 * 2048 * 4


def draw(rng):
    kind = rng.choice(("embed", "embed_grad", "embed_grad", "distill", "distill", "ce"))
    vocab = rng.choice((_log_int(rng, 1000, 131072), 50257, 50304, 32000))
    batch = rng.randint(1, 8)
    ids = rng.choice(("int32", "int64"))
    if kind.startswith("embed"):
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        hidden = rng.choice((256, 768, 1024, 1280, 1536, 1600, 1920, 2048, 2304, 4096, _log_int(rng, 64, 4096)))
        seq = _log_int(rng, 1, 8192)
        shards = rng.choice((1, 1, 1, 2, 4, 8))
        vocab -= vocab % shards
        while vocab // shards * hidden * 4 > _MOST_TABLE_BYTES:
            hidden //= 2
        while seq * batch * hidden * 4 > _MOST_TABLE_BYTES:
            seq //= 2
        case = _embed("", kind, seq, batch, vocab, hidden, dtype, ids, shards if kind == "embed_grad" else 1,
                      kind == "embed_grad" and rng.random() < 0.5)
    else:
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        form = rng.choice(("train", "train", "eval", "split"))
        seq = _log_int(rng, 1, 4096)
        es = 4 if dtype == "fp32" else 2
        while seq * batch * vocab * es > _MOST_LOGIT_BYTES // 2:
            seq = max(1, seq // 2)
        unused = rng.choice((0, 0, rng.randint(1, 64)))
        if kind == "ce":
            case = _loss("", kind, form, seq, batch, vocab, dtype, ids=ids, unused=unused)
        else:
            case = _loss("", kind, form, seq, batch, vocab, dtype, _log_int(rng, 1, 256),
                         rng.choice((1.0, 2.0, 4.0, round(rng.uniform(0.5, 5.0), 2))),
                         rng.choice((1.0, 0.5, round(rng.uniform(0.1, 0.9), 2))), ids,
                         rng.choice(("fp16", "bf16", "fp32")), unused)
    del case["name"]
    return case


# ------------------------------------------------------------------------------- preparation
def _tokens(case, g):
    """``[seq, batch]`` ids (a transposed view).  A token's frequency falls as one over its rank, as in text: rank r has the
    probability log((r + 2) / (r + 1)) / log(vocab + 1).  Ranks are spread over the vocabulary."""
    vocab = case["vocab"]
    u = torch.rand(case["batch"], case["seq"], device="cuda", generator=g, dtype=torch.float64)
    rank = ((vocab + 1.0) ** u - 1.0).long().clamp_(0, vocab - 1)
    spread = torch.randperm(vocab, device="cuda", generator=g)
    return spread[rank].to(_IDS[case["ids"]]).t()


def _prepare_embed(case, g):
    dt, rows, hidden = _DTYPE[case["dtype"]], case["vocab"] // case["shards"], case["hidden"]
    tokens = _tokens(case, g)
    n = case["seq"] * case["batch"]
    if case["kind"] == "embed":
        weight = (torch.randn(rows, hidden, device="cuda", generator=g) * 0.02).to(dt)
        return {"kind": "embed", "ids": tokens, "weight": weight, "scale": math.sqrt(hidden),
                "out": torch.empty(n, hidden, device="cuda", dtype=dt)}
    dy = (torch.randn(n, hidden, device="cuda", generator=g) * 1e-2).to(dt)
    # (the most frequent ids are spread: any one of a few hundred tokens serves as the padding token)
    return {"kind": "embed_grad", "ids": tokens, "dy": dy, "scale": math.sqrt(hidden),
            "first_row": rows * (case["shards"] // 3), "padding_id": int(tokens[-1, -1]) if case["padding"] else None,
            "dweight": torch.empty(rows, hidden, device="cuda")}


def _prepare_loss(case, g):
    dt, vocab, top = _DTYPE[case["dtype"]], case["vocab"], case["top"]
    n = case["seq"] * case["batch"]
    logits = torch.empty(n, vocab, device="cuda", dtype=dt).normal_(0.0, 2.5, generator=g)
    if case["unused"]:
        logits[:, vocab - case["unused"]:] = -math.inf
    used = vocab - case["unused"]
    labels = _tokens(case, g)
    if used < vocab:
        labels = (labels.t() % used).t()
    # the model has learnt something: what it should answer stands out
    rows = torch.arange(n, device="cuda")
    logits[rows, labels.reshape(-1).long()] += 6.0
    # the end of every sequence is padding
    filled = case["seq"] - int(case["seq"] * 0.08)
    labels = labels.t().clone().t()
    labels[filled:] = _IGNORE
    s = {"kind": case["kind"], "form": case["form"], "logits": logits, "labels": labels,
         "loss": torch.empty(n, device="cuda"), "scale": 1024.0 / max(1, filled * case["batch"]),
         "dlogits": torch.empty_like(logits) if case["form"] != "eval" else None,
         "grad_loss": torch.rand(n, device="cuda", generator=g) if case["form"] == "split" else None}
    if case["kind"] == "distill":
        # distinct ids, one in each of `top` equal parts of the vocabulary, in the order of the teacher's logits
        part = max(1, used // top)
        top = min(top, used)
        ids = torch.arange(top, device="cuda") * part
        ids = ids + torch.randint(0, part, (n, top), device="cuda", generator=g)
        # turned by the row, so that the largest logits lie anywhere in the vocabulary
        ids = (ids + torch.randint(0, used, (n, 1), device="cuda", generator=g)) % used
        t = (torch.randn(n, top, device="cuda", generator=g) * 2.0 + 4.0).sort(-1, descending=True)[0]
        near = t + torch.randn(n, top, device="cuda", generator=g)
        logits.scatter_(1, ids, near.to(dt))
        # some answers of the teacher have fewer entries, and the padded end has none
        keep = torch.randint(max(1, top // 2), top + 1, (n, 1), device="cuda", generator=g)
        absent = torch.arange(top, device="cuda") >= keep
        absent[filled * case["batch"]:] = True
        s |= {"teacher_ids": ids.masked_fill(absent, -1).to(_IDS[case["ids"]]),
              "teacher_logits": t.masked_fill(absent, math.nan).to(_DTYPE[case["teacher"]]),
              "temperature": case["temperature"], "teacher_weight": case["teacher_weight"]}
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _prepare_embed(case, g) if case["kind"].startswith("embed") else _prepare_loss(case, g)


# ------------------------------------------------------------------------------- one pass
def _run_own(s):
    from terapipe_b200.ops import functional as F
    if s["kind"] == "embed":
        return F.embedding_fwd(s["ids"], s["weight"], s["out"], scale=s["scale"])
    if s["kind"] == "embed_grad":
        return F.embedding_bwd(s["ids"], s["dy"], s["dweight"], scale=s["scale"], first_row=s["first_row"],
                               padding_id=s["padding_id"], accumulate=False)
    if s["kind"] == "ce":
        if s["form"] == "train":
            loss, dlogits = F.cross_entropy_fwd_bwd(s["logits"], s["labels"], ignore_id=_IGNORE, grad_scale=s["scale"],
                                                    loss=s["loss"], dlogits=s["dlogits"])
            return {"loss": loss, "dlogits": dlogits}
        loss, stats = F.cross_entropy_fwd(s["logits"], s["labels"], ignore_id=_IGNORE, loss=s["loss"])
        if s["form"] == "eval":
            return {"loss": loss}
        dlogits = F.cross_entropy_bwd(s["logits"], stats, s["labels"], ignore_id=_IGNORE, grad_loss=s["grad_loss"],
                                      grad_scale=s["scale"], dlogits=s["dlogits"])
        return {"loss": loss, "dlogits": dlogits}
    how = {"temperature": s["temperature"], "teacher_weight": s["teacher_weight"], "ignore_id": _IGNORE}
    if s["form"] == "train":
        loss, dlogits = F.distill_fwd_bwd(s["logits"], s["teacher_ids"], s["teacher_logits"], s["labels"], **how,
                                          grad_scale=s["scale"], loss=s["loss"], dlogits=s["dlogits"])
        return {"loss": loss, "dlogits": dlogits}
    loss, stats = F.distill_fwd(s["logits"], s["teacher_ids"], s["teacher_logits"], s["labels"], **how, loss=s["loss"])
    if s["form"] == "eval":
        return {"loss": loss}
    dlogits = F.distill_bwd(s["logits"], stats, s["teacher_ids"], s["teacher_logits"], s["labels"], **how,
                            grad_loss=s["grad_loss"], grad_scale=s["scale"], dlogits=s["dlogits"])
    return {"loss": loss, "dlogits": dlogits}


def _run_plain_embed(s):
    ids = s["ids"].reshape(-1).long()
    if s["kind"] == "embed":
        w = s["weight"]
        return (w[ids].float() * s["scale"]).to(w.dtype)
    dy, rows = s["dy"].float(), s["dweight"].shape[0]
    local = ids - s["first_row"]
    out = (local < 0) | (local >= rows)
    if s["padding_id"] is not None:
        out = out | (ids == s["padding_id"])
    # tokens of no row of this table are added to a row behind it
    table = torch.zeros(rows + 1, dy.shape[1], device=dy.device)
    table.index_add_(0, local.masked_fill(out, rows), dy)
    return table[:rows] * s["scale"]


def _run_plain_loss(s):
    z, labels = s["logits"].float(), s["labels"].reshape(-1, 1).long()
    weight, temperature = s.get("teacher_weight", 0.0), s.get("temperature", 1.0)
    has = labels != _IGNORE
    at = labels.masked_fill(~has, 0)
    shifted = z - z.max(-1, keepdim=True)[0]
    e = shifted.exp()
    denom = e.sum(-1, keepdim=True)
    picked = shifted.gather(1, at)
    loss = (1 - weight) * (denom.log() - picked).masked_fill(~has, 0.0)
    if s["kind"] == "distill":
        ids, t = s["teacher_ids"].long(), s["teacher_logits"].float() / temperature
        absent = (ids < 0) | (ids >= z.shape[1])
        some = ~absent.all(-1, keepdim=True)
        t = t.masked_fill(absent, -math.inf)
        t = t - t.max(-1, keepdim=True)[0].masked_fill(~some, 0.0)
        p = t.exp()
        total = p.sum(-1, keepdim=True).masked_fill(~some, 1.0)
        p = p / total
        cool = shifted / temperature
        ec = cool.exp()
        denom_c = ec.sum(-1, keepdim=True)
        where = ids.masked_fill(absent, 0)
        # log p - log q of the present entries
        gap = (t - total.log()) - (cool.gather(1, where) - denom_c.log())
        kl = (p * gap).masked_fill(absent | (p == 0), 0.0).sum(-1, keepdim=True)
        loss = loss + weight * temperature ** 2 * kl
    loss = loss.squeeze(1)
    if s["form"] == "eval":
        return {"loss": loss}
    grad = (e / denom).scatter_add_(1, at, torch.full_like(picked, -1.0)) * ((1 - weight) * has)
    if s["kind"] == "distill":
        cold = (ec / denom_c).scatter_add_(1, where, -p.masked_fill(absent, 0.0))
        grad = grad + cold * (weight * temperature * some)
    grad = grad * s["scale"]
    if s["grad_loss"] is not None:
        grad = grad * s["grad_loss"].unsqueeze(1)
    return {"loss": loss, "dlogits": grad.to(s["logits"].dtype)}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain_embed(state) if state["kind"].startswith("embed") else _run_plain_loss(state)


# ------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definitions: rows picked one product at a time, gradients as sums over a one-hot matrix's columns (a
    sorted order and differences of running sums), losses through logarithms of probabilities."""
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return torch.nn.functional.embedding(s["ids"].reshape(-1).long(), s["weight"].double()) * s["scale"]
    if case["kind"] == "embed_grad":
        ids, rows = s["ids"].reshape(-1).long(), s["dweight"].shape[0]
        keep = (ids >= s["first_row"]) & (ids < s["first_row"] + rows)
        if s["padding_id"] is not None:
            keep &= ids != s["padding_id"]
        which = keep.nonzero().squeeze(1)
        table = torch.zeros(rows, case["hidden"], device="cuda", dtype=torch.float64)
        if len(which) == 0:
            return table
        order = torch.argsort(ids[which], stable=True)
        found, counts = torch.unique_consecutive(ids[which][order], return_counts=True)
        ends = counts.cumsum(0)
        for lo in range(0, case["hidden"], 256):      # columns by columns: running sums in 64 bits
            sums = s["dy"][which][order][:, lo:lo + 256].double().cumsum(0)
            upto = sums[ends - 1]
            table[found - s["first_row"], lo:lo + 256] = torch.cat([upto[:1], upto[1:] - upto[:-1]]) * s["scale"]
        return table
    n, vocab = s["logits"].shape
    weight, temperature = s.get("teacher_weight", 0.0), s.get("temperature", 1.0)
    labels = s["labels"].reshape(-1)
    loss = torch.zeros(n, device="cuda", dtype=torch.float64)
    grad = None if case["form"] == "eval" else torch.zeros(n, vocab, device="cuda", dtype=torch.float64)
    step = max(1, (1 << 27) // vocab)
    for lo in range(0, n, step):
        part = slice(lo, min(n, lo + step))
        z = s["logits"][part].double()
        at = torch.arange(z.shape[0], device="cuda")
        y = labels[part].long()
        real = y != _IGNORE
        log_s = torch.log_softmax(z, -1)
        loss[part] += torch.where(real, -(1 - weight) * log_s[at, y * real], 0.0)
        g = log_s.exp()
        g[at, y * real] -= 1.0
        g *= ((1 - weight) * real).unsqueeze(1)
        if case["kind"] == "distill":
            ids, t = s["teacher_ids"][part].long(), s["teacher_logits"][part].double()
            there = (ids >= 0) & (ids < vocab)
            some = there.any(-1)
            p = torch.where(there, t, -math.inf).div(temperature).softmax(-1)
            p = torch.where(there, p, 0.0)
            log_q = torch.log_softmax(z / temperature, -1)
            entropy = torch.special.xlogy(p, p).sum(-1)
            crossed = torch.where(p > 0, p * log_q.gather(1, ids * there), 0.0).sum(-1)
            loss[part] += weight * temperature ** 2 * torch.where(some, entropy - crossed, 0.0)
            q = log_q.exp().scatter_add(1, ids * there, -p)
            g += q * (weight * temperature * some).unsqueeze(1)
        if grad is not None:
            g *= s["scale"]
            grad[part] = g if s["grad_loss"] is None else g * s["grad_loss"][part].double().unsqueeze(1)
    return {"loss": loss} if grad is None else {"loss": loss, "dlogits": grad}


# ------------------------------------------------------------------------------- what it takes
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    n, vocab = case["seq"] * case["batch"], case["vocab"]
    id_bytes = 4 if case["ids"] == "int32" else 8
    if case["kind"] == "embed":
        # the rows of the tokens that occur, as many as are to be expected (see _tokens)
        r = torch.arange(vocab, dtype=torch.float64)
        p = torch.log((r + 2) / (r + 1)) / math.log(vocab + 1)
        distinct = float((1 - (1 - p) ** n).sum())
        return {"bytes": n * id_bytes + (distinct + n) * case["hidden"] * es, "flops": n * case["hidden"]}
    if case["kind"] == "embed_grad":
        rows, mine = vocab // case["shards"], n / case["shards"]
        return {"bytes": n * id_bytes + mine * case["hidden"] * es + rows * case["hidden"] * 4,
                "flops": mine * case["hidden"] + rows * case["hidden"]}
    # logits once forward and once more in a separate backward; their gradient once
    passes = {"eval": 1, "train": 2, "split": 3}[case["form"]]
    small = n * (id_bytes + 4) + n * case["top"] * (id_bytes + (4 if case["teacher"] == "fp32" else 2))
    softmaxes = 2 if case["kind"] == "distill" and case["teacher_weight"] < 1 else 1
    # difference, exponential and sum of each softmax, product and difference of its gradient
    per_logit = softmaxes * (3 if case["form"] == "eval" else 5)
    return {"bytes": n * vocab * es * passes + small, "flops": n * vocab * per_logit}
