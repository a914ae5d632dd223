"""Workloads of the vocabulary operators: embedding lookup and its gradient,
cross-entropy loss and its gradient, and the rules that edit logits before a
token is chosen (penalties for repeated tokens, biases, grammar masks).

``listed()`` gives the workloads, ``prepare`` their inputs on the GPU,
``run`` one pass (the plain torch form, or with ``own`` the framework's
operators), ``exact`` the same results from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
#: logits + gradient of the largest listed workload: no drawn one moves more bytes
MOST_BYTES = 2 * 8192 * 128000 * 2


def listed():
    return [
        # the lookup of one decoding step: one token from each of 64 sequences
        dict(name="lookup, one step", op="lookup", tokens=64, vocab=32000, dim=1024, dtype="bf16", scale=1.0),
        # the lookup of a training batch, rows scaled by sqrt(dim)
        dict(name="lookup, batch", op="lookup", tokens=32768, vocab=128000, dim=4096, dtype="bf16", scale=64.0),
        # the gradient of a small f32 model with rows that are no multiple of 16 bytes
        dict(name="embedding grad, small odd", op="lookup_grad", tokens=500, vocab=8000, dim=511, dtype="f32", scale=1.0),
        # the gradient of a large vocabulary: most rows get no token and are written as zeros
        dict(name="embedding grad, wide vocab", op="lookup_grad", tokens=16384, vocab=128000, dim=2048, dtype="bf16", scale=45.25),
        # the gradient of a long batch: a few tokens make up much of it
        dict(name="embedding grad, many tokens", op="lookup_grad", tokens=65536, vocab=32000, dim=1024, dtype="f32", scale=1.0),
        # loss and gradient of a character-sized model: latency counts
        dict(name="loss+grad, small", op="loss_grad", rows=64, vocab=1000, dtype="f32", reduction="mean", smoothing=0.0, z=0.0),
        # loss and gradient of a training batch over a large vocabulary
        dict(name="loss+grad, batch", op="loss_grad", rows=8192, vocab=128000, dtype="bf16", reduction="mean", smoothing=0.0, z=0.0),
        # per-token losses with label smoothing and a log-sum-exp penalty, scaled gradients in f16, rows that start unaligned
        dict(name="loss+grad, odd smoothed", op="loss_grad", rows=2048, vocab=50021, dtype="f16", reduction="none", smoothing=0.1, z=1e-4),
        # per-token losses alone: evaluation of a model
        dict(name="loss, evaluation", op="loss", rows=4096, vocab=32000, dtype="f32", reduction="none", smoothing=0.0, z=0.0),
        # the logit rules of one sequence with a short history
        dict(name="logit rules, one row", op="rules", rows=1, vocab=32000, history=200, biases=4, dtype="f32", grammar=True),
        # a serving batch with prompts of some thousand tokens
        dict(name="logit rules, batch", op="rules", rows=64, vocab=128000, history=4096, biases=32, dtype="bf16", grammar=True),
        # a large batch with long contexts and an odd vocabulary
        dict(name="logit rules, long odd", op="rules", rows=384, vocab=50021, history=32768, biases=300, dtype="f32", grammar=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["lookup", "lookup_grad", "loss_grad", "loss", "rules"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        if op in ("lookup", "lookup_grad"):
            case = dict(op=op, tokens=_log(rng, 1, 65536), vocab=_log(rng, 256, 200000), dim=_log(rng, 64, 8192), dtype=dtype,
                        scale=rng.choice([1.0, 8.0, 45.25]))
        elif op in ("loss", "loss_grad"):
            case = dict(op=op, rows=_log(rng, 1, 16384), vocab=_log(rng, 256, 200000), dtype=dtype,
                        reduction=rng.choice(["mean", "sum", "none"]), smoothing=rng.choice([0.0, 0.1]), z=rng.choice([0.0, 1e-4]))
        else:
            case = dict(op=op, rows=_log(rng, 1, 512), vocab=_log(rng, 256, 200000), history=_log(rng, 1, 32768),
                        biases=_log(rng, 1, 300), dtype=dtype, grammar=rng.random() < 0.5)
        if work(case)["bytes"] <= MOST_BYTES:
            return case


def _distinct(tokens, vocab):
    """Expected number of distinct ids among `tokens` draws of _text_ids."""
    v = np.arange(1, vocab + 1, dtype=np.float64)
    p = np.log1p(1.0 / v) / math.log(vocab + 1)
    return float(np.sum(-np.expm1(tokens * np.log1p(-p))))


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "lookup":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        return {"bytes": 4 * n + s * d * (_distinct(n, v) + n), "flops": n * d}
    if case["op"] == "lookup_grad":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        return {"bytes": 4 * n + s * d * (n + v), "flops": n * d}
    if case["op"] == "rules":
        b, v = case["rows"], case["vocab"]
        side = 4 * (case["history"] * 3 // 4 + 2 * case["biases"] + 5)  # lengths are 3/4 of the buffer on average
        return {"bytes": b * (2 * s * v + (v / 8 if case["grammar"] else 0) + side), "flops": 4 * b * v}
    n, v = case["rows"], case["vocab"]
    outs = 4 * (n if case["reduction"] == "none" else 1)
    if case["op"] == "loss":
        return {"bytes": n * (s * v + 4) + outs, "flops": 4 * n * v}
    return {"bytes": n * (2 * s * v + 4) + outs, "flops": 8 * n * v}


def _text_ids(shape, vocab, g):
    """Token ids with the frequencies of text: P(id) ~ log(1 + 1 / (id + 1)), about 1 / rank."""
    u = torch.rand(shape, device="cuda", generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1.0).floor().clamp_(0, vocab - 1).to(torch.int32)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = {}
    if case["op"] == "lookup":
        s["table"] = torch.randn(case["vocab"], case["dim"], device="cuda", generator=g, dtype=t)
        s["ids"] = _text_ids((case["tokens"],), case["vocab"], g)
    elif case["op"] == "lookup_grad":
        s["table"] = torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=t)
        s["ids"] = _text_ids((case["tokens"],), case["vocab"], g)
        s["dy"] = torch.randn(case["tokens"], case["dim"], device="cuda", generator=g, dtype=t)
    elif case["op"] in ("loss", "loss_grad"):
        n, v = case["rows"], case["vocab"]
        targets = _text_ids((n,), v, g)
        logits = torch.randn(n, v, device="cuda", generator=g, dtype=t).mul_(2.5)
        right = torch.rand(n, device="cuda", generator=g) * 12.0  # the model has learnt some of its targets
        at = torch.arange(n, device="cuda")
        logits[at, targets.long()] += right.to(t)
        s["logits"] = logits
        s["targets"] = torch.where(torch.rand(n, device="cuda", generator=g) < 0.05, -100, targets)  # padding
        s["seed"] = None
        if case["op"] == "loss_grad" and case["reduction"] != "mean":  # per-token weights / a loss scale, as f16 gradients need
            shape = (n,) if case["reduction"] == "none" else ()
            s["seed"] = 64.0 * (0.5 + torch.rand(shape, device="cuda", generator=g))
    else:
        b, v, h, k = case["rows"], case["vocab"], case["history"], case["biases"]
        s["logits"] = torch.randn(b, v, device="cuda", generator=g, dtype=t).mul_(3.0)
        s["tokens"] = _text_ids((b, h), v, g)
        # sequences fill half of the buffer or more; a third of a sequence is its prompt
        s["lengths"] = torch.randint(h // 2, h + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
        s["prompt_lengths"] = s["lengths"] // 3
        s["repetition"] = 1.0 + 0.5 * torch.rand(b, device="cuda", generator=g)
        s["presence"] = torch.rand(b, device="cuda", generator=g)
        s["frequency"] = 0.5 * torch.rand(b, device="cuda", generator=g)
        s["bias_tokens"] = torch.randint(0, v, (b, k), device="cuda", generator=g, dtype=torch.int32)
        s["bias"] = 5.0 * torch.randn(b, k, device="cuda", generator=g)
        s["allowed"] = None
        if case["grammar"]:  # from nearly everything to a handful of tokens
            words = (b, -(-v // 32))
            bits = [torch.randint(-2 ** 31, 2 ** 31, words, device="cuda", generator=g, dtype=torch.int32) for _ in range(4)]
            few = (torch.arange(b, device="cuda") % 2 == 1)[:, None]
            s["allowed"] = torch.where(few, bits[0] & bits[1] & bits[2] & bits[3], bits[0] | bits[1] | bits[2] | bits[3])
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        import fugatensor_b200 as ft
        kinds = {torch.float32: ft.fp32, torch.float16: ft.fp16, torch.bfloat16: ft.bf16, torch.int32: ft.int32}
        state = {k: None if v is None else ft.tensor(v, dtype=kinds[v.dtype]) for k, v in state.items()}
    return {**state, "case": case}


def run(state):
    case = state["case"]
    form = _own if own else _plain
    return form[case["op"]](state, case)


# ------------------------------------------------------- the framework ---
def _own_lookup(s, case):
    import fugatensor_b200 as ft
    import fugatensor_b200.nn.functional as F
    return ft.evaluate(F.embedding(s["table"], s["ids"], scale=case["scale"])).torch()


def _own_lookup_grad(s, case):
    import fugatensor_b200 as ft
    import fugatensor_b200.nn.functional as F
    y = F.embedding(s["table"], s["ids"], scale=case["scale"])
    return ft.evaluate(ft.grad(y, s["table"], seed=s["dy"])).torch()


def _own_loss(s, case):
    import fugatensor_b200 as ft
    import fugatensor_b200.nn.functional as F
    loss = F.cross_entropy(s["logits"], s["targets"], label_smoothing=case["smoothing"], z_loss=case["z"],
                           reduction=case["reduction"])
    return ft.evaluate(loss).torch()


def _own_loss_grad(s, case):
    import fugatensor_b200 as ft
    import fugatensor_b200.nn.functional as F
    loss = F.cross_entropy(s["logits"], s["targets"], label_smoothing=case["smoothing"], z_loss=case["z"],
                           reduction=case["reduction"])
    dlogits = ft.grad(loss, s["logits"], seed=s["seed"])
    ft.evaluate(loss, dlogits)
    return {"loss": loss.torch(), "dlogits": dlogits.torch()}


def _own_rules(s, case):
    import fugatensor_b200 as ft
    import fugatensor_b200.nn.functional as F
    out = F.adjust_logits(s["logits"], s["tokens"], s["lengths"], prompt_lengths=s["prompt_lengths"],
                          repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                          bias_tokens=s["bias_tokens"], bias=s["bias"], allowed=s["allowed"])
    return ft.evaluate(out).torch()


_own = {"lookup": _own_lookup, "lookup_grad": _own_lookup_grad, "loss": _own_loss, "loss_grad": _own_loss_grad, "rules": _own_rules}


# --------------------------------------------------------- plain forms ---
def _plain_lookup(s, case):
    return (s["table"][s["ids"].long()].float() * case["scale"]).to(s["table"].dtype)


def _plain_lookup_grad(s, case):
    acc = torch.zeros(s["table"].shape, device="cuda", dtype=torch.float32)
    acc.index_add_(0, s["ids"].long(), s["dy"].float())
    return (acc * case["scale"]).to(s["table"].dtype)


def _plain_row_losses(s, case):
    x, t, v = s["logits"].float(), s["targets"].long(), case["vocab"]
    counts = t >= 0
    at = torch.where(counts, t, 0)[:, None]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = (m + torch.log(total))[:, 0]
    loss = lse - (1.0 - case["smoothing"]) * x.gather(1, at)[:, 0]
    if case["smoothing"]:
        loss = loss - case["smoothing"] / v * x.sum(1)
    if case["z"]:
        loss = loss + case["z"] * lse * lse
    return torch.where(counts, loss, 0.0), lse, e, total, at, counts


def _reduced(loss, counts, reduction):
    if reduction == "none":
        return loss
    return loss.sum() if reduction == "sum" else loss.sum() / counts.sum().clamp(min=1)


def _plain_loss(s, case):
    loss, _, _, _, _, counts = _plain_row_losses(s, case)
    return _reduced(loss, counts, case["reduction"])


def _plain_loss_grad(s, case):
    loss, lse, e, total, at, counts = _plain_row_losses(s, case)
    d = e / total
    if case["z"]:
        d = d * (1.0 + 2.0 * case["z"] * lse)[:, None]
    if case["smoothing"]:
        d = d - case["smoothing"] / case["vocab"]
    d.scatter_add_(1, at, torch.full_like(at, -(1.0 - case["smoothing"]), dtype=torch.float32))
    g = counts.float() if s["seed"] is None else counts.float() * s["seed"]
    if case["reduction"] == "mean":
        g = g / counts.sum().clamp(min=1)
    return {"loss": _reduced(loss, counts, case["reduction"]), "dlogits": (d * g[:, None]).to(s["logits"].dtype)}


def _plain_rules(s, case):
    x, v = s["logits"].float(), case["vocab"]
    at = torch.arange(case["history"], device="cuda")[None, :]
    told = (at < s["prompt_lengths"][:, None]).float()
    made = ((at >= s["prompt_lengths"][:, None]) & (at < s["lengths"][:, None])).float()
    ids = s["tokens"].long()
    prompt = torch.zeros_like(x).scatter_add_(1, ids, told)
    count = torch.zeros_like(x).scatter_add_(1, ids, made)
    r = s["repetition"][:, None]
    x = torch.where(prompt + count > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    x = x + torch.zeros_like(x).scatter_add_(1, s["bias_tokens"].long(), s["bias"])
    if s["allowed"] is not None:
        ids = torch.arange(v, device="cuda")
        x = torch.where(((s["allowed"][:, ids >> 5] >> (ids & 31)) & 1) != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


_plain = {"lookup": _plain_lookup, "lookup_grad": _plain_lookup_grad, "loss": _plain_loss, "loss_grad": _plain_loss_grad,
          "rules": _plain_rules}


# ------------------------------------------------------ 64-bit results ---
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "lookup":
        return torch.index_select(s["table"], 0, s["ids"]).double() * case["scale"]
    if case["op"] == "lookup_grad":
        # running sums over the tokens in sorted order, differenced at each id's end
        order = torch.argsort(s["ids"], stable=True)
        ends = torch.searchsorted(s["ids"][order].contiguous(), torch.arange(-1, case["vocab"], device="cuda", dtype=torch.int32), right=True)
        out = torch.empty(case["vocab"], case["dim"], device="cuda", dtype=torch.float64)
        for c in range(0, case["dim"], 256):
            part = s["dy"][:, c:c + 256].double()[order]
            run_ = torch.cat([torch.zeros_like(part[:1]), torch.cumsum(part, 0)])
            out[:, c:c + 256] = (run_[ends[1:]] - run_[ends[:-1]]) * case["scale"]
        out[ends[1:] == ends[:-1]] = 0.0
        return out
    if case["op"] == "rules":
        return _exact_rules(s, case)
    return _exact_loss(s, case)


def _exact_loss(s, case):
    n, v, eps, z = case["rows"], case["vocab"], case["smoothing"], case["z"]
    counted = s["targets"] != -100
    rows = torch.zeros(n, device="cuda", dtype=torch.float64)
    grads = torch.empty(n, v, device="cuda", dtype=torch.float64) if case["op"] == "loss_grad" else None
    weight = counted.double()
    if s["seed"] is not None:
        weight = weight * s["seed"].double()
    if case["reduction"] == "mean":
        weight = weight / max(1, int(counted.sum()))
    for i in range(0, n, 256):
        x = s["logits"][i:i + 256].double()
        want = torch.full_like(x, eps / v)  # the smoothed target distribution
        pick = counted[i:i + 256].nonzero()[:, 0]
        want[pick, s["targets"][i:i + 256][pick].long()] += 1.0 - eps
        lse = torch.logsumexp(x, 1)
        rows[i:i + 256] = torch.where(counted[i:i + 256], lse - (want * x).sum(1) + z * lse ** 2, 0.0)
        if grads is not None:
            p = torch.softmax(x, 1)
            grads[i:i + 256] = weight[i:i + 256, None] * (p + 2.0 * z * lse[:, None] * p - want)
    total = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / max(1, int(counted.sum()))}[case["reduction"]]
    return total if grads is None else {"loss": total, "dlogits": grads}


def _exact_rules(s, case):
    v, h = case["vocab"], case["history"]
    out = torch.empty(case["rows"], v, device="cuda", dtype=torch.float64)
    for i in range(case["rows"]):
        n, p = int(s["lengths"][i]), int(s["prompt_lengths"][i])
        line = s["tokens"][i, :n].long()
        seen, count = torch.bincount(line, minlength=v), torch.bincount(line[p:], minlength=v)
        x = s["logits"][i].double()
        r, f, a = (float(s[k][i]) for k in ("repetition", "frequency", "presence"))
        x = torch.where(seen > 0, torch.minimum(x, x * 0) * r + torch.maximum(x, x * 0) / r, x)
        x -= f * count + a * (count > 0)
        x += torch.bincount(s["bias_tokens"][i].long(), weights=s["bias"][i].double(), minlength=v)
        if s["allowed"] is not None:
            word = s["allowed"][i].cpu().numpy().astype("<i4").view(np.uint8)
            bits = torch.from_numpy(np.unpackbits(word, bitorder="little")[:v].astype(bool)).cuda()
            x[~bits] = -math.inf
        out[i] = x
    return out
