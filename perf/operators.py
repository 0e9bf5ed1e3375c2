"""Cases of the operators on output rows (speech_amd.logits): what they are run on, and their plain forms.

A row is the logits of one token over the vocabulary.  `pick` and `constrain` are the serving side (penalties for repeated
tokens, biases, grammar masks, then the token); `top` is what a teacher leaves of its rows; `distill` is a student's training
step on that.  `own` selects the framework's calls; without it every operator is computed in elementary torch operations."""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # one request's next token over a mid-sized word-piece vocabulary, a grammar and a few biased words
        _serve("pick_one", "pick", 1, 32000, "float32", 300, 8, True),
        # the letters of a batch of utterances (28 letters and the end): latency only
        _serve("pick_letters", "pick", 32, 29, "float32", 200, 0, True),
        # a full serving batch, odd vocabulary, long answers
        _serve("pick_batch", "pick", 64, 50021, "bfloat16", 2048, 64, True),
        # a few requests whose sampler wants the logits back
        _serve("constrain_few", "constrain", 16, 32000, "float16", 1000, 16, False),
        # many requests over a large vocabulary
        _serve("constrain_many", "constrain", 256, 131072, "float32", 4096, 128, True),
        # a teacher's frames of 32 utterances (498 frames each) over letters
        _top("top_letters", 15936, 29, 8, "float32", 1.0),
        # a teacher's tokens over word pieces
        _top("top_pieces", 4096, 32000, 64, "bfloat16", 2.0),
        # a handful of rows of a large odd vocabulary: one interactive request
        _top("top_few", 8, 131071, 100, "float32", 1.0),
        # a student's batch over letters: 32 utterances of 100 tokens
        _distill("distill_letters", 3200, 29, 8, "float32", 2.0, 0.5, True, False),
        # a student's batch over word pieces, soft and hard targets
        _distill("distill_pieces", 4096, 32000, 64, "bfloat16", 2.0, 0.7, True, False),
        # padded batch, odd vocabulary, the teacher's list alone
        _distill("distill_padded", 1000, 50021, 20, "float16", 1.0, 1.0, False, True),
        # a large vocabulary in 32 bits
        _distill("distill_large", 2048, 131072, 64, "float32", 2.0, 0.7, True, False),
    ]


def _serve(name, op, rows, vocab, dtype, history, biases, grammar):
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "history": history, "biases": biases,
            "grammar": grammar}


def _top(name, rows, vocab, k, dtype, temperature):
    return {"name": name, "op": "top", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temperature": temperature}


def _distill(name, rows, vocab, k, dtype, temperature, alpha, rest, padded):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temperature": temperature,
            "alpha": alpha, "rest": rest, "padded": padded}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pick", "constrain", "top", "distill"])
    vocab, dtype = _log(rng, 29, 131072), rng.choice(sorted(_TYPES))
    if op in ("pick", "constrain"):
        c = _serve("", op, _log(rng, 1, 256), vocab, dtype, _log(rng, 1, 4096), min(_log(rng, 1, 128), vocab) - 1,
                   rng.random() < 0.5)
    else:
        rows = _log(rng, 1, min(16384, (1 << 27) // vocab))
        k = min(_log(rng, 1, 100), vocab - 1)
        if op == "top":
            c = _top("", rows, vocab, k, dtype, rng.choice([1.0, 2.0]))
        else:
            c = _distill("", rows, vocab, k, dtype, rng.choice([1.0, 2.0, 4.0]), rng.choice([0.5, 0.7, 1.0]),
                         rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


def _rows(g, rows, vocab, dtype):
    """Logits as a trained model gives them: a wide bulk and a few tokens that stand out."""
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    x.mul_(1.7).sub_(2.0)
    u = torch.rand(rows, vocab, device="cuda", generator=g)
    share = min(0.25, 12.0 / vocab)
    x = torch.where(u < share, u * (8 / share) + 3, x)
    return x.to(_TYPES[dtype])


def _denom(case):
    """The loss is a mean over rows; in float16 it is scaled as such training has it, or small gradients would be lost."""
    return case["rows"] / (1024.0 if case["dtype"] == "float16" else 1.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, v = case["rows"], case["vocab"]
    s = {"case": case, "logits": _rows(g, n, v, case["dtype"])}

    def uniform(lo, hi, *shape):
        return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo

    if case["op"] in ("pick", "constrain"):
        # frequent tokens come again and again; requests are of different lengths
        s["history"] = (uniform(0, 1, n, case["history"]).pow(3) * v).long().clamp_(max=v - 1)
        s["lengths"] = torch.randint(case["history"] // 2, case["history"] + 1, (n,), device="cuda", generator=g).int()
        s["repetition"], s["presence"], s["frequency"] = uniform(1.0, 1.4, n), uniform(0, 0.5, n), uniform(0, 0.2, n)
        s["bias_ids"] = s["bias_values"] = s["mask"] = s["states"] = None
        if case["biases"]:
            order = torch.randperm(v, device="cuda", generator=g)  # the tokens of a row's biases differ
            at = torch.arange(case["biases"], device="cuda")[None] + 17 * torch.arange(n, device="cuda")[:, None]
            s["bias_ids"], s["bias_values"] = order[at % v], uniform(-4, 4, n, case["biases"])
        if case["grammar"]:
            words = torch.randint(-(1 << 31), 1 << 31, (24, (v + 31) // 32), device="cuda", generator=g)
            words[:, 0] |= 1  # a token is left in every state
            s["mask"] = words.int()
            s["states"] = torch.randint(-1, 24, (n,), device="cuda", generator=g).int()  # -1: a request without a grammar
    elif case["op"] == "distill":
        k = case["k"]
        teacher = s["logits"].float() + 0.7 * torch.randn(n, v, device="cuda", generator=g)
        s["values"], s["ids"] = torch.topk(teacher, k, dim=1)
        s["rest"] = None
        if case["rest"]:
            teacher.scatter_(1, s["ids"], -math.inf)
            s["rest"] = torch.logsumexp(teacher / case["temperature"], 1)
        del teacher
        s["targets"] = torch.randint(0, v, (n,), device="cuda", generator=g) if case["alpha"] < 1 else None
        s["weights"] = (uniform(0, 1, n) < 0.8).float() if case["padded"] else None
        s["logits"].requires_grad_(True)
    return s


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _run_own(s):
    from speech_amd import logits, ops
    c = s["case"]
    if c["op"] == "top":
        values, ids, rest = logits.top_logits(s["logits"], c["k"], temperature=c["temperature"])
        return {"values": values, "ids": ids, "rest": rest}
    if c["op"] == "distill":
        x = s["logits"]
        x.grad = None
        loss = logits.DistillLoss(temperature=c["temperature"], alpha=c["alpha"], denom=_denom(c))(
            x, s["values"], s["ids"], rest=s["rest"], targets=s["targets"], weights=s["weights"])
        ops.backward(loss)
        return {"loss": loss.detach(), "grad": x.grad}
    call = logits.pick if c["op"] == "pick" else logits.constrain
    out = call(s["logits"], history=s["history"], lengths=s["lengths"], repetition=s["repetition"], presence=s["presence"],
               frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"],
               states=s["states"])
    return {"tokens": out[0], "logp": out[1]} if c["op"] == "pick" else {"logits": out}


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _run_plain(s):
    with torch.no_grad():
        c = s["case"]
        if c["op"] == "top":
            return _plain_top(s["logits"], c["k"], c["temperature"])
        if c["op"] == "distill":
            return _plain_distill(s)
        x = _plain_constrain(s)
        if c["op"] == "constrain":
            return {"logits": x.to(s["logits"].dtype)}
        top = x.max(1, keepdim=True).values
        place = torch.arange(x.shape[1], device=x.device)
        return {"tokens": torch.where(x == top, place, x.shape[1]).min(1).values, "logp": -(x - top).exp().sum(1).log()}


def _plain_constrain(s):
    x, (n, v) = s["logits"].float(), s["logits"].shape
    place = torch.arange(s["history"].shape[1], device=x.device)
    at = torch.where(place < s["lengths"][:, None], s["history"], v)
    count = torch.zeros(n, v + 1, device=x.device).scatter_add_(1, at, torch.ones_like(at, dtype=torch.float32))[:, :v]
    r = s["repetition"][:, None]
    less = torch.where(x > 0, x / r, x * r) - count * s["frequency"][:, None] - s["presence"][:, None]
    x = torch.where(count > 0, less, x)
    if s["bias_ids"] is not None:
        x = x + torch.zeros(n, v, device=x.device).scatter_(1, s["bias_ids"], s["bias_values"])
    if s["mask"] is not None:
        token = torch.arange(v, device=x.device)
        bits = (s["mask"][s["states"].clamp(min=0).long()][:, token // 32] >> (token % 32)) & 1
        x = torch.where((bits != 0) | (s["states"] < 0)[:, None], x, -math.inf)
    return x


def _plain_top(logits, k, temperature):
    values, ids = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    tail = values[:, k:] / temperature
    top = tail[:, :1]
    return {"values": values[:, :k].contiguous(), "ids": ids[:, :k].contiguous(), "rest": top[:, 0] + (tail - top).exp().sum(1).log()}


def _plain_distill(s):
    c, x = s["case"], s["logits"].float()
    n, v = x.shape
    t, alpha = c["temperature"], c["alpha"]
    w = (s["weights"] if s["weights"] is not None else torch.ones(n, device=x.device)) / _denom(c)
    z = s["values"] / t
    if s["rest"] is not None:
        z = torch.cat([z, s["rest"][:, None]], 1)
    z = z - z.max(1, keepdim=True).values
    logq = z - z.exp().sum(1, keepdim=True).log()
    q = logq.exp()
    y = x / t
    top = y.max(1, keepdim=True).values
    e = (y - top).exp()
    total = e.sum(1, keepdim=True)
    logp = y.gather(1, s["ids"]) - top - total.log()
    grad = e / total
    if s["rest"] is not None:
        tail = e.scatter(1, s["ids"], 0.0)
        left = tail.sum(1, keepdim=True)
        logp = torch.cat([logp, (left / total).log()], 1)
        grad -= tail * (q[:, -1:] / left)
    grad.scatter_add_(1, s["ids"], -q[:, :c["k"]])
    row, grad = alpha * t * t * (q * (logq - logp)).sum(1), alpha * t * grad
    if alpha < 1:
        top = x.max(1, keepdim=True).values
        e = (x - top).exp()
        total = e.sum(1, keepdim=True)
        at = s["targets"][:, None]
        row = row + (1 - alpha) * (top + total.log() - x.gather(1, at))[:, 0]
        grad += (1 - alpha) * (e / total).scatter_add_(1, at, torch.full_like(total, -1.0))
    return {"loss": (w * row).sum().reshape(1), "grad": (w[:, None] * grad).to(s["logits"].dtype)}


# ---- the work and the definition in 64 bits ------------------------------------------------------------------------------
def work(case):
    n, v, size = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    logits = n * v
    if case["op"] in ("pick", "constrain"):
        nbytes = logits * size + n * (8 * case["history"] + 16 + 12 * case["biases"])
        if case["grammar"]:
            nbytes += min(n, 24) * 4 * ((v + 31) // 32) + 4 * n
        nbytes += n * 12 if case["op"] == "pick" else logits * size
        return {"bytes": nbytes, "flops": (4 if case["op"] == "pick" else 1) * logits}
    if case["op"] == "top":
        return {"bytes": logits * size + n * (12 * case["k"] + 4), "flops": 4 * logits}
    sums = 2 if case["alpha"] < 1 and case["temperature"] != 1 else 1
    return {"bytes": 2 * logits * size + n * (12 * case["k"] + 16), "flops": (4 * sums + 4) * logits}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].detach().double()
    rows = torch.arange(x.shape[0], device=x.device)[:, None]
    if case["op"] in ("pick", "constrain"):
        n, v = x.shape
        for b in range(n):
            seen, count = torch.unique(s["history"][b, :int(s["lengths"][b])], return_counts=True)
            u, r = x[b, seen], s["repetition"][b].double()
            u = torch.maximum(u, torch.zeros_like(u)) / r + torch.minimum(u, torch.zeros_like(u)) * r
            x[b, seen] = u - (count * s["frequency"][b].double() + s["presence"][b].double())
        if s["bias_ids"] is not None:
            x[rows, s["bias_ids"]] += s["bias_values"].double()
        if s["mask"] is not None:
            held = s["states"] >= 0
            shift = torch.arange(32, device=x.device, dtype=torch.int32)
            allowed = ((s["mask"][..., None] >> shift) & 1).bool().flatten(1)[:, :v]
            x[held] = x[held].masked_fill(~allowed[s["states"][held].long()], -math.inf)
        if case["op"] == "constrain":
            return {"logits": x}
        return {"tokens": None, "logp": torch.log_softmax(x, 1).max(1).values}
    t = case["temperature"]
    if case["op"] == "top":
        order = torch.sort(x, dim=1, descending=True, stable=True)
        return {"values": order.values[:, :case["k"]], "ids": None, "rest": torch.logsumexp(order.values[:, case["k"]:] / t, 1)}
    x.requires_grad_(True)
    teacher = s["values"].double() / t
    if s["rest"] is not None:
        teacher = torch.cat([teacher, s["rest"].double()[:, None]], 1)
    logq = torch.log_softmax(teacher, 1)
    inside = torch.zeros_like(x, dtype=torch.bool)
    inside[rows, s["ids"]] = True
    norm = torch.logsumexp(x / t, 1, keepdim=True)
    logp = x[rows, s["ids"]] / t - norm
    if s["rest"] is not None:
        logp = torch.cat([logp, torch.logsumexp((x / t).masked_fill(inside, -math.inf), 1, keepdim=True) - norm], 1)
    row = case["alpha"] * t * t * (logq.exp() * (logq - logp)).sum(1)
    if case["alpha"] < 1:
        row = row + (1 - case["alpha"]) * torch.nn.functional.cross_entropy(x, s["targets"], reduction="none")
    if s["weights"] is not None:
        row = row * s["weights"]
    loss = row.sum() / _denom(case)
    loss.backward()
    return {"loss": loss.detach().reshape(1), "grad": x.grad}
