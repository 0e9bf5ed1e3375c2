"""Plain restatements of the operators on output rows (speech_amd/logits.py) in 64 bits on the CPU: test infrastructure."""
import math

import torch


def constrain(logits, history=None, lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None,
              bias_values=None, mask=None, states=None):
    """The constrained rows in 64 bits, token by token as the formulas say."""
    x = logits.detach().cpu().double().clone()
    rows, V = x.shape

    def per_row(v, neutral):
        if v is None:
            return [neutral] * rows
        return [float(t) for t in v.cpu().double()] if torch.is_tensor(v) else [float(v)] * rows

    rep, pre, fre = per_row(repetition, 1.0), per_row(presence, 0.0), per_row(frequency, 0.0)
    for b in range(rows):
        if history is not None:
            n = history.shape[1] if lengths is None else min(max(int(lengths[b]), 0), history.shape[1])
            count = {}
            for t in history[b, :n].tolist():
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + 1
            for t, c in count.items():
                u = float(x[b, t])
                u = u / rep[b] if u > 0 else u * rep[b]
                x[b, t] = u - c * fre[b] - pre[b]
        if bias_ids is not None:
            last = {t: v for t, v in zip(bias_ids[b].tolist(), bias_values[b].cpu().double().tolist()) if 0 <= t < V}
            for t, v in last.items():
                x[b, t] += v
        if mask is not None:
            state = b if states is None else int(states[b])
            if 0 <= state < mask.shape[0]:
                words = mask[state].cpu().numpy().view("uint32")
                token = torch.arange(V)
                bits = (torch.from_numpy(words.astype("int64"))[token // 32] >> (token % 32)) & 1
                x[b][bits == 0] = -math.inf
    return x


def pick(x):
    """(tokens, log-probabilities) of constrained rows in 64 bits."""
    tokens, logp = [], []
    for row in x:
        if bool((row == -math.inf).all()):
            tokens.append(-1), logp.append(-math.inf)
            continue
        if bool(row.isnan().any()):
            tokens.append(int(row.isnan().nonzero()[0])), logp.append(math.nan)
            continue
        t = int((row == row.max()).nonzero()[0])
        tokens.append(t)
        if math.isinf(float(row[t])):
            logp.append(-math.log(int((row == row[t]).sum())))
        else:
            logp.append(float(torch.log_softmax(row, 0)[t]))
    return torch.tensor(tokens), torch.tensor(logp, dtype=torch.float64)


def top_logits(logits, k, temperature=1.0):
    """NaN above everything, ties to the lowest id."""
    x = logits.detach().cpu().double()
    order = torch.sort(torch.where(x.isnan(), math.inf, x), dim=-1, descending=True, stable=True).indices
    if bool(x.isnan().any()):  # NaN before +inf, each in the order of the ids
        rank = torch.where(x.isnan(), 0, torch.where(x == math.inf, 1, 2))
        by = torch.sort(torch.gather(rank, -1, order), dim=-1, stable=True).indices
        order = torch.gather(order, -1, by)
    values = torch.gather(x, -1, order)
    tail = values[..., k:] / temperature
    rest = torch.logsumexp(tail, -1) if tail.shape[-1] else torch.full(x.shape[:-1], -math.inf, dtype=torch.float64)
    return values[..., :k], order[..., :k], rest


def distill(logits, values, ids, rest=None, targets=None, weights=None, temperature=1.0, alpha=1.0, denom=None):
    """(loss, gradient, row losses) in 64 bits: the definition through log_softmax, the gradient by autograd, row by row."""
    V = logits.shape[-1]
    x = logits.detach().cpu().double().reshape(-1, V)
    n = x.shape[0]
    k = values.shape[-1]
    denom = float(denom) if denom else float(n)
    grad, losses = torch.zeros_like(x), torch.zeros(n, dtype=torch.float64)
    values, ids = values.cpu().double().reshape(n, k), ids.cpu().reshape(n, k)
    for i in range(n):
        w = 1.0 if weights is None else float(weights.reshape(-1)[i])
        if w == 0.0:
            continue
        xi = x[i].clone().requires_grad_(True)
        there = (ids[i] >= 0) & (ids[i] < V)
        at = ids[i][there]
        a = values[i][there] / temperature
        lp = torch.log_softmax(xi / temperature, 0)
        terms = lp[at]
        if rest is not None:
            a = torch.cat([a, rest.cpu().double().reshape(-1)[i:i + 1]])
            outside = torch.ones(V, dtype=torch.bool)
            outside[at] = False
            tail = torch.logsumexp(lp[outside], 0) if bool(outside.any()) else torch.tensor(-math.inf, dtype=torch.float64)
            terms = torch.cat([terms, tail.reshape(1)])
        row = torch.zeros((), dtype=torch.float64)
        if a.numel() and float(a.max()) > -math.inf and alpha > 0:
            logq = torch.log_softmax(a, 0)
            on = logq > -math.inf
            row = row + alpha * temperature ** 2 * (logq[on].exp() * (logq[on] - terms[on])).sum()
        if alpha < 1 and targets is not None:
            y = int(targets.reshape(-1)[i])
            if 0 <= y < V:
                row = row - (1 - alpha) * torch.log_softmax(xi, 0)[y]
        row = row * w / denom
        losses[i] = row.detach()
        if row.requires_grad:
            grad[i], = torch.autograd.grad(row, xi)
    return losses.sum(), grad.reshape(logits.shape), losses
