"""Plain 64-bit forms of the operators around a training step's products, on the CPU, with the error
bounds that the tests hold the kernels to.

Bounds: a sum of n terms in 32 bits, in any order, is off by at most c sqrt(n) u times the sum of the
terms' magnitudes with u = 2^-23 and c = 4 for random rounding errors; a value rounded to a 16-bit type
by u of that type (2^-8 bf16, 2^-10 fp16: twice the half unit) plus, in fp16, half its smallest number.
"""

import math

import torch

U32 = 2.0**-23
ROUNDING = {torch.float32: (U32, 0.0), torch.bfloat16: (2.0**-8, 0.0), torch.float16: (2.0**-10, 2.0**-25)}


def cross_entropy(hidden, weight, target, ignore_index=-100):
    """(loss, lse, bound of both) in 64 bits."""
    x, w = hidden.double(), weight.double()
    logits = x @ w.t()
    keep = target != ignore_index
    lse = torch.logsumexp(logits, 1)
    hit = logits.gather(1, torch.where(keep, target, 0).long()[:, None])[:, 0]
    logit_bound = 4 * math.sqrt(x.shape[1]) * U32 * (x.abs() @ w.abs().t()).amax(1)
    bound = 2 * logit_bound + 8 * U32 * (4 + lse.abs() + math.sqrt(w.shape[0]))
    zero = torch.zeros_like(lse)
    return torch.where(keep, lse - hit, zero), torch.where(keep, lse, zero), bound


def cross_entropy_grads(grad_loss, hidden, weight, target, lse, ignore_index=-100):
    """(grad_hidden, grad_weight) in 64 bits and their elementwise bounds."""
    x, w, g = hidden.double(), weight.double(), grad_loss.double()
    keep = target != ignore_index
    x = torch.where(keep[:, None], x, 0.0)
    g = torch.where(keep, g, 0.0)
    p = torch.exp(torch.where(keep[:, None], x @ w.t() - lse.double()[:, None], 0.0))
    hot = torch.zeros_like(p).scatter_(1, torch.where(keep, target, 0).long()[:, None], 1.0)
    dl = (p - hot) * g[:, None]
    u, tiny = ROUNDING[hidden.dtype]
    logit_bound = 4 * math.sqrt(x.shape[1]) * U32 * (x.abs() @ w.abs().t()).amax(1, keepdim=True)
    dl_bound = (p * (logit_bound + 8 * U32 * (2 + lse.double().abs()[:, None])) + U32) * g.abs()[:, None]
    if hidden.dtype != torch.float32:
        dl_bound = dl_bound + u * dl.abs() + 2.0**-38 * g.abs().max()
    out = []
    for a, b, da in ((dl, w, dl_bound), (dl.t(), x, dl_bound.t())):
        exact, size = a @ b, a.abs() @ b.abs()
        out += [exact, da @ b.abs() + 4 * math.sqrt(a.shape[1] + 1) * U32 * size + u * exact.abs() + tiny]
    return out[0], out[2], out[1], out[3]


def route(logits, top_k, normalize, mask=None):
    """experts, gates, slots, counts, routed, balance loss, and which rows take part; loops and 64 bits."""
    rows, n = logits.shape
    values = logits.double()
    experts = torch.full((rows, top_k), -1, dtype=torch.int32)
    gates = torch.zeros(rows, top_k, dtype=torch.float64)
    p_sum = torch.zeros(n, dtype=torch.float64)
    part = torch.zeros(rows, dtype=torch.bool)
    for t in range(rows):
        row = values[t].tolist()
        if (mask is not None and not mask[t]) or all(v == -math.inf for v in row):
            continue
        part[t] = True
        p = torch.softmax(values[t], 0)
        p_sum += p
        order = sorted((e for e in range(n) if row[e] > -math.inf), key=lambda e: (-row[e], e))[:top_k]
        for k, e in enumerate(order):
            experts[t, k], gates[t, k] = e, p[e]
        if normalize and order:
            gates[t] /= gates[t].sum()
    counts = torch.zeros(n, dtype=torch.int32)
    slots = torch.full((rows, top_k), -1, dtype=torch.int32)
    slot = 0
    for e in range(n):
        for t, k in torch.nonzero(experts == e).tolist():
            slots[t, k] = slot
            slot += 1
            counts[e] += 1
    routed = int(part.sum())
    loss = n * float((counts.double() / max(1, slot) * p_sum / max(1, routed)).sum())
    return experts, gates, slots, counts, routed, loss, part


def route_grad(grad_gates, grad_loss, logits, experts, counts, routed, normalize, part):
    """The logits' gradient in 64 bits by automatic differentiation of the definition."""
    leaf = logits.double().clone().requires_grad_()
    total = torch.zeros((), dtype=torch.float64)
    share = counts.double() / max(1, int(counts.sum())) * logits.shape[1] / max(1, routed)
    for t in torch.nonzero(part)[:, 0].tolist():
        p = torch.softmax(leaf[t], 0)
        chosen = [e for e in experts[t].tolist() if e >= 0]
        gates = p[chosen]
        if normalize:
            gates = gates / gates.sum()
        total = total + float(grad_loss) * (share * p).sum() + (gates * grad_gates[t, : len(chosen)].double()).sum()
    if part.any():
        total.backward()
    return leaf.grad if leaf.grad is not None else torch.zeros_like(leaf)
