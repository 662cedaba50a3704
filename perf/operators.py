"""The operators around a training step's products, as cases that can be timed and compared.

A case is one direction of one operator, on tensors that are already on the GPU:
  "ce_forward", "ce_backward"        the output head's product with softmax cross entropy, whose
                                     logits are never kept;
  "route_forward", "route_backward"  the router of a mixture of experts: the chosen experts with
                                     their gates, counts and packed rows, and the balance loss;
  "clip"                             the global norm of many gradients, and the clipped gradients.
With `own` false `run` computes an operator from elementary torch operations in 32 bits.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_IGNORE = -100
_EPS = 1e-6
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _operators():
    package = os.path.join(_ROOT, "flash-train_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import flash_train.torch

    return flash_train.torch


def _ce(kind, tokens, hidden, classes, dtype, ignored):
    return {"kind": kind, "tokens": tokens, "hidden": hidden, "classes": classes, "dtype": dtype, "ignored": ignored}


def _route(kind, tokens, experts, top_k, dtype, normalize, masked):
    return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "normalize": normalize, "masked": masked}


def _clip(layers, width, inner, dtype, clips):
    return {"kind": "clip", "layers": layers, "width": width, "inner": inner, "dtype": dtype, "clips": clips}


def listed():
    cases = {
        # Sixteen tokens scored against a vocabulary of odd size: all of it is reading the weight.
        "ce_few": _ce("ce_forward", 16, 4096, 32003, "bf16", 0.0),
        # The loss of an evaluation batch: the large product alone.
        "ce_loss": _ce("ce_forward", 8192, 4096, 65536, "bf16", 0.0),
        # Tuning of a small model on answers: odd sizes, a third of the tokens without a target.
        "ce_grad_small": _ce("ce_backward", 500, 1024, 5003, "fp16", 0.3),
        # Full precision training with padding.
        "ce_grad_fp32": _ce("ce_backward", 2048, 2048, 32003, "fp32", 0.1),
        # Pretraining: the gradients of a large vocabulary's head.
        "ce_grad": _ce("ce_backward", 8192, 4096, 131072, "bf16", 0.0),
        # A micro batch of a few tokens over few experts: launches and latency.
        "route_few": _route("route_forward", 64, 8, 2, "bf16", True, 0.0),
        # A training batch over 64 experts, some of it padding.
        "route_batch": _route("route_forward", 16384, 64, 2, "bf16", True, 0.1),
        # A large batch over many small experts.
        "route_many": _route("route_forward", 131072, 256, 8, "fp32", False, 0.0),
        # The router's gradient over the training batch.
        "route_grad": _route("route_backward", 16384, 64, 2, "bf16", True, 0.1),
        # The router's gradient with many small experts, an odd number of tokens.
        "route_grad_many": _route("route_backward", 100003, 160, 6, "fp32", False, 0.0),
        # The gradients of a small network, odd sizes in full precision, below the limit.
        "clip_small": _clip(3, 127, 97, "fp32", False),
        # The gradients of eight experts, clipped.
        "clip_experts": _clip(8, 4096, 14336, "bf16", True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, low, high, step=1):
    """A whole number of `step` between low and high, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    kind = rng.choice(["ce_forward", "ce_backward", "ce_backward", "route_forward", "route_backward", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("ce"):
        step = 1 if rng.random() < 0.2 else 8
        tokens = _log(rng, 1 if kind == "ce_forward" else 16, 16384)
        case = _ce(kind, tokens, _log(rng, 256, 8192, step), _log(rng, 1000, 131072, 1 if rng.random() < 0.5 else 8),
                   dtype, rng.choice([0.0, 0.1, 0.3, 0.7]) if tokens >= 64 else 0.0)
        most = 5e11 if dtype == "fp32" else 2.6e13
        while work(case)["flops"] > most:
            side = max(("tokens", "classes"), key=lambda s: case[s])
            case[side] = max(16, case[side] * 2 // 3)
        return case
    if kind.startswith("route"):
        experts = _log(rng, 4, 256)
        return _route(kind, _log(rng, 16, 131072), experts, min(experts, rng.randint(1, 8)), dtype,
                      rng.random() < 0.5, rng.choice([0.0, 0.1]))
    return _clip(_log(rng, 1, 64), _log(rng, 64, 4096), _log(rng, 64, 4096), dtype, rng.random() < 0.7)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ce_inputs(case, seed):
    """Hidden states of unit spread that have partly learned their targets, so that probabilities
    run from near nothing to near one, and a head's weight; both rounded to the case's type."""
    gen = _generator(seed)
    t, h, v, dtype = case["tokens"], case["hidden"], case["classes"], _TYPES[case["dtype"]]
    weight = (torch.randn(v, h, generator=gen, device="cuda") * (2.0 / math.sqrt(h))).to(dtype)
    target = torch.randint(0, v, (t,), generator=gen, device="cuda")
    learned = 4.0 * torch.rand(t, 1, generator=gen, device="cuda")
    hidden = (torch.randn(t, h, generator=gen, device="cuda") + learned * weight[target].float()).to(dtype)
    drop = torch.rand(t, generator=gen, device="cuda") < case["ignored"]
    target = torch.where(drop, torch.full_like(target, _IGNORE), target)
    if case["kind"] == "ce_forward":
        return {"hidden": hidden, "weight": weight, "target": target}
    lse = torch.empty(t, device="cuda")
    rows = max(1, (1 << 28) // v)
    for first in range(0, t, rows):
        lse[first:first + rows] = torch.logsumexp(hidden[first:first + rows].float() @ weight.float().t(), 1)
    lse = torch.where(drop, torch.zeros_like(lse), lse)
    # The mean over the tokens, each with a weight of its own.
    grad = (0.5 + torch.rand(t, generator=gen, device="cuda")) / max(1, int((~drop).sum()))
    return {"hidden": hidden, "weight": weight, "target": target, "lse": lse, "grad_loss": grad}


def _chosen(logits, top_k):
    """The top_k highest logits of each row, ties to the lowest index; -1 where fewer than top_k are
    above minus infinity."""
    left, index = logits.clone(), torch.arange(logits.size(1), device=logits.device)
    picks = []
    for _ in range(top_k):
        best = left.amax(1, keepdim=True)
        pick = torch.where(left == best, index, logits.size(1)).amin(1, keepdim=True)
        picks.append(torch.where(best > -math.inf, pick, -1))
        left.scatter_(1, pick.clamp(max=logits.size(1) - 1), -math.inf)
    return torch.cat(picks, 1)


def _route_inputs(case, seed):
    """Logits of a router with favourite experts; padding is masked."""
    gen = _generator(seed)
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(t, e, generator=gen, device="cuda") + 0.5 * torch.randn(e, generator=gen, device="cuda")
    logits = logits.to(_TYPES[case["dtype"]])
    mask = None
    if case["masked"] > 0:
        mask = torch.rand(t, generator=gen, device="cuda") >= case["masked"]
    state = {"logits": logits, "top_k": k, "normalize": case["normalize"], "mask": mask}
    if case["kind"] == "route_backward":
        experts = _chosen(logits.float(), k)
        if mask is not None:
            experts = torch.where(mask[:, None], experts, -1)
        state["experts"] = experts.int()
        state["counts"] = torch.bincount(experts[experts >= 0], minlength=e).int()
        state["routed"] = torch.full((1,), t if mask is None else int(mask.sum()), device="cuda", dtype=torch.int32)
        state["grad_gates"] = torch.randn(t, k, generator=gen, device="cuda") / t
        state["grad_loss"] = torch.full((), 0.01, device="cuda")
    return state


def _clip_inputs(case, seed):
    """A layer's gradients: two matrices and a vector of odd length each, of different spreads."""
    gen = _generator(seed)
    n, a, b, dtype = case["layers"], case["width"], case["inner"], _TYPES[case["dtype"]]
    grads = []
    for layer in range(n):
        scale = 1e-4 * (1.0 + layer % 5)
        for shape in ((a, b), (b, a), (a + 1,)):
            kind = dtype if len(shape) == 2 else torch.float32
            grads.append(torch.randn(*shape, generator=gen, device="cuda", dtype=kind).mul_(scale))
    expected = math.sqrt(sum(g.numel() * (1e-4 * (1.0 + i // 3 % 5)) ** 2 for i, g in enumerate(grads)))
    return {"grads": grads, "max_norm": expected * (0.3 if case["clips"] else 4.0)}


def prepare(case, seed):
    if case["kind"].startswith("ce"):
        return dict(_ce_inputs(case, seed), kind=case["kind"])
    if case["kind"].startswith("route"):
        return dict(_route_inputs(case, seed), kind=case["kind"])
    state = dict(_clip_inputs(case, seed), kind="clip")
    # The optimiser's copy of the gradients, which a program keeps from step to step.
    state["out"] = [torch.empty_like(g) for g in state["grads"]]
    return state


def _run_own(s):
    op = _operators()
    if s["kind"] == "ce_forward":
        return op.linear_cross_entropy_forward(s["hidden"], s["weight"], s["target"], ignore_index=_IGNORE)
    if s["kind"] == "ce_backward":
        return op.linear_cross_entropy_backward(s["grad_loss"], s["hidden"], s["weight"], s["target"], s["lse"],
                                                ignore_index=_IGNORE)
    if s["kind"] == "route_forward":
        return op.moe_route_forward(s["logits"], s["top_k"], normalize=s["normalize"], mask=s["mask"])
    if s["kind"] == "route_backward":
        return op.moe_route_backward(s["grad_gates"], s["grad_loss"], s["logits"], s["experts"], s["counts"],
                                     s["routed"], normalize=s["normalize"], mask=s["mask"])
    norm = op.clip_grad_norm(s["grads"], s["max_norm"], eps=_EPS, out=s["out"])
    return [norm] + s["out"]


def _softmax(logits):
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    return p / p.sum(1, keepdim=True)


def _run_plain(s):
    if s["kind"] == "ce_forward":
        keep = s["target"] != _IGNORE
        logits = s["hidden"].float() @ s["weight"].float().t()
        top = logits.amax(1, keepdim=True)
        lse = top[:, 0] + torch.log(torch.exp(logits - top).sum(1))
        hit = logits.gather(1, torch.where(keep, s["target"], 0)[:, None])[:, 0]
        zero = torch.zeros_like(lse)
        return torch.where(keep, lse - hit, zero), torch.where(keep, lse, zero)
    if s["kind"] == "ce_backward":
        x, w, keep = s["hidden"].float(), s["weight"].float(), s["target"] != _IGNORE
        grad = torch.exp(x @ w.t() - s["lse"][:, None])
        grad.scatter_add_(1, torch.where(keep, s["target"], 0)[:, None], -torch.ones_like(grad[:, :1]))
        grad = torch.where(keep[:, None], grad * s["grad_loss"][:, None], 0.0)
        return (grad @ w).to(s["hidden"].dtype), (grad.t() @ x).to(s["weight"].dtype)
    if s["kind"] == "route_forward":
        logits = s["logits"].float()
        t, e = logits.shape
        p, experts = _softmax(logits), _chosen(logits, s["top_k"])
        if s["mask"] is not None:
            experts = torch.where(s["mask"][:, None], experts, -1)
            p = torch.where(s["mask"][:, None], p, 0.0)
        gates = torch.where(experts >= 0, p.gather(1, experts.clamp(min=0)), 0.0)
        if s["normalize"]:
            total = gates.sum(1, keepdim=True)
            gates = torch.where(total > 0, gates / total, 0.0)
        flat = torch.where(experts >= 0, experts, e).flatten()
        counts = torch.bincount(flat, minlength=e + 1)[:e].int()
        order = torch.sort(flat, stable=True).indices
        slots = torch.empty_like(order)
        slots[order] = torch.arange(t * s["top_k"], device=flat.device)
        slots = torch.where(experts >= 0, slots.view_as(experts), -1)
        routed = torch.full((1,), t, device=flat.device, dtype=torch.int32)
        if s["mask"] is not None:
            routed = s["mask"].sum(dtype=torch.int32).view(1)
        share = counts.float() / counts.sum().clamp(min=1)
        loss = e * (share * p.sum(0) / routed.clamp(min=1)).sum()
        return experts.int(), gates, slots.int(), counts, routed, loss
    if s["kind"] == "route_backward":
        logits, experts = s["logits"].float(), s["experts"].long()
        e, p = logits.size(1), _softmax(logits)
        kept, at = experts >= 0, experts.clamp(min=0)
        share = s["counts"].float() / s["counts"].sum().clamp(min=1)
        balance = (s["grad_loss"] * e * share / s["routed"].clamp(min=1))[None, :]
        gates_grad = torch.where(kept, s["grad_gates"], 0.0)
        picked = torch.where(kept, p.gather(1, at), 0.0)
        if s["normalize"]:
            total = picked.sum(1, keepdim=True)
            gate = torch.where(total > 0, picked / total, 0.0)
            chosen = gate * (gates_grad - (gate * gates_grad).sum(1, keepdim=True))
            grad = p * (balance - (p * balance).sum(1, keepdim=True))
            grad = grad.scatter_add(1, at, torch.where(kept, chosen, 0.0))
        else:
            dp = balance.expand_as(p).scatter_add(1, at, gates_grad)
            grad = p * (dp - (p * dp).sum(1, keepdim=True))
        if s["mask"] is not None:
            grad = torch.where(s["mask"][:, None], grad, 0.0)
        return grad.to(s["logits"].dtype)
    total = torch.zeros((), device="cuda")
    for g in s["grads"]:
        total = total + g.float().square().sum()
    norm = torch.sqrt(total)
    scale = (s["max_norm"] / (norm + _EPS)).clamp(max=1.0)
    return [norm] + [(g.float() * scale).to(g.dtype) for g in s["grads"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def exact(case, seed):
    if case["kind"].startswith("ce"):
        return _ce_exact(case, _ce_inputs(case, seed))
    if case["kind"].startswith("route"):
        return _route_exact(case, _route_inputs(case, seed))
    s = _clip_inputs(case, seed)
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in s["grads"]]))
    coef = min(1.0, s["max_norm"] / (float(norm) + _EPS))
    return [norm] + [g.double() * coef for g in s["grads"]]


def _ce_exact(case, s):
    """In pieces of the vocabulary, as the definition's sums over it."""
    x, target = s["hidden"].double(), s["target"]
    keep = target != _IGNORE
    step = max(256, (1 << 27) // case["tokens"])
    pieces = [(v, min(v + step, case["classes"])) for v in range(0, case["classes"], step)]
    if case["kind"] == "ce_forward":
        lse, hit = torch.full_like(x[:, 0], -math.inf), torch.zeros_like(x[:, 0])
        for low, high in pieces:
            logits = x @ s["weight"][low:high].double().t()
            lse = torch.logaddexp(lse, torch.logsumexp(logits, 1))
            rows = torch.nonzero((target >= low) & (target < high))[:, 0]
            hit[rows] = logits[rows, target[rows] - low]
        return (lse - hit) * keep, lse * keep
    dx = torch.zeros_like(x)
    dw = torch.empty(case["classes"], case["hidden"], device="cuda", dtype=torch.float64)
    scale = (s["grad_loss"].double() * keep)[:, None]
    for low, high in pieces:
        w = s["weight"][low:high].double()
        dl = (x @ w.t()).sub_(s["lse"].double()[:, None]).exp_()
        rows = torch.nonzero((target >= low) & (target < high))[:, 0]
        dl[rows, target[rows] - low] -= 1.0
        dl.mul_(scale)
        dx += dl @ w
        dw[low:high] = dl.t() @ x
    return dx, dw


def _route_exact(case, s):
    logits = s["logits"].double()
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    keep = torch.ones(t, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    p = torch.softmax(logits, 1) * keep[:, None]
    if case["kind"] == "route_forward":
        experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        gates = torch.gather(p, 1, experts)
        if s["normalize"]:
            gates = gates / gates.sum(1, keepdim=True)
        gates = torch.where(keep[:, None], gates, 0.0)
        experts = torch.where(keep[:, None], experts, e)
        counts = torch.stack([(experts == i).sum() for i in range(e)])
        slots, first = torch.full((t * k,), -1, device="cuda"), 0
        for i in range(e):
            rows = torch.nonzero(experts.flatten() == i)[:, 0]
            slots[rows] = torch.arange(first, first + rows.numel(), device="cuda")
            first += rows.numel()
        n = keep.sum()
        loss = e * torch.dot(counts.double() / counts.sum(), p.sum(0) / n)
        return (torch.where(keep[:, None], experts, -1).int(), gates, slots.view(t, k).int(), counts.int(), n.int().view(1),
                loss)
    leaf = logits.requires_grad_()
    with torch.enable_grad():
        q = torch.softmax(leaf, 1)[keep]
        gates = torch.gather(q, 1, s["experts"][keep].long())
        if s["normalize"]:
            gates = gates / gates.sum(1, keepdim=True)
        f = s["counts"].double() / s["counts"].sum()
        loss = s["grad_loss"].double() * e * (f * q.sum(0)).sum() / int(s["routed"])
        (loss + (gates * s["grad_gates"][keep].double()).sum()).backward()
    return leaf.grad


def work(case):
    if case["kind"].startswith("ce"):
        t, h, v, size = case["tokens"], case["hidden"], case["classes"], 4 if case["dtype"] == "fp32" else 2
        operands = size * h * (t + v)
        if case["kind"] == "ce_forward":
            return {"bytes": operands + 16 * t, "flops": 2 * t * h * v}
        return {"bytes": 2 * operands + 16 * t, "flops": 6 * t * h * v}
    if case["kind"].startswith("route"):
        t, e, k, size = case["tokens"], case["experts"], case["top_k"], 4 if case["dtype"] == "fp32" else 2
        masks = t if case["masked"] > 0 else 0
        if case["kind"] == "route_forward":
            return {"bytes": size * t * e + masks + 12 * t * k + 4 * e + 8, "flops": 8 * t * e}
        return {"bytes": 2 * size * t * e + masks + 8 * t * k + 4 * e + 8, "flops": 12 * t * e}
    n, a, b, size = case["layers"], case["width"], case["inner"], 4 if case["dtype"] == "fp32" else 2
    return {"bytes": 2 * n * (2 * a * b * size + 4 * (a + 1)) + 4, "flops": 3 * n * (2 * a * b + a + 1)}
