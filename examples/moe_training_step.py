#!/usr/bin/env python3
"""Trains a small language model with a mixture of experts on one GPU, on synthetic tokens.

The model is an embedding, one layer of experts and an output head over a large vocabulary, in bf16:
  flash_train.torch.moe_route             chooses each token's experts, packs the choices by expert, and
                                          gives the balance loss;
  the grouped products (flash_train.capi) multiply the packed tokens by their experts' weights, forward
                                          and for both gradients;
  flash_train.torch.linear_cross_entropy  is the head: the loss without the logits in memory;
  flash_train.torch.clip_grad_norm        limits the gradients before the update.

  python examples/moe_training_step.py [--steps 30] [--tokens 2048] [--hidden 512] [--classes 32003]
"""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-train_amd"))

import torch  # noqa: E402

import flash_train.capi as capi  # noqa: E402
import flash_train.torch as ft  # noqa: E402


def _grouped(kind: str, **roles) -> None:
    """One execution of a grouped product on the current stream.  The groups' sizes are this step's, so
    the Plan is too."""
    ops = capi.GroupedOps(kind)
    one, zero = capi.HostScalar(1.0), capi.HostScalar(0.0)
    args = ops.args(alpha=one.view, beta=zero.view, **roles)
    try:
        plan = args.plan()
    finally:
        args.close()
    plan.execute(0, torch.cuda.current_stream().cuda_stream)
    # The Plan's table of groups is device memory of its own, read by the kernels until they end.
    torch.cuda.current_stream().synchronize()


def _packed(t: torch.Tensor, rows: list, transposed: bool = False) -> capi.GroupedSpec:
    """Rows packed by group (or each group's rows as columns)."""
    n, width = len(rows), t.shape[1]
    view = capi.matrix(t) if t.shape[0] else capi.View(None, list(t.shape), numeric_type=capi.TORCH_NUMERIC_TYPES[t.dtype])
    if not transposed:
        return capi.GroupedSpec(view, n, dims=[(r, width) for r in rows])
    first = [sum(rows[:i]) * width for i in range(n)]
    return capi.GroupedSpec(view, n, dims=[(width, r) for r in rows], strides=[(1, width)] * n, offsets=first)


class ExpertProducts(torch.autograd.Function):
    """y = x_e @ w_e for the rows x_e of every expert e; w: experts x in x out."""

    @staticmethod
    def forward(ctx, x, w, rows):
        n, k, m = w.shape
        y = x.new_empty(x.shape[0], m)
        _grouped("abcd", a=_packed(x, rows), b=capi.GroupedSpec(capi.matrix(w[0]), n),
                 c=capi.GroupedSpec(capi.View(None, [0, m], numeric_type=capi.BF16), n, dims=[(r, m) for r in rows]),
                 d=_packed(y, rows))
        ctx.save_for_backward(x, w)
        ctx.rows = rows
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (x, w), rows = ctx.saved_tensors, ctx.rows
        n, k, m = w.shape
        dy = dy.contiguous()
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        transposed = capi.View(w.data_ptr(), [m, k], numeric_type=capi.BF16)
        _grouped("abcd", a=_packed(dy, rows),
                 b=capi.GroupedSpec(transposed, n, dims=[(m, k)] * n, strides=[(1, m)] * n, offsets=[e * k * m for e in range(n)]),
                 c=capi.GroupedSpec(capi.View(None, [0, k], numeric_type=capi.BF16), n, dims=[(r, k) for r in rows]),
                 d=_packed(dx, rows))
        _grouped("ab", a=_packed(x, rows, transposed=True), b=_packed(dy, rows),
                 c=[capi.View(None, [k, m], numeric_type=capi.BF16) for _ in range(n)], d=[capi.matrix(e) for e in dw])
        return dx, dw, None


class Model:
    def __init__(self, hidden: int, classes: int, experts: int, top_k: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape, scale):
            return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16().requires_grad_()

        self.top_k = top_k
        self.embedding = weight(classes, hidden, scale=1.0)
        self.router = weight(experts, hidden, scale=hidden**-0.5)
        self.up = weight(experts, hidden, 2 * hidden, scale=hidden**-0.5)
        self.down = weight(experts, 2 * hidden, hidden, scale=(2 * hidden) ** -0.5)
        self.head = weight(classes, hidden, scale=hidden**-0.5)

    def parameters(self) -> list:
        return [self.embedding, self.router, self.up, self.down, self.head]

    def loss(self, tokens: torch.Tensor, target: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        x = self.embedding[tokens]
        routing = ft.moe_route(x @ self.router.t(), self.top_k, normalize=True, mask=mask)
        # Each choice's row of the packed tokens; a masked token has none and takes no part.
        kept = torch.nonzero(routing.slots >= 0, as_tuple=True)
        slots = routing.slots[kept].long()
        source = torch.empty_like(slots).scatter_(0, slots, kept[0])
        rows = routing.counts.tolist()
        packed = x.index_select(0, source)
        y = ExpertProducts.apply(torch.nn.functional.silu(ExpertProducts.apply(packed, self.up, rows)), self.down, rows)
        gates = routing.gates[kept].bfloat16()
        out = x.index_add(0, kept[0], y.index_select(0, slots) * gates[:, None])
        return ft.linear_cross_entropy(out, self.head, target) + 0.01 * routing.balance_loss


def train(steps: int, tokens: int, hidden: int, classes: int, experts: int = 8, top_k: int = 2, seed: int = 0) -> list:
    """Losses of `steps` steps on one batch: each token's target is a fixed function of it, and a tenth
    of the tokens is padding (no target, no experts)."""
    model = Model(hidden, classes, experts, top_k, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    batch = torch.randint(0, classes, (tokens,), generator=g, device="cuda")
    mask = torch.rand(tokens, generator=g, device="cuda") >= 0.1
    target = torch.where(mask, (batch * 7 + 3) % classes, -100)
    losses = []
    for _ in range(steps):
        for p in model.parameters():
            p.grad = None
        loss = model.loss(batch, target, mask)
        loss.backward()
        ft.clip_grad_norm([p.grad for p in model.parameters()], 1.0)
        with torch.no_grad():
            for p in model.parameters():
                p -= 2.0 * p.grad
        losses.append(float(loss.detach()))
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--classes", type=int, default=32003)
    args = ap.parse_args()
    for step, loss in enumerate(train(args.steps, args.tokens, args.hidden, args.classes)):
        print(f"step {step:3d}  loss {loss:.4f}", flush=True)


if __name__ == "__main__":
    main()
