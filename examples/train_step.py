"""Training steps of a small model whose middle is a contraction of this engine.

    token numbers -> rows of a table -> hidden = x * mixing -> softmax cross entropy over the same table

Rows come from `EmbeddingPlan`, the mixing and its gradients are contractions (`Plan`, fp32), loss and gradients come from
`VocabLossPlan`, the table's two gradients are added up by `EmbeddingPlan.execute_grad(accumulate=True)`, and the mixing
matrix moves by its momentum orthogonalised (`OrthogonalPlan`).  Run as `python examples/train_step.py [steps]` on a machine
with a GPU; prints the mean loss of each step, which falls."""
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
tc = importlib.import_module("cgo2019-ae_b200")


class Model:
    def __init__(self, tokens=1024, dim=256, vocab=4096, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.tokens, self.dim, self.vocab = tokens, dim, vocab
        self.table = (torch.randn(vocab, dim, device="cuda", generator=gen) * dim ** -0.5).bfloat16()
        self.mixing = torch.eye(dim, device="cuda") + 0.1 * torch.randn(dim, dim, device="cuda", generator=gen) * dim ** -0.5
        self.momentum = torch.zeros(dim, dim, device="cuda")
        self.rows = tc.EmbeddingPlan(tokens, vocab, dim, scale=dim ** 0.5).commit()
        self.loss = tc.VocabLossPlan(tokens, dim, vocab).commit()
        self.update = tc.OrthogonalPlan(dim, dim, dtype=tc.F32).commit()
        # row-major matrices [t][d] are column-major tensors (d, t): index d is the fastest
        sizes = {"d": dim, "e": dim, "t": tokens}
        named = lambda line: line.format(**sizes)  # noqa: E731
        self.forward = tc.Plan(named("h [e,{e},t,{t}] = sum(d,{d}) * w [e,d] * x [d,t];"), tc.F32).commit()
        self.to_rows = tc.Plan(named("x [d,{d},t,{t}] = sum(e,{e}) * w [e,d] * h [e,t];"), tc.F32).commit()
        self.to_mixing = tc.Plan(named("w [e,{e},d,{d}] = sum(t,{t}) * h [e,t] * x [d,t];"), tc.F32).commit()

    def step(self, ids, targets, rate=0.02, table_rate=0.5, inertia=0.9):
        """One step on `ids` -> `targets` (below zero: not asked); the mean loss, on the GPU."""
        t, d = self.tokens, self.dim
        half = lambda *shape: torch.empty(*shape, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        single = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        rows, hidden = half(t, d), single(t, d)
        self.rows.execute(rows, self.table, ids)
        x = rows.float()
        self.forward.execute(hidden, self.mixing, x)
        hidden = hidden.bfloat16()

        losses, lse = single(t), single(t)
        self.loss.execute(losses, lse, hidden, self.table, targets)
        asked = (targets >= 0).sum().clamp(min=1)
        weights = (1.0 / asked).float().expand(t).contiguous()
        dhidden, dtable = half(t, d), half(self.vocab, d)
        self.loss.execute_grad(dhidden, dtable, hidden, self.table, targets, lse, weights)

        dhidden, dx, dmixing = dhidden.float(), single(t, d), single(d, d)
        self.to_rows.execute(dx, self.mixing, dhidden)
        self.to_mixing.execute(dmixing, dhidden, x)
        self.rows.execute_grad(dtable, dx.bfloat16(), ids, accumulate=True)

        self.momentum.mul_(inertia).add_(dmixing)
        update = half(d, d)
        self.update.execute(update, self.momentum)
        self.mixing.sub_(update.float(), alpha=rate)
        self.table.sub_(dtable, alpha=table_rate)
        return losses.sum() / asked


def main(steps=20):
    model = Model()
    gen = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, model.vocab, (model.tokens,), device="cuda", generator=gen)
    targets = (ids * 7 + 3) % model.vocab  # something to learn; one in eight is not asked
    targets[::8] = -1
    losses = [model.step(ids, targets) for _ in range(steps)]
    for k, value in enumerate(losses):
        print("step %2d  mean loss %.4f" % (k, value.item()))
    return [v.item() for v in losses]


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 20)
