"""The operators at the two ends of a model's training step and of its weight update, as measurable cases.

Between a model's first and last layer lie contractions; around them a program that trains it looks rows up in a table and
sums gradients back into it (`EmbeddingPlan`), takes the softmax cross entropy over the vocabulary and its gradient
without holding the logits (`VocabLossPlan`), and orthogonalises the update of each matrix (`OrthogonalPlan`).  A case is
one pass through one of them.  With `own` false the same results come from elementary torch operations in 32 bits.
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of x, x^3 and x^5 in one step of the iteration
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # evaluating a handful of tokens: one pass over the table, no gradient
        {"name": "loss_eval_16", "op": "loss", "type": "bf16", "tokens": 16, "dim": 512, "vocab": 32000, "ignored": 0.0, "grad": False},
        # a fine-tuning step in half precision with scaled gradients: prompts masked, nothing a multiple of anything
        {"name": "loss_odd_f16", "op": "loss", "type": "f16", "tokens": 1023, "dim": 777, "vocab": 50001, "ignored": 0.4, "grad": True},
        # a training step of a small model
        {"name": "loss_train_2048", "op": "loss", "type": "bf16", "tokens": 2048, "dim": 1024, "vocab": 32768, "ignored": 0.0, "grad": True},
        # a training step over a large vocabulary: what the operator is for
        {"name": "loss_train_8192", "op": "loss", "type": "bf16", "tokens": 8192, "dim": 2048, "vocab": 131072, "ignored": 0.05, "grad": True},
        # the next tokens of a few sequences
        {"name": "lookup_8", "op": "lookup", "type": "bf16", "tokens": 8, "dim": 2048, "vocab": 131072, "ignored": 0.0},
        # a batch of packed sequences
        {"name": "lookup_16384", "op": "lookup", "type": "bf16", "tokens": 16384, "dim": 2048, "vocab": 131072, "ignored": 0.05},
        # gradient in single precision with odd rows, as tables outside of a model's trunk have
        {"name": "table_grad_odd_f32", "op": "table_grad", "type": "f32", "tokens": 3001, "dim": 301, "vocab": 10007, "ignored": 0.1},
        # gradient of a large table: some tokens in thousands of places, most rows in none
        {"name": "table_grad_16384", "op": "table_grad", "type": "bf16", "tokens": 16384, "dim": 2048, "vocab": 131072, "ignored": 0.05},
        # a stack of small projections, single precision in
        {"name": "orth_12x128x64_f32", "op": "orth", "type": "f32", "out": "bf16", "batch": 12, "rows": 128, "cols": 64},
        # odd extents, taller than wide
        {"name": "orth_1333x1000_f16", "op": "orth", "type": "f16", "out": "f16", "batch": 1, "rows": 1333, "cols": 1000},
        # the wide projections of several layers
        {"name": "orth_4x1024x4096", "op": "orth", "type": "bf16", "out": "bf16", "batch": 4, "rows": 1024, "cols": 4096},
        # one large square projection
        {"name": "orth_4096x4096", "op": "orth", "type": "bf16", "out": "bf16", "batch": 1, "rows": 4096, "cols": 4096},
    ]


def draw(rng):
    def size(lo, hi):
        """Spread over the logarithm; odd every other time, else a multiple of 8."""
        n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
        return min(hi, n | 1) if rng.random() < 0.5 else max(lo, n // 8 * 8)

    op = rng.choice(["loss", "loss", "lookup", "table_grad", "orth", "orth"])
    if op == "orth":
        kind = rng.choice(["bf16", "f16", "f32"])
        rows, cols = size(16, 4096), size(16, 4096)
        small, large = min(rows, cols), max(rows, cols)
        most = max(1, min(16, int(4096 ** 3 / (small * small * large))))
        return {"op": op, "type": kind, "out": rng.choice(["bf16", "f16"]), "batch": rng.randint(1, most), "rows": rows, "cols": cols}
    ignored = rng.choice([0.0, 0.05, 0.4])
    if op == "loss":
        return {"op": op, "type": rng.choice(["bf16", "bf16", "f16"]), "tokens": size(1, 8192), "dim": size(64, 2048), "vocab": size(1000, 131072),
                "ignored": ignored, "grad": rng.random() < 0.75}
    return {"op": op, "type": rng.choice(["bf16", "f16", "f32"]), "tokens": size(1, 16384), "dim": size(64, 2048), "vocab": size(1000, 65536), "ignored": ignored}


def _tokens(gen, case):
    """Token numbers whose frequencies fall as 1 / rank; -1 where there is none."""
    u = torch.rand(case["tokens"], device="cuda", generator=gen, dtype=torch.float64)
    ids = (torch.exp(u * math.log(case["vocab"])) - 1.0).long().clamp_(0, case["vocab"] - 1)
    if case["ignored"]:
        ids[1:][torch.rand(case["tokens"] - 1, device="cuda", generator=gen) < case["ignored"]] = -1
    return ids


def _inputs(case, seed):
    """The case's inputs, the same for everybody who asks with the same seed."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "orth":
        # a gradient's momentum: a few directions that dominate, and noise
        b, m, n = case["batch"], case["rows"], case["cols"]
        few = max(1, min(m, n) // 16)
        x = normal(b, m, few) @ normal(b, few, n) * (2.0 / few ** 0.5) + normal(b, m, n)
        return {"x": (x * 1e-3).to(kind)}
    if case["op"] == "loss":
        ids = _tokens(gen, case)
        weight = (normal(case["vocab"], case["dim"]) / case["dim"] ** 0.5).to(kind)
        # rows that lean towards their target's, as a trained model's do
        hidden = (normal(case["tokens"], case["dim"]) + 4.0 * weight[ids.clamp(min=0)].float()).to(kind)
        # the gradient of the mean; scaled, as programs do that train in half precision
        n = (ids >= 0).sum().clamp(min=1)
        grad = ((65536.0 if case["type"] == "f16" else 1.0) / n).float().expand(case["tokens"]).contiguous()
        return {"hidden": hidden, "weight": weight, "targets": ids, "grad": grad}
    ids = _tokens(gen, case)
    if case["op"] == "lookup":
        return {"table": normal(case["vocab"], case["dim"]).to(kind), "ids": ids, "scale": math.sqrt(case["dim"])}
    return {"grad": normal(case["tokens"], case["dim"]).to(kind), "ids": ids, "scale": math.sqrt(case["dim"])}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        # the plan and the buffers for results that a program keeps from step to step
        tc = importlib.import_module("cgo2019-ae_b200")
        codes = {"bf16": tc.BF16, "f16": tc.F16, "f32": tc.F32}
        kind, code = TYPES[case["type"]], codes[case["type"]]
        new = lambda *shape, dtype=kind: torch.empty(*shape, device="cuda", dtype=dtype)
        if case["op"] == "orth":
            b, m, n = case["batch"], case["rows"], case["cols"]
            state["plan"] = tc.OrthogonalPlan(m, n, batch=b, dtype=code, out_dtype=codes[case["out"]], steps=STEPS,
                                              coefficients=COEFFICIENTS, eps=EPS).commit()
            state["out"] = new(b, m, n, dtype=TYPES[case["out"]])
        elif case["op"] == "loss":
            t, d, v = case["tokens"], case["dim"], case["vocab"]
            state["plan"] = tc.VocabLossPlan(t, d, v, dtype=code).commit()
            state["loss"], state["lse"] = new(t, dtype=torch.float32), new(t, dtype=torch.float32)
            if case["grad"]:
                state["dhidden"], state["dweight"] = new(t, d), new(v, d)
        else:
            t, d, v = case["tokens"], case["dim"], case["vocab"]
            state["plan"] = tc.EmbeddingPlan(t, v, d, dtype=code, scale=state["scale"]).commit()
            state["out"] = new(t, d) if case["op"] == "lookup" else new(v, d)
    return state


def _orthogonal(x, kind):
    x = x.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum(dim=(1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.transpose(1, 2) if tall else x).to(kind).contiguous()


def _loss(s, with_grad):
    targets, kind = s["targets"], s["hidden"].dtype
    part = targets >= 0
    hidden = torch.where(part[:, None], s["hidden"].float(), 0.0)
    weight = s["weight"].float()
    logits = hidden @ weight.T
    top = logits.amax(dim=1, keepdim=True)
    at = targets.clamp(min=0)[:, None]
    hit = logits.gather(1, at)
    p = logits.sub_(top).exp_()
    total = p.sum(dim=1, keepdim=True)
    lse = top + total.log()
    out = {"loss": torch.where(part, (lse - hit)[:, 0], 0.0), "lse": torch.where(part, lse[:, 0], 0.0)}
    if with_grad:
        p = p.div_(total).scatter_add_(1, at, torch.full_like(hit, -1.0))
        p = p.mul_(torch.where(part, s["grad"], 0.0)[:, None])
        out["dhidden"], out["dweight"] = (p @ weight).to(kind), (p.T @ hidden).to(kind)
    return out


def run(state):
    case = state["case"]
    if case["op"] == "orth":
        if not own:
            return _orthogonal(state["x"], TYPES[case["out"]])
        state["plan"].execute(state["out"], state["x"])
        return state["out"]
    if case["op"] == "loss":
        if not own:
            return _loss(state, case["grad"])
        state["plan"].execute(state["loss"], state["lse"], state["hidden"], state["weight"], state["targets"])
        if not case["grad"]:
            return {"loss": state["loss"], "lse": state["lse"]}
        state["plan"].execute_grad(state["dhidden"], state["dweight"], state["hidden"], state["weight"], state["targets"], state["lse"], state["grad"])
        return {k: state[k] for k in ("loss", "lse", "dhidden", "dweight")}
    if case["op"] == "lookup":
        if own:
            state["plan"].execute(state["out"], state["table"], state["ids"])
            return state["out"]
        rows = state["table"][state["ids"].clamp(min=0)].float() * state["scale"]
        return torch.where((state["ids"] >= 0)[:, None], rows, 0.0).to(state["table"].dtype)
    if own:
        state["plan"].execute_grad(state["out"], state["grad"], state["ids"])
        return state["out"]
    rows = torch.where((state["ids"] >= 0)[:, None], state["grad"].float() * state["scale"], 0.0)
    table = torch.zeros(case["vocab"], case["dim"], device="cuda")
    return table.index_add_(0, state["ids"].clamp(min=0), rows).to(state["grad"].dtype)


def work(case):
    es = 4 if case["type"] == "f32" else 2
    if case["op"] == "orth":
        b, small, large = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        # per step two products whose result is symmetric, of which half is needed, and one that is not
        step = small * small * large + small ** 3 + 2 * small * small * large
        return {"bytes": b * small * large * (es + 2), "flops": b * STEPS * step}
    t, d, v = case["tokens"], case["dim"], case["vocab"]
    part = max(1, round(t * (1.0 - case["ignored"])))
    if case["op"] == "loss":
        # one product for the logits; one more for each gradient
        n = 3 if case["grad"] else 1
        return {"bytes": es * d * (part + v) + 16 * t + (es * d * (t + v) + 4 * t if case["grad"] else 0), "flops": 2 * n * part * d * v}
    if case["op"] == "lookup":
        return {"bytes": es * d * (min(part, v) + t) + 8 * t, "flops": t * d}
    return {"bytes": es * d * (part + v) + 8 * t, "flops": part * d}


def _exact_loss(s, with_grad):
    """Over pieces of the vocabulary: the sum first, then each piece's probabilities again."""
    targets = s["targets"]
    t, (v, d) = targets.shape[0], s["weight"].shape
    kept = torch.nonzero(targets >= 0)[:, 0]
    h = s["hidden"][kept].double()
    goal = targets[kept]
    piece = max(1, min(v, (1 << 27) // max(1, kept.numel())))
    sums, top = [], []
    for at in range(0, v, piece):
        z = h @ s["weight"][at:at + piece].double().T
        top.append(z.amax(dim=1))
        sums.append((z - top[-1][:, None]).exp().sum(dim=1).log() + top[-1])
    lse_kept = torch.logsumexp(torch.stack(sums), dim=0)
    hit = (h * s["weight"][goal].double()).sum(dim=1)
    loss, lse = (torch.zeros(t, dtype=torch.float64, device="cuda") for _ in range(2))
    loss[kept], lse[kept] = lse_kept - hit, lse_kept
    out = {"loss": loss, "lse": lse}
    if with_grad:
        g = s["grad"][kept].double()
        dh = torch.zeros_like(h)
        dw = torch.empty(v, d, dtype=torch.float64, device="cuda")
        for at in range(0, v, piece):
            w = s["weight"][at:at + piece].double()
            p = (h @ w.T - lse_kept[:, None]).exp()
            here = torch.nonzero((goal >= at) & (goal < at + w.shape[0]))[:, 0]
            p[here, goal[here] - at] -= 1.0
            p *= g[:, None]
            dh += p @ w
            dw[at:at + w.shape[0]] = p.T @ h
        out["dhidden"] = torch.zeros(t, d, dtype=torch.float64, device="cuda")
        out["dhidden"][kept] = dh
        out["dweight"] = dw
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "loss":
        return _exact_loss(s, case["grad"])
    if case["op"] == "orth":
        # on the singular values: the iteration is an odd polynomial of each
        out = []
        for x in s["x"].double():
            wide = x if x.shape[0] <= x.shape[1] else x.T
            start = 1.0 / (torch.linalg.matrix_norm(wide) + EPS)
            # f(X) = p(X X^T) X with a polynomial p of eigenvalues of X X^T: X's own small directions stay what they are
            values, vectors = torch.linalg.eigh(wide @ wide.T * start ** 2)
            sigma = values.clamp(min=0.0).sqrt()
            factor = torch.ones_like(sigma)  # of sigma, after the steps so far
            a, b, c = COEFFICIENTS
            for _ in range(STEPS):
                square = (factor * sigma) ** 2
                factor = factor * (a + b * square + c * square ** 2)
            y = vectors @ ((vectors.T @ wide) * (factor * start)[:, None])
            out.append(y if wide is x else y.T)
        return torch.stack(out)
    kept = torch.nonzero(s["ids"] >= 0)[:, 0]
    if case["op"] == "lookup":
        out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
        out[kept] = s["table"][s["ids"][kept]].double() * s["scale"]
        return out
    out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
    return out.index_put_((s["ids"][kept],), s["grad"][kept].double() * s["scale"], accumulate=True)
