"""The operators around the contractions inside of a model's block, as measurable cases.

A block of a model is contractions with little between them: a norm before and after, gated and scaled onto the residual stream
(`ResidualNormPlan`); operands in microscaled 4-bit floating point and the product of two such matrices (`MicroscalePlan`,
`MicroProductPlan`); and an activation function whose input is kept in 8 bits until the backward pass reads it
(`CheckpointPlan`).  A case is one pass through one of them.  With `own` false the same results come from elementary torch
operations in 32 bits.

Microscaled numbers come in blocks of 32 along a row that share a scale 2^e, the smallest (from 2^-127 on) for which no value
of the block exceeds the largest element: 6 of it where elements are e2m1 (4 bits), 448 where they are e4m3 (8 bits).
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
RESIDUAL_SCALE = 0.875


def listed():
    return [
        # weights laid out for their gradient's product: quantised along the other index, nothing a multiple of anything
        {"name": "quantise_odd_f16", "op": "quantise", "type": "f16", "rows": 1001, "cols": 1777, "transposed": True},
        # the activations of a batch of sequences before a 4-bit product
        {"name": "quantise_8192x4096", "op": "quantise", "type": "bf16", "rows": 8192, "cols": 4096, "transposed": False},
        # the next token of one sequence through a square projection: the weights' bytes
        {"name": "linear_1x4096x4096", "op": "linear", "type": "bf16", "out": "bf16", "tokens": 1, "outputs": 4096, "inner": 4096},
        # odd extents, results in single precision
        {"name": "linear_odd_f16", "op": "linear", "type": "f16", "out": "f32", "tokens": 333, "outputs": 1001, "inner": 777},
        # a training step's batch through a wide projection
        {"name": "linear_8192x8192x4096", "op": "linear", "type": "bf16", "out": "bf16", "tokens": 8192, "outputs": 8192, "inner": 4096},
        # a gated activation, forward and backward, of a training step's batch
        {"name": "act_gated_8192", "op": "act", "type": "bf16", "tokens": 8192, "dim": 4096, "activation": "silu", "gated": True},
        # a small batch in single precision, odd rows
        {"name": "act_odd_f32", "op": "act", "type": "f32", "tokens": 513, "dim": 1111, "activation": "gelu", "gated": False},
        # the weight gradient of the projection behind the activation, whose input is computed again from the 8 bits
        {"name": "weight_8192x4096x2048", "op": "weight", "type": "bf16", "tokens": 8192, "dim": 4096, "outputs": 2048, "activation": "silu", "gated": False},
        # the weight gradient of a projection whose own input was kept, odd extents
        {"name": "weight_odd_f16", "op": "weight", "type": "f16", "tokens": 1023, "dim": 777, "outputs": 555, "activation": "none", "gated": False},
        # the next token of one sequence: latency
        {"name": "norm_1x4096", "op": "norm", "type": "bf16", "tokens": 1, "dim": 4096, "gate": "channel", "grad": False},
        # single precision, odd rows, a gate of its own for each token, forward and backward
        {"name": "norm_odd_f32", "op": "norm", "type": "f32", "tokens": 777, "dim": 1003, "gate": "token", "grad": True},
        # forward and backward of a training step's batch
        {"name": "norm_train_8192", "op": "norm", "type": "bf16", "tokens": 8192, "dim": 4096, "gate": "channel", "grad": True},
    ]


def draw(rng):
    def size(lo, hi):
        """Spread over the logarithm; odd every other time, else a multiple of 8."""
        n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
        return min(hi, n | 1) if rng.random() < 0.5 else max(lo, n // 8 * 8)

    op = rng.choice(["quantise", "linear", "linear", "act", "weight", "norm", "norm"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    tokens = size(1, 8192)
    if op == "quantise":
        return {"op": op, "type": kind, "rows": tokens, "cols": size(16, 8192), "transposed": rng.random() < 0.5}
    if op == "linear":
        return {"op": op, "type": kind, "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "tokens": tokens, "outputs": size(64, 8192), "inner": size(64, 4096)}
    activation, gated = rng.choice(["silu", "gelu"]), rng.random() < 0.5
    if op == "act":
        return {"op": op, "type": kind, "tokens": tokens, "dim": size(16, 4096), "activation": activation, "gated": gated}
    if op == "weight":
        plain = rng.random() < 0.5
        return {"op": op, "type": "bf16" if kind == "f32" else kind, "tokens": tokens, "dim": size(64, 4096), "outputs": size(64, 4096),
                "activation": "none" if plain else activation, "gated": gated and not plain}
    return {"op": op, "type": kind, "tokens": tokens, "dim": size(16, 8192 if kind != "f32" else 4096), "gate": rng.choice(["none", "channel", "token"]),
            "grad": rng.random() < 0.6}


# ---- microscaled numbers, plainly ----
def _power(e):
    """2^e of whole numbers above -150, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64).float()


def _blocks(x):
    """[rows, cols] in 32 bits as [rows, blocks, 32], the last block filled up with zeros."""
    return torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))


def _scales(b, share, exponent):
    """e of each block, where the largest element is share * 2^exponent (1/2 <= share < 1)."""
    m, e = torch.frexp(b.abs().amax(dim=2))
    return torch.where(m > 0, e - exponent + (m > share).int(), -127).clamp(min=-127)


def _e2m1(v):
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(v / step) * step


def _e4m3(v):
    step = _power(torch.frexp(v)[1].clamp(min=-5) - 4)
    return torch.round(v / step) * step


def _micro4(x):
    """[rows, cols] rounded to microscaled 4-bit numbers, in 32 bits."""
    b = _blocks(x)
    s = _power(_scales(b, 0.75, 3))[:, :, None]
    return (_e2m1(b / s) * s).flatten(1)[:, :x.shape[1]]


def _micro8(x):
    b = _blocks(x)
    s = _power(_scales(b, 0.875, 9))[:, :, None]
    return (_e4m3(b / s) * s).flatten(1)[:, :x.shape[1]]


E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _pack(w):
    """Codes [rows, 16 * blocks] (two elements a byte, the first in the low half) and scales (e + 127) of a matrix, the scales in
    pieces of 128 rows by 4 blocks: [rows / 128, blocks / 4, 32, 4, 4] with row 32 j + i of a piece at [i, j]."""
    b = _blocks(w)
    e = _scales(b, 0.75, 3)
    v = _e2m1(b / _power(e)[:, :, None])
    code = torch.bucketize(v.abs(), torch.tensor(E2M1, device=w.device)).to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
    codes = (code[:, :, 0::2] + 16 * code[:, :, 1::2]).flatten(1).contiguous()
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -e.shape[1] % 4, 0, -e.shape[0] % 128))
    scales = scales.unflatten(1, (-1, 4)).unflatten(0, (-1, 4, 32)).permute(0, 3, 2, 1, 4).contiguous()
    return codes, scales


def _unpack(codes, scales, cols):
    """The 32-bit values that packed codes and scales stand for."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], dim=2).flatten(1).unflatten(1, (-1, 32))
    e = scales.permute(0, 3, 2, 1, 4).flatten(3, 4).flatten(0, 2)[:v.shape[0], :v.shape[1]].long() - 127
    return (v * _power(e)[:, :, None]).flatten(1)[:, :cols]


# ---- inputs ----
def _inputs(case, seed):
    """The case's inputs, the same for everybody who asks with the same seed."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def activations(rows, cols):
        """Some columns far larger than the rest, as a model's activations have."""
        return normal(rows, cols) * (1.0 + 8.0 * (torch.rand(cols, device="cuda", generator=gen) < 0.02).float())

    if case["op"] == "quantise":
        x = activations(case["rows"], case["cols"]).to(kind)
        return {"x": x.T.contiguous() if case["transposed"] else x}
    if case["op"] == "linear":
        codes, scales = _pack(normal(case["outputs"], case["inner"]) / case["inner"] ** 0.5)
        return {"x": activations(case["tokens"], case["inner"]).to(kind), "codes": codes, "scales": scales}
    t, d = case["tokens"], case["dim"]
    if case["op"] in ("act", "weight"):
        width = d * (2 if case["gated"] else 1)
        out = d if case["op"] == "act" else case["outputs"]
        return {"x": activations(t, width).to(kind), "dy": (normal(t, out) * 1e-2).to(kind)}
    s = {"x": activations(t, d).to(kind), "f": (normal(t, d) * 0.3).to(kind), "post": (1.0 + 0.1 * normal(d)).to(kind), "pre": (1.0 + 0.1 * normal(d)).to(kind)}
    if case["gate"] != "none":
        s["gate"] = torch.sigmoid(normal(*((d,) if case["gate"] == "channel" else (t, d)))).to(kind)
    if case["grad"]:
        s["dh"], s["dn"] = (normal(t, d) * 1e-2).to(kind), (normal(t, d) * 1e-2).to(kind)
    return s


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        # the plans and the buffers that a program keeps from step to step
        tc = importlib.import_module("cgo2019-ae_b200")
        number = {"bf16": tc.BF16, "f16": tc.F16, "f32": tc.F32}
        kind, code = TYPES[case["type"]], number[case["type"]]
        new = lambda *shape, dtype=kind: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
        small = lambda shapes: tuple(new(*shape, dtype=torch.uint8) for shape in shapes)  # noqa: E731
        if case["op"] == "quantise":
            plan = state["plan"] = tc.MicroscalePlan(case["rows"], case["cols"], dtype=code).commit()
            state["kept"], state["out"] = small((plan.codes_shape, plan.scales_shape)), new(case["rows"], case["cols"])
        elif case["op"] == "linear":
            t, n, k = case["tokens"], case["outputs"], case["inner"]
            plan = state["plan"] = tc.MicroscalePlan(t, k, dtype=code).commit()
            state["kept"] = small((plan.codes_shape, plan.scales_shape))
            state["product"] = tc.MicroProductPlan(t, n, k, out_dtype=number[case["out"]]).commit()
            state["out"] = new(t, n, dtype=TYPES[case["out"]])
        elif case["op"] in ("act", "weight"):
            t, d = case["tokens"], case["dim"]
            plan = state["plan"] = tc.CheckpointPlan(t, d, dtype=code, activation=case["activation"], gated=case["gated"]).commit()
            state["kept"] = small((plan.codes_shape, plan.scales_shape))
            if case["op"] == "act":
                state["out"] = {"y": new(t, d), "dx": new(*state["x"].shape)}
            else:
                state["out"] = new(case["outputs"], d)
        else:
            t, d = case["tokens"], case["dim"]
            state["plan"] = tc.ResidualNormPlan(t, d, dtype=code, gate=case["gate"], residual_scale=RESIDUAL_SCALE, eps=EPS).commit()
            state["out"] = {"h": new(t, d), "n": new(t, d)}
            if case["grad"]:
                state["out"].update({"dx": new(t, d), "df": new(t, d), "dpost": new(d), "dpre": new(d)})
                if case["gate"] != "none":
                    state["out"]["dgate"] = new(*state["gate"].shape)
    return state


# ---- the passes ----
def _activate(case, x):
    """An activation's result and its derivative by each half of x (by x where there is no gate)."""
    a = x[:, :case["dim"]]
    if case["activation"] == "silu":
        share = 1.0 / (1.0 + torch.exp(-a))
        f, slope = a * share, share * (1.0 + a * (1.0 - share))
    elif case["activation"] == "gelu":
        share = 0.5 * torch.erfc(a * -(0.5 ** 0.5))
        f, slope = a * share, share + a * torch.exp(-0.5 * a * a) * (0.5 / math.pi) ** 0.5
    else:
        f, slope = a, torch.ones_like(a)
    if not case["gated"]:
        return f, slope
    b = x[:, case["dim"]:]
    return f * b, torch.cat([slope * b, f], dim=1)


def _kept8(case, x):
    """What is left of an activation's input in 8 bits: each half has blocks of its own."""
    return torch.cat([_micro8(x[:, :case["dim"]]), _micro8(x[:, case["dim"]:])], dim=1) if case["gated"] else _micro8(x)


def _norm(s, case):
    kind, d = s["x"].dtype, case["dim"]
    x, f, post, pre = (s[k].float() for k in ("x", "f", "post", "pre"))
    gate = s["gate"].float() if "gate" in s else torch.ones_like(post)
    r = torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS)
    u = f * r
    h = RESIDUAL_SCALE * x + gate * (u * post)
    n = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * pre
    out = {"h": h.to(kind), "n": n.to(kind)}
    if case["grad"]:
        # at h as it was stored
        h, dn = out["h"].float(), s["dn"].float()
        q = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
        v = h * q
        dh = s["dh"].float() + q * (dn * pre - v * (dn * pre * v).mean(dim=1, keepdim=True))
        dp = dh * gate
        out["df"] = (r * (dp * post - u * (dp * post * u).mean(dim=1, keepdim=True))).to(kind)
        out["dx"] = (RESIDUAL_SCALE * dh).to(kind)
        out["dpost"], out["dpre"] = (dp * u).sum(dim=0).to(kind), (dn * v).sum(dim=0).to(kind)
        if "gate" in s:
            dgate = dh * u * post
            out["dgate"] = (dgate if case["gate"] == "token" else dgate.sum(dim=0)).to(kind)
    return out


def run(state):
    case = state["case"]
    if case["op"] == "quantise":
        if not own:
            return _micro4(state["x"].T if case["transposed"] else state["x"]).to(state["x"].dtype)
        state["plan"].execute(*state["kept"], state["x"], transposed=case["transposed"])
        state["plan"].restore(state["out"], *state["kept"])
        return state["out"]
    if case["op"] == "linear":
        if not own:
            return (_micro4(state["x"]) @ _unpack(state["codes"], state["scales"], case["inner"]).T).to(TYPES[case["out"]])
        state["plan"].execute(*state["kept"], state["x"])
        state["product"].execute(state["out"], *state["kept"], state["codes"], state["scales"])
        return state["out"]
    if case["op"] == "act":
        if own:
            # the input in 8 bits and the result; on the way back the input's gradient from those
            state["plan"].execute(*state["kept"], state["x"], y=state["out"]["y"])
            state["plan"].execute_grad(state["out"]["dx"], *state["kept"], state["dy"])
            return state["out"]
        y = _activate(case, state["x"].float())[0]
        slope = _activate(case, _kept8(case, state["x"]))[1]
        dy = state["dy"].float()
        return {"y": y.to(state["x"].dtype), "dx": (slope * (torch.cat([dy, dy], dim=1) if case["gated"] else dy)).to(state["x"].dtype)}
    if case["op"] == "weight":
        if own:
            state["plan"].execute(*state["kept"], state["x"])
            state["plan"].execute_product(state["out"], state["dy"], *state["kept"])
            return state["out"]
        return (state["dy"].float().T @ _activate(case, _kept8(case, state["x"]))[0]).to(state["x"].dtype)
    if not own:
        return _norm(state, case)
    o, gate = state["out"], state.get("gate")
    state["plan"].execute(o["h"], o["n"], state["x"], state["f"], state["post"], state["pre"], gate=gate)
    if case["grad"]:
        state["plan"].execute_grad(o["dx"], o["df"], o["dpost"], o["dpre"], state["dh"], state["dn"], o["h"], state["f"], state["post"], state["pre"],
                                   gate=gate, dgate=o.get("dgate"))
    return o


def work(case):
    es = 4 if case["type"] == "f32" else 2
    if case["op"] == "quantise":
        values = case["rows"] * case["cols"]
        # in, the codes, and out again
        return {"bytes": values * (2 * es + 2 * (0.5 + 1 / 32)), "flops": 4 * values}
    if case["op"] == "linear":
        t, n, k = case["tokens"], case["outputs"], case["inner"]
        return {"bytes": t * k * es + n * k * (0.5 + 1 / 32) + t * n * (4 if case["out"] == "f32" else 2), "flops": 2 * t * n * k}
    t, d = case["tokens"], case["dim"]
    if case["op"] in ("act", "weight"):
        parts = 2 if case["gated"] else 1
        kept = t * d * parts * (1 + 1 / 32)
        if case["op"] == "act":
            return {"bytes": 2 * kept + t * d * es * (2 * parts + 2), "flops": 20 * t * d}
        n = case["outputs"]
        return {"bytes": 2 * kept + t * d * parts * es + (t + d) * n * es, "flops": 2 * t * d * n}
    gate = {"none": 0, "channel": d, "token": t * d}[case["gate"]]
    # forward x, f, h, n; backward dh, dn, h, f, dx, df
    return {"bytes": es * (t * d * (10 if case["grad"] else 4) + (3 if case["grad"] else 1) * gate + (6 if case["grad"] else 2) * d), "flops": t * d * (40 if case["grad"] else 10)}


# ---- the definitions in 64 bits ----
def _nearest(v, values):
    """The nearest of ascending non-negative values by magnitude, the one at an even place where two are."""
    values = torch.tensor(values, dtype=torch.float64, device=v.device)
    middle = (values[1:] + values[:-1]) / 2
    at = torch.searchsorted(middle, v.abs(), right=False)
    tie = (at < middle.numel()) & (middle[at.clamp(max=middle.numel() - 1)] == v.abs()) & (at % 2 == 1)
    return torch.where(v < 0, -1.0, 1.0) * values[(at + tie.long()).clamp(max=values.numel() - 1)]


def _two_to(e):
    """Powers of two by a table: the device's functions may be a last place off."""
    return torch.tensor([2.0 ** k for k in range(-200, 201)], dtype=torch.float64, device=e.device)[e.long() + 200]


def _exact_micro(x, values):
    rows, cols = x.shape
    x = torch.cat([x.double(), torch.zeros(rows, -cols % 32, dtype=torch.float64, device=x.device)], dim=1).view(rows, -1, 32)
    top = x.abs().amax(dim=2, keepdim=True) / values[-1]
    e = torch.where(top > 0, torch.ceil(torch.log2(torch.where(top > 0, top, 1.0))), -127.0)
    # where the logarithm was rounded over a whole number
    e = torch.where(_two_to(e) < top, e + 1, torch.where((_two_to(e - 1) >= top) & (top > 0), e - 1, e)).clamp(min=-127.0)
    s = _two_to(e)
    return (_nearest(x / s, values) * s).view(rows, -1)[:, :cols]


def _e4m3_values():
    return [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]


def _exact_weights(codes, scales, rows, cols):
    code = torch.stack([codes & 15, codes >> 4], dim=2).view(rows, -1).long()[:, :cols]
    size = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)[code & 7] * torch.where(code > 7, -1.0, 1.0)
    row, block = torch.arange(rows, device=codes.device)[:, None], torch.arange(-(-cols // 32), device=codes.device)[None]
    e = scales[row // 128, block // 4, row % 32, row % 128 // 32, block % 4].double() - 127
    return size * _two_to(e).repeat_interleave(32, dim=1)[:, :cols]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quantise":
        return _exact_micro(s["x"].T if case["transposed"] else s["x"], E2M1)
    if case["op"] == "linear":
        return _exact_micro(s["x"], E2M1) @ _exact_weights(s["codes"], s["scales"], case["outputs"], case["inner"]).T
    if case["op"] in ("act", "weight"):
        def function(x):
            a, b = (x[:, :case["dim"]], x[:, case["dim"]:]) if case["gated"] else (x, 1.0)
            return b * (a * torch.sigmoid(a) if case["activation"] == "silu" else a * torch.special.ndtr(a) if case["activation"] == "gelu" else a)

        x = s["x"].double()
        kept = torch.cat([_exact_micro(p, _e4m3_values()) for p in x.split(case["dim"], dim=1)], dim=1)
        if case["op"] == "weight":
            return s["dy"].double().T @ function(kept)
        kept.requires_grad_()
        return {"y": function(x), "dx": torch.autograd.grad(function(kept), kept, s["dy"].double())[0]}
    part = {k: v.double().requires_grad_(case["grad"]) for k, v in s.items() if k in ("x", "f", "post", "pre", "gate")}

    def unit(v):
        return v / (v.square().mean(dim=1, keepdim=True) + EPS).sqrt()

    h = RESIDUAL_SCALE * part["x"] + part.get("gate", 1.0) * (unit(part["f"]) * part["post"])
    out = {"h": h.detach(), "n": (unit(h) * part["pre"]).detach()}
    if case["grad"]:
        stored = h + (h.detach().to(s["x"].dtype).double() - h.detach())
        names = sorted(part)
        grads = torch.autograd.grad([stored, unit(stored) * part["pre"]], [part[k] for k in names], [s["dh"].double(), s["dn"].double()])
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out
