"""The operators inside of a model's block where their other kernels run: several rows a thread, several rows and tiles a block, sums and
rows of every length; and the precision of what they keep.  Sizes follow the rules of the sources by the device's multiprocessors."""
import pytest
import torch

from test_block_operators import (Block, block_inputs, E2M1, E4M3, EPS, TYPES, activate, code, function, kept, micro, micro_values, new_gen, norm_inputs,
                                  norm_reference, norm_share, pack4, product_bound, product_case, quantised, randn, rounded, rows_apart, spread, tail, tiny, unit,
                                  within)


def multiprocessors():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ------------------------------------------------------------------------------------------- several rows a thread ----
def many_rows(cols):
    """Rows from which on a thread takes several, and three more: the last group is filled partly."""
    rows = -(-16 * 16 * multiprocessors() // -(-cols // 128))
    return rows // 4 * 4 + 7


MANY = [("bf16", 256, 0), ("f16", 250, 0), ("f32", 256, 4), ("bf16", 136, 1), ("f32", 131, 0), ("f16", 512, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cols,extra", MANY)
def test_microscaled_numbers_of_many_rows(pkg, kind, cols, extra):
    rows = many_rows(cols)
    x = spread(new_gen(cols), rows, cols, kind)
    x[::7, ::3] = 0
    plan, codes, scales = quantised(pkg, rows_apart(x, extra, 3.0), kind)
    want, want_scales = micro(x, E2M1)
    want4, laid_out = pack4(want, want_scales)
    assert torch.equal(codes, want4) and torch.equal(scales, laid_out)
    back = torch.full((rows, cols + extra), 7.0, device="cuda").to(TYPES[kind])
    plan.restore(back[:, :cols], codes, scales)
    assert torch.equal(back[:, :cols].double(), micro_values(want, want_scales, E2M1, cols)) and bool((back[:, cols:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cols,extra", MANY)
@pytest.mark.parametrize("name,gated", [("none", False), ("silu", True), ("gelu", False)])
def test_kept_activations_of_many_rows(pkg, kind, cols, extra, name, gated):
    tokens, dim, parts = many_rows(cols), cols, 2 if gated else 1
    gen = new_gen(cols + parts)
    x, dy = spread(gen, tokens, parts * dim, kind), randn(gen, tokens, dim).to(TYPES[kind])
    plan = pkg.CheckpointPlan(tokens, dim, dtype=code(pkg, kind), activation=name, gated=gated)
    codes, scales = (torch.full(s, 0xA5, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    y, dx = (torch.full((tokens, n + extra), 7.0, device="cuda").to(TYPES[kind]) for n in (dim, parts * dim))
    plan.execute(codes, scales, rows_apart(x, extra, 3.0), y=y[:, :dim])
    parts_of = [micro(p, E4M3) for p in x.chunk(parts, dim=1)]
    assert torch.equal(codes, torch.cat([c.flatten(1) for c, _ in parts_of], dim=1).to(torch.uint8))
    assert torch.equal(scales, torch.cat([s for _, s in parts_of], dim=1).to(torch.uint8))
    share = 1.01 * unit(kind) + FINE[name]
    ref = function(name, gated, x.double())
    within(y[:, :dim], ref, share * ref.abs() + tiny(kind) + tail(x, gated), "result")
    v = kept(x, gated).requires_grad_()
    ref = function(name, gated, v)
    plan.restore(y[:, :dim], codes, scales)
    within(y[:, :dim], ref.detach(), share * ref.detach().abs() + tiny(kind) + tail(v.detach(), gated), "restored")
    plan.execute_grad(dx[:, :parts * dim], codes, scales, rows_apart(dy, extra))
    want, = torch.autograd.grad(ref, v, dy.double())
    within(dx[:, :parts * dim], want, 1.01 * unit(kind) * want.abs() + gradient_terms(name, gated, v.detach(), dy.double()) + tiny(kind), "gradient")
    assert bool((y[:, dim:] == 7.0).all()) and bool((dx[:, parts * dim:] == 7.0).all())


# Relative errors of the fp32 arithmetic, in units of 2^-24: the device's exponential of half the exponent is off by 2^-22.5 relative to itself
# (5.7 units in its square), its reciprocal by 2.
#   silu   the square and the correction by the exponent's rest 2, 1 + t 1, the reciprocal 2, two products 2: 13
#   gelu   the exponential with two corrections 9; q = 1 / (z + k) 3; u = 1 - 5 q off by up to 7 of its own unit, at which the polynomial's
#          logarithm has a slope of at most 0.6: 4; the polynomial 2 and its fit 1; three products 3: 22
FINE = {"none": 0.0, "silu": 13 * 2.0 ** -24, "gelu": 22 * 2.0 ** -24}


def gradient_terms(name, gated, v, dy):
    """What an activation's gradient may be off by beside its rounding: its slope is a sum of f(a) / a and a term a s(-a), or a times
    the normal density, each off by its share; the product with the other half and with dy two roundings more."""
    a = v[:, :dy.shape[1]]
    if name == "none":
        slope, share = torch.ones_like(a), 2.0 ** -23
    else:
        s = torch.sigmoid(a) if name == "silu" else 0.5 * torch.erfc(a * -(0.5 ** 0.5))
        rest = a.abs() * s * torch.sigmoid(-a) if name == "silu" else a.abs() * torch.exp(-0.5 * a * a) * 0.3989422804014327
        slope, share = s + rest, FINE[name] + 4 * 2.0 ** -24
    # both terms of a slope far out on the left may be subnormal in fp32
    low = 0.0 if name == "none" else (1 + a.abs()) * 2.0 ** -149
    if not gated:
        return dy.abs() * (share * slope + low)
    b, f = v[:, dy.shape[1]:].abs(), activate(name, a).abs()
    # the product with b rounds a subnormal number to a multiple of 2^-149, before the one with dy
    return torch.cat([dy.abs() * (b * (share * slope + low) + 2.0 ** -150), dy.abs() * (share * f + tail(a, False))], dim=1)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_activations_to_their_last_places(pkg, name):
    """In single precision over the whole line; the gradient at what eight bits hold."""
    n = 1 << 15
    x = torch.cat([torch.linspace(-110.0, 110.0, 4 * n), torch.linspace(-6.0, 6.0, 4 * n), torch.logspace(-30, 2, 2 * n), -torch.logspace(-30, 2, 2 * n)]).view(-1, 32).cuda()
    plan = pkg.CheckpointPlan(x.shape[0], 32, dtype=pkg.F32, activation=name)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    plan.execute(codes, scales, x, y=y)
    ref = activate(name, x.double())
    within(y, ref, FINE[name] * ref.abs() + tiny("f32") + tail(x, False), "result")
    v, dy = kept(x, False).requires_grad_(), torch.ones_like(x)
    plan.execute_grad(dx, codes, scales, dy)
    want, = torch.autograd.grad(activate(name, v).sum(), v)
    within(dx, want, 2.0 ** -24 * want.abs() + gradient_terms(name, False, v.detach(), dy.double()) + tiny("f32"), "slope")


# ---------------------------------------------------------------------------------- the weight's gradient, precisely ----
PRECISE = [  # tokens, dim, outputs, type, activation, gated, elements behind each row of dy, gradient's type
    (1, 33, 5, "bf16", "silu", True, 0, "f32"), (4, 520, 136, "bf16", "gelu", True, 8, "bf16"), (64, 300, 257, "f16", "silu", False, 1, "f32"),
    (500, 2100, 1030, "bf16", "silu", True, 0, "f32"), (1000, 256, 256, "f16", "gelu", False, 0, "f16"), (3000, 200, 1033, "f16", "gelu", True, 0, "f32"),
    (2048, 1024, 512, "bf16", "silu", False, 0, "f32"), (4096, 100, 130, "bf16", "none", True, 1, "f32"), (4000, 64, 72, "bf16", "silu", False, 0, "bf16"),
    (1500, 3000, 2504, "bf16", "gelu", False, 0, "f32"), (130, 72, 64, "f16", "none", False, 0, "f32")]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,outputs,kind,name,gated,extra,out", PRECISE)
def test_weight_gradient_takes_the_function_as_it_is(pkg, tokens, dim, outputs, kind, name, gated, extra, out):
    """Tokens that are all alike, so that roundings of the function's value add up as its value does."""
    gen = new_gen(tokens + dim + outputs)
    x = randn(gen, 1, dim * (2 if gated else 1)).to(TYPES[kind]).expand(tokens, -1).contiguous()
    dy = (1 + 0.5 * torch.rand(1, outputs, device="cuda", generator=gen)).to(TYPES[kind]).expand(tokens, -1).contiguous()
    plan = pkg.CheckpointPlan(tokens, dim, dtype=code(pkg, kind), activation=name, gated=gated)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    plan.execute(codes, scales, x)
    f = function(name, gated, kept(x, gated))
    ref, size = dy.double().T @ f, dy.double().abs().T @ f.abs()
    # the value is the sum of two numbers of the operands' type: off by a rounding of what the first leaves
    share = 0.0 if name == "none" and not gated else 1.01 * unit(kind) ** 2 + FINE[name] + 2.0 ** -24
    tol = (2 * tokens * 2.0 ** -23 + share) * size + tokens * dy.double().abs().max() * tiny(kind)
    dw = torch.empty(outputs, dim, device="cuda", dtype=TYPES[out])
    plan.execute_product(dw, rows_apart(dy, extra), codes, scales)
    within(dw, ref, tol + 1.01 * unit(out) * (ref.abs() + tol) + tiny(out), "weight")
    assert plan.status() == 0


# ------------------------------------------------------------------------------------- several rows and tiles a block ----
RINGS = [  # dim, type, type of the weights, gate, elements behind each row
    (96, "bf16", "bf16", "channel", 0), (96, "f16", "f32", "none", 0), (200, "bf16", "bf16", "token", 0), (400, "f16", "f16", "channel", 0), (400, "bf16", "f32", "token", 8),
    (1024, "bf16", "bf16", "none", 0), (1024, "bf16", "bf16", "channel", 0), (1032, "f16", "f16", "token", 0), (136, "f32", "f32", "channel", 0), (600, "f32", "f32", "token", 0),
    (4104, "bf16", "f32", "channel", 0), (8192, "bf16", "bf16", "token", 0), (4096, "f32", "f32", "token", 0), (16384, "f32", "f32", "token", 0), (16384, "bf16", "bf16", "channel", 0),
    # unaligned
    (5, "bf16", "bf16", "token", 0), (97, "f16", "f16", "channel", 0), (301, "f32", "f32", "token", 2), (2051, "f16", "f16", "none", 0), (2051, "f16", "f16", "channel", 0),
    (2051, "f16", "f32", "token", 0), (1003, "f32", "f32", "none", 0), (1003, "f32", "f32", "channel", 0), (1003, "f32", "f32", "token", 0), (1024, "bf16", "bf16", "channel", 1),
    (8191, "bf16", "bf16", "token", 0), (4095, "f32", "f32", "token", 0), (9001, "f32", "f32", "token", 0), (9001, "bf16", "bf16", "token", 0), (16383, "f32", "f32", "token", 0),
    (16383, "bf16", "bf16", "none", 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kind,wkind,gate,extra", RINGS)
def test_norms_whose_blocks_take_several_rows(pkg, dim, kind, wkind, gate, extra):
    """Three rows and more for each block that the device holds at most: 32 of one warp a multiprocessor, a warp for every 256 columns at least."""
    gen = new_gen(dim)
    warps = max(1, -(-dim // 1024))  # four pieces of eight columns a lane
    tokens = 3 * multiprocessors() * min(32, max(1, 32 // warps)) + 2
    s = norm_inputs(gen, tokens, dim, kind, wkind, gate)
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=code(pkg, kind), gate=gate, residual_scale=0.75, eps=EPS, weight_dtype=code(pkg, wkind))
    wide = {k: torch.full((tokens, dim + extra), 7.0, device="cuda").to(TYPES[kind]) for k in ("h", "n", "dx", "df", "dgate")}
    o = {k: v[:, :dim] for k, v in wide.items()}
    far = {k: v if v is None or v.ndim == 1 else rows_apart(v, extra, 5.0) for k, v in s.items()}
    plan.execute(o["h"], None, far["x"], far["f"], s["post"], s["pre"], gate=far["gate"])
    alone = o["h"].clone()
    o["h"].fill_(7.0)
    plan.execute(o["h"], o["n"], far["x"], far["f"], s["post"], s["pre"], gate=far["gate"])
    assert torch.equal(alone, o["h"])
    if gate != "token":
        o["dgate"] = torch.empty(dim, device="cuda", dtype=TYPES[kind]) if gate == "channel" else None
    vectors = {k: torch.empty(dim, device="cuda", dtype=TYPES[wkind]) for k in ("dpost", "dpre")}
    plan.execute_grad(o["dx"], o["df"], vectors["dpost"], vectors["dpre"], far["dh"], far["dn"], o["h"], far["f"], s["post"], s["pre"], gate=far["gate"], dgate=o["dgate"])
    for k, (want, size) in norm_reference(s, 0.75, stored=o["h"]).items():
        got = vectors[k] if k in vectors else o[k]
        n = dim + (tokens if k in ("dpost", "dpre") or (k == "dgate" and gate == "channel") else 0)
        rounding = unit(wkind if k in vectors else kind)
        within(got, want, norm_share(n) * size + 1.01 * rounding * want.abs() + tiny(wkind if k in vectors else kind), k)
    assert all(bool((w[:, dim:] == 7.0).all()) for w in wide.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 2000, 2001, 17000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("h_power,dn_power", [(50, 90), (-40, -100), (-45, -115)])
def test_norm_gradients_whose_products_leave_32_bits(pkg, dim, kind, h_power, dn_power):
    """The sum of dn pre h, where the sums of squares stay in range; among rows whose dn is zero."""
    gen = new_gen(dim)
    tokens, eps = 12, 1e-30
    s = norm_inputs(gen, tokens, dim, kind, kind, "none")
    s["x"], s["f"] = (randn(gen, tokens, dim).double() * 2.0 ** h_power).to(TYPES[kind]), randn(gen, tokens, dim).to(TYPES[kind])
    s["post"] = (s["post"].double() * 2.0 ** h_power).to(TYPES[kind])
    s["dn"], s["dh"] = ((s[k].double() * 2.0 ** dn_power).to(TYPES[kind]) for k in ("dn", "dh"))
    s["dn"][3::4] = 0
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=code(pkg, kind), eps=eps)
    o = {k: torch.empty(tokens, dim, device="cuda", dtype=TYPES[kind]) for k in ("h", "n", "dx", "dpre")}
    o["dpre"] = torch.empty(dim, device="cuda", dtype=TYPES[kind])
    plan.execute(o["h"], o["n"], s["x"], s["f"], s["post"], s["pre"])
    plan.execute_grad(o["dx"], None, None, o["dpre"], s["dh"], s["dn"], o["h"], s["f"], s["post"], s["pre"])
    ref = norm_reference(s, 1.0, stored=o["h"], eps=eps)
    for k in ("h", "n", "dx", "dpre"):
        want, size = ref[k]
        # 2^-126 and below: single precision's subnormal numbers
        within(o[k], want, norm_share(dim + tokens) * size + 1.01 * unit(kind) * want.abs() + 2.0 ** -140, k)


STACKED = [  # rows, cols, inner, result: more tiles than multiprocessors
    (5, 40000, 300, "bf16"), (16, 38000, 64, "f32"), (20, 39001, 513, "f16"), (64, 65536, 512, "bf16"), (100, 60007, 260, "f32"), (300, 30000, 256, "bf16"),
    (64, 512, 11008, "bf16"), (300, 700, 16383, "f32")]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,inner,kind", STACKED)
def test_micro_products_of_several_tiles_a_block(pkg, rows, cols, inner, kind):
    gen = new_gen(rows + cols + inner)
    qa, qb, a, b = product_case(pkg, gen, rows, cols, inner)
    plan = pkg.MicroProductPlan(rows, cols, inner, out_dtype=code(pkg, kind))
    out = torch.full((rows, cols + 1), 7.0, device="cuda").to(TYPES[kind])
    plan.execute(out[:, :cols], *qa, *qb)
    ref = a @ b.T
    within(out[:, :cols], ref, product_bound(a, b, inner, kind, ref), "product")
    assert bool((out[:, cols:] == 7.0).all()) and plan.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,outputs", [(1000, 520, 264), (33, 129, 70), (2050, 1024, 512)])
def test_gradients_by_micro_products(pkg, tokens, dim, outputs):
    """Both gradients of a projection, whose operands are quantised along the sums' index."""
    gen = new_gen(tokens)
    x, w, dy = (randn(gen, *s).bfloat16() for s in ((tokens, dim), (outputs, dim), (tokens, outputs)))
    by = lambda t, **kw: quantised(pkg, t, "bf16", **kw)[1:]  # noqa: E731
    for got, (a, b), (qa, qb) in ((torch.empty(outputs, dim, device="cuda"), (dy.T, x.T), (by(dy, transposed=True), by(x, transposed=True))),
                                  (torch.empty(tokens, dim, device="cuda"), (dy, w.T), (by(dy), by(w, transposed=True)))):
        inner = a.shape[1]
        pkg.MicroProductPlan(*got.shape, inner, out_dtype=pkg.F32).execute(got, *qa, *qb)
        a, b = rounded(a, E2M1), rounded(b, E2M1)
        within(got, a @ b.T, product_bound(a, b, inner, "f32", a @ b.T), "gradient")


# --------------------------------------------------------------------------- results over arguments (no GPU for refusals) ----
INVALID = 2


def test_norms_refuse_results_that_share_memory(pkg):
    """Addresses that no call gets as far as using."""
    lib, at = pkg.lib(), [1 << k for k in range(20, 34)]
    for dim in (40, 20000):
        row = 2 * dim
        token, channel = pkg.ResidualNormPlan(8, dim, gate="token"), pkg.ResidualNormPlan(8, dim, gate="channel")

        def forward(plan=token, h=at[0], n=at[1], x=at[2], f=at[3], post=at[4], pre=at[5], gate=at[6], ld=dim):
            return lib.tc_residual_norm_execute(plan._h, h, ld, n, ld, x, ld, f, ld, post, pre, gate, ld, 8, None)

        # shifted by a row or by one element, on either side; between rows as far as the row's own end
        shifts = [{"h": at[2] + row}, {"h": at[2] - row}, {"h": at[2] + 7 * row}, {"h": at[2] + 2}, {"n": at[3] + 2 * row}, {"n": at[0] + row}, {"n": at[6] - 7 * row},
                  {"h": at[4]}, {"n": at[5] + row - 2}, {"h": at[5] - 8 * row + 2}, {"ld": 2 * dim + 8, "h": at[2] + row - 2}, {"ld": 2 * dim + 8, "n": at[3] - row + 2}]
        assert [forward(**s) for s in shifts] == [INVALID] * len(shifts)
        assert forward(plan=channel, h=at[6] - row) == INVALID and forward(plan=channel, n=at[6]) == INVALID
        wide = lib.tc_residual_norm_execute(token._h, at[0], dim + 8, None, dim, at[0] + row, dim, at[3], dim, None, None, at[6], dim, 8, None)
        assert wide == INVALID  # rows of two pitches meet from the second on

        def backward(plan=channel, dx=at[0], df=at[1], dgate=at[2], dpost=at[3], dpre=at[4], dh=at[5], dn=at[6], h=at[7], f=at[8], post=at[9], pre=at[10], gate=at[11]):
            return lib.tc_residual_norm_execute_grad(plan._h, dx, dim, df, dim, dgate, dim, dpost, dpre, dh, dim, dn, dim, h, dim, f, dim, post, pre, gate, dim, 8, None, 0, None)

        shifts = [{"dpost": at[9]}, {"dpost": at[4]}, {"dpre": at[9]}, {"dpre": at[10] + 16}, {"dpre": at[11]}, {"dpost": at[2]}, {"dgate": at[11]}, {"dgate": at[9]},
                  {"dpost": at[0] + 3 * row}, {"dpre": at[7] + row}, {"dx": at[5] + row}, {"df": at[8] - 2 * row}, {"dx": at[1] + 2}, {"dgate": at[1] + 7 * row}]
        assert [backward(**s) for s in shifts] == [INVALID] * len(shifts)
        assert backward(plan=token, dgate=at[11] + row) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 41, 17000])
def test_norms_of_columns_of_one_matrix(pkg, dim):
    """Rows that lie between one another's share nothing: every argument of a call beside the others."""
    gen = new_gen(dim)
    tokens = 9
    s = norm_inputs(gen, tokens, dim, "bf16", "bf16", "token")
    plan = pkg.ResidualNormPlan(tokens, dim, gate="token")
    names = ["x", "f", "gate", "dh", "dn", "h", "n", "dx", "df", "dgate"]
    both = []
    for step in (0, dim):
        wide = torch.zeros(tokens, dim * len(names), device="cuda").bfloat16()
        t = {k: wide[:, i * dim:(i + 1) * dim] if step else torch.zeros(tokens, dim, device="cuda").bfloat16() for i, k in enumerate(names)}
        for k in names[:5]:
            t[k].copy_(s[k])
        dpost, dpre = (torch.empty(dim, device="cuda").bfloat16() for _ in range(2))
        plan.execute(t["h"], t["n"], t["x"], t["f"], s["post"], s["pre"], gate=t["gate"])
        plan.execute_grad(t["dx"], t["df"], dpost, dpre, t["dh"], t["dn"], t["h"], t["f"], s["post"], s["pre"], gate=t["gate"], dgate=t["dgate"])
        both.append((t, dpost, dpre))
    (a, *va), (b, *vb) = both
    for k, (want, size) in norm_reference(s, 1.0, stored=b["h"], eps=1e-6).items():
        got = vb[["dpost", "dpre"].index(k)] if k in ("dpost", "dpre") else b[k]
        within(got, want, norm_share(dim + tokens) * size + 1.01 * unit("bf16") * want.abs() + tiny("bf16"), k)
    assert all(torch.equal(a[k], s[k]) and torch.equal(b[k], s[k]) for k in names[:5])


def test_activations_refuse_results_that_share_memory(pkg):
    lib, at = pkg.lib(), [1 << k for k in range(20, 26)]
    for gated in (False, True):
        width = 80 if gated else 40
        p = pkg.CheckpointPlan(8, 40, activation="silu", gated=gated)
        call = lambda y=at[0], c=at[1], s=at[2], x=at[3]: lib.tc_checkpoint_execute(p._h, y, 40, c, s, x, width, 8, None)  # noqa: E731
        shifts = [{"y": at[3] + 80}, {"y": at[3] - 7 * 80}, {"c": at[3] + 32}, {"s": at[3] + 1}, {"s": at[1] + 64}, {"c": at[0]}, {"s": at[0] + 639}]
        assert [call(**s) for s in shifts] == [INVALID] * len(shifts)
        back = lambda y=at[0], c=at[1], s=at[2]: lib.tc_checkpoint_restore(p._h, y, 40, c, s, 8, None)  # noqa: E731
        assert back(y=at[1] + 2) == INVALID and back(s=at[0] + 5) == INVALID
        grad = lambda dx=at[0], dy=at[3], c=at[1], s=at[2]: lib.tc_checkpoint_execute_grad(p._h, dx, width, dy, 40, c, s, 8, None)  # noqa: E731
        assert grad(dx=at[3] + 80) == INVALID and grad(dy=at[0] - 80) == INVALID and grad(dx=at[1] + 16) == INVALID and grad(s=at[0] + 1) == INVALID
        product = lambda dw=at[0], dy=at[3], c=at[1], s=at[2]: lib.tc_checkpoint_execute_product(p._h, dw, 40, pkg.F32, dy, 5, c, s, 5, 8, 0, None, 0, None)  # noqa: E731
        assert product(dw=at[3] + 76) == INVALID and product(dy=at[0] + 798) == INVALID and product(c=at[0] + 784) == INVALID and product(s=at[0]) == INVALID


@pytest.mark.gpu
def test_activations_of_columns_of_one_matrix(pkg):
    gen = new_gen(3)
    tokens, dim = 21, 48
    plan = pkg.CheckpointPlan(tokens, dim, activation="silu", gated=True)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    wide = randn(gen, tokens, 6 * dim).bfloat16()
    given = wide.clone()
    x, y, dy, dx = (wide[:, a * dim:b * dim] for a, b in ((0, 2), (2, 3), (3, 4), (4, 6)))
    plan.execute(codes, scales, x, y=y)
    plan.execute_grad(dx, codes, scales, dy)
    want = torch.empty(tokens, dim, device="cuda").bfloat16(), torch.empty(tokens, 2 * dim, device="cuda").bfloat16()
    plan.execute(codes, scales, given[:, :2 * dim].contiguous(), y=want[0])
    plan.execute_grad(want[1], codes, scales, given[:, 3 * dim:4 * dim].contiguous())
    assert torch.equal(y, want[0]) and torch.equal(dx, want[1]) and torch.equal(x, given[:, :2 * dim]) and torch.equal(dy, given[:, 3 * dim:4 * dim])


def test_microscaled_numbers_refuse_results_that_share_memory(pkg):
    lib, at = pkg.lib(), [1 << k for k in range(20, 26)]
    m, q = pkg.MicroscalePlan(8, 40), pkg.MicroProductPlan(8, 16, 40)
    call = lambda c=at[0], s=at[1], x=at[2], t=0: lib.tc_microscale_execute(m._h, c, 32, s, x, 8 if t else 40, t, 8, None)  # noqa: E731
    for t in (0, 1):
        shifts = [{"c": at[2] + 80}, {"c": at[2] - 240}, {"s": at[2] + 16}, {"s": at[0] + 240}, {"x": at[0] + 254}, {"x": at[1] + 510}]
        assert [call(t=t, **s) for s in shifts] == [INVALID] * len(shifts)
    back = lambda x=at[2], c=at[0], s=at[1]: lib.tc_microscale_restore(m._h, x, 40, c, 32, s, 8, None)  # noqa: E731
    assert back(x=at[0] + 16) == INVALID and back(s=at[2] + 624) == INVALID
    product = lambda o=at[0], a=at[1], sa=at[2], b=at[3], sb=at[4]: lib.tc_micro_product_execute(q._h, o, 16, a, 32, sa, b, 32, sb, 8, 0, None, 0, None)  # noqa: E731
    assert [product(o=at[k] + 16) for k in (1, 2, 3, 4)] == [INVALID] * 4
    assert [product(**{k: at[0] + 240}) for k in ("a", "sa", "b", "sb")] == [INVALID] * 4


@pytest.mark.gpu
def test_microscaled_numbers_beside_each_other(pkg):
    """Codes in the gaps of a matrix's rows, a product's result behind its operands' columns."""
    gen = new_gen(4)
    rows, cols = 40, 64
    memory = torch.zeros(rows, 512, device="cuda", dtype=torch.uint8)
    x = memory[:, :128].view(torch.bfloat16)
    x.copy_(randn(gen, rows, cols))
    plan = pkg.MicroscalePlan(rows, cols)
    codes, scales = memory[:, 128:160], torch.zeros(plan.scales_shape, device="cuda", dtype=torch.uint8)
    plan.execute(codes, scales, x)
    back, out = memory[:, 160:288].view(torch.bfloat16), memory[:, 288:448].view(torch.float32)
    plan.restore(back, codes, scales)
    ref = rounded(x, E2M1)
    assert torch.equal(back.double(), ref)
    pkg.MicroProductPlan(rows, rows, cols, out_dtype=pkg.F32).execute(out, codes, scales, codes, scales)
    within(out, ref @ ref.T, product_bound(ref, ref, cols, "f32", ref @ ref.T), "product")
    assert torch.equal(rounded(x, E2M1), ref)


# ------------------------------------------------------------------------------------------------ calls by ctypes ----
WITHOUT = """
import sys
class Missing:
    def find_spec(self, name, path=None, target=None):
        if name.endswith("._tc_calls"):
            raise ImportError(name)
sys.meta_path.insert(0, Missing())
sys.path.insert(0, {root!r})
import __graft_entry__
pkg = __graft_entry__.load_package()
assert pkg.parse("C [a,2,b,3] += sum(c,4) * A [a,c] * B [c,b];") and pkg.Plan("C [a,2,b,3] += sum(c,4) * A [a,c] * B [c,b];").cost()
assert type(pkg._calls).__name__ == "_CtypesCalls"
import torch
for call in (lambda: pkg.MicroscalePlan(4, 32).execute(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), torch.zeros(4, 32)),
             lambda: pkg.ResidualNormPlan(4, 4).execute(None, None, None, None)):
    try:
        call()
    except TypeError:
        continue
    raise SystemExit("not refused")
"""


def test_the_package_works_without_its_extension(pkg):
    """Neither contractions nor the plans need the calls past ctypes."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", WITHOUT.format(root=root)], capture_output=True, text=True, cwd=root)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_a_block_by_ctypes(pkg, monkeypatch):
    inputs = block_inputs(70, 96)
    block = Block(pkg, 70, 96, 64)
    want = {k: v.clone() for k, v in block.run(*inputs).items()}
    for v in block.o.values():
        v.fill_(5.0)
    by_ctypes = pkg._CtypesCalls(pkg.lib())
    assert type(pkg._calls) is not type(by_ctypes)  # both are there to be compared
    monkeypatch.setattr(pkg, "_calls", by_ctypes)
    got = block.run(*inputs)
    assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("tokens,dim,activation,gated,most", [(1, 4096, "silu", False, 1 << 18), (32, 4096, "none", False, 5 << 20), (300, 1024, "none", True, 35 << 20),
                                                              (8192, 4096, "none", False, 121 << 20), (8192, 4096, "silu", True, 188 << 20)])
def test_a_weight_gradients_workspace(pkg, tokens, dim, activation, gated, most):
    """As the header states it: two bytes an element and term, columns of dy, slices where there may be some."""
    size = pkg.CheckpointPlan(tokens, dim, activation=activation, gated=gated).describe()["workspace_bytes"]
    terms = 1 if activation == "none" and not gated else 2
    assert 2 * tokens * dim * terms <= size <= most
    assert pkg.CheckpointPlan(tokens, dim, activation=activation, gated=gated, products=False).describe()["workspace_bytes"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7])
def test_a_weight_gradient_of_more_columns_than_a_panel(pkg, tokens):
    gen = new_gen(tokens)
    dim, outputs = 40, 70001
    x, dy = randn(gen, tokens, dim).bfloat16(), randn(gen, tokens, outputs).bfloat16()
    plan = pkg.CheckpointPlan(tokens, dim, activation="gelu")
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    plan.execute(codes, scales, x)
    dw = torch.empty(outputs, dim, device="cuda")
    plan.execute_product(dw, dy, codes, scales)
    f = function("gelu", False, kept(x, False))
    ref, size = dy.double().T @ f, dy.double().abs().T @ f.abs()
    within(dw, ref, (2 * (tokens + 1) * 2.0 ** -23 + 1.01 * unit("bf16") ** 2 + FINE["gelu"]) * size + tiny("bf16"), "weight")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,outputs,name,gated", [(1, 7, 5, "silu", False), (300, 96, 131, "gelu", True), (2000, 512, 256, "silu", False)])
def test_a_weight_gradient_in_single_precision(pkg, tokens, dim, outputs, name, gated):
    """By a contraction of what is restored, since execute_product has 16-bit operands."""
    gen = new_gen(tokens)
    x, dy = randn(gen, tokens, dim * (2 if gated else 1)), randn(gen, tokens, outputs)
    plan = pkg.CheckpointPlan(tokens, dim, dtype=pkg.F32, activation=name, gated=gated)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    plan.execute(codes, scales, x)
    f, dw = torch.empty(tokens, dim, device="cuda"), torch.empty(outputs, dim, device="cuda")
    plan.restore(f, codes, scales)
    pkg.Plan("C [i,%d,o,%d] = sum(t,%d) * A [i,t] * B [o,t];" % (dim, outputs, tokens), dtype=pkg.F32).execute(dw, f, dy)
    v = function(name, gated, kept(x, gated))
    # three products of eleven bits each: what they leave is 2^-21 of a term, their sums are in fp32
    within(dw, dy.double().T @ v, (3 * tokens * 2.0 ** -23 + 2.0 ** -20 + FINE[name]) * (dy.double().abs().T @ v.abs()), "weight")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_weight_gradients_numbers_far_out(pkg, kind):
    """The function's values beyond fp16's range come from both of their terms; what is not finite keeps to its rows and columns."""
    tokens, dim, outputs = 5, 96, 40
    gen = new_gen(9)
    x = (randn(gen, tokens, 2 * dim) * 0.5).to(TYPES[kind])
    for col, (a, b) in enumerate(((256.0, 256.0), (320.0, -320.0), (448.0, 280.0))):
        x[:, 32 * col], x[:, dim + 32 * col] = a, b  # 65536, -102400 and, since 280 is kept as 288, 129024
    dy = (1 + torch.rand(tokens, outputs, device="cuda", generator=gen)).to(TYPES[kind])
    plan = pkg.CheckpointPlan(tokens, dim, dtype=code(pkg, kind), activation="silu", gated=True)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    dw = torch.empty(outputs, dim, device="cuda")

    def run():
        plan.execute(codes, scales, x)
        plan.execute_product(dw, dy, codes, scales)
        return dw

    f = function("silu", True, kept(x, True))
    assert [float(f[0, c].round()) for c in (0, 32, 64)] == [65536.0, -102400.0, 129024.0]
    ref, size = dy.double().T @ f, dy.double().abs().T @ f.abs()
    bound = (2 * (tokens + 16) * 2.0 ** -23 + 1.01 * unit(kind) ** 2 + FINE["silu"] + 2.0 ** -24) * size + tokens * 2 * tiny(kind)
    within(run(), ref, bound, "weight")
    x[1, 0], x[1, dim] = 448.0, 448.0  # 200704: in fp16 beyond both terms
    run()
    assert bool(torch.isfinite(dw[:, 1:]).all()) and bool(torch.isfinite(dw[:, 0]).all()) == (kind == "bf16")
    x[1, 0], x[1, dim] = 256.0, 256.0
    dy[2, 7] = float("inf")
    run()
    others = torch.arange(outputs, device="cuda") != 7
    within(dw[others], ref[others], bound[others], "other rows")
    assert not bool(torch.isfinite(dw[7]).any())
    dy[2, 7] = 1.0
    x[3, 40] = float("nan")  # of columns 32 to 63
    run()
    assert bool(torch.isnan(dw[:, 32:64]).all()) and bool(torch.isfinite(dw[:, :32]).all()) and bool(torch.isfinite(dw[:, 64:]).all())
