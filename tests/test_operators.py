"""The operators around contractions: embedding, vocabulary loss, orthogonalised updates, against plain 64-bit implementations.

Tolerances come from the number formats: `unit(type)` is half of the last place of one.  An fp32 sum of n terms, in an order
and a rounding of the hardware's choice, is taken to be off by at most n * 2^-23 of the terms' sizes."""
import ctypes

import pytest
import torch

INVALID, UNSUPPORTED, EXTENT, ALIGNMENT, STATE, WORKSPACE = 2, 3, 4, 6, 7, 8
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def code(pkg, name):
    return {"bf16": pkg.BF16, "f16": pkg.F16, "f32": pkg.F32}[name]


def unit(name):
    return {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}[name]


def tiny(name):
    """Half of the smallest subnormal."""
    return {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}[name]


def randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def new_gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), what
    off = (got - ref).abs() - tol
    assert off.numel() == 0 or bool((off <= 0).all()), "%s: %.3e over its bound" % (what, off.max().item())


# ------------------------------------------------------------------------------------------------ refusals (no GPU) ----
def create(pkg, name, *args):
    h = ctypes.c_void_p()
    st = getattr(pkg.lib(), "tc_op_create_" + name)(*args, ctypes.byref(h))
    if st == 0:
        pkg.lib().tc_op_destroy(h)
    return st


def test_plans_refuse_what_they_cannot_do(pkg):
    coef = (ctypes.c_double * 6)(1, 2, 3, 4, 5, 6)
    assert create(pkg, "embedding", 8, 16, 4, pkg.F32, 1.0) == 0
    assert create(pkg, "embedding", 8, 16, 4, pkg.F64, 1.0) == INVALID
    assert create(pkg, "embedding", 8, 16, 4, pkg.F32, float("nan")) == INVALID
    assert create(pkg, "embedding", 0, 16, 4, pkg.F32, 1.0) == EXTENT
    assert create(pkg, "embedding", 8, 1 << 31, 4, pkg.F32, 1.0) == UNSUPPORTED
    assert create(pkg, "vocab_loss", 8, 4, 16, pkg.BF16) == 0
    assert create(pkg, "vocab_loss", 8, 4, 16, pkg.F32) == UNSUPPORTED
    assert create(pkg, "vocab_loss", 8, 4, 16, 9) == INVALID
    assert create(pkg, "vocab_loss", 8, 0, 16, pkg.BF16) == EXTENT
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.BF16, 2, coef, 1e-7) == 0
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.F32, 2, coef, 1e-7) == INVALID
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.BF16, 0, coef, 1e-7) == UNSUPPORTED
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.BF16, 2, None, 1e-7) == INVALID
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.BF16, 2, coef, -1.0) == INVALID
    assert create(pkg, "orthogonal", 0, 4, 4, pkg.F32, pkg.BF16, 2, coef, 0.0) == EXTENT
    coef[1] = float("inf")
    assert create(pkg, "orthogonal", 1, 4, 4, pkg.F32, pkg.BF16, 2, coef, 0.0) == INVALID
    lib = pkg.lib()
    assert lib.tc_op_create_embedding(8, 16, 4, pkg.F32, 1.0, None) == INVALID
    assert lib.tc_op_commit(None) == INVALID and lib.tc_op_status(None, None) == INVALID
    lib.tc_op_destroy(None)


def test_python_plans_check_their_arguments(pkg):
    with pytest.raises(pkg.TcError):
        pkg.EmbeddingPlan(0, 4, 4)
    with pytest.raises(pkg.TcError):
        pkg.VocabLossPlan(4, 4, 4, dtype=pkg.F64)
    with pytest.raises(ValueError):
        pkg.OrthogonalPlan(4, 4, steps=3, coefficients=[(1, 2, 3)] * 2)
    with pytest.raises(TypeError):
        pkg.EmbeddingPlan(4, 4, 4).execute(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        pkg.OrthogonalPlan(4, 4).execute(torch.zeros(4, 4), torch.zeros(4, 4))
    assert pkg.VocabLossPlan(8192, 2048, 131072).describe()["pieces"] > 1
    assert pkg.OrthogonalPlan(64, 128, batch=3).describe()["operator"] == "orthogonal"
    assert pkg.EmbeddingPlan(64, 128, 32).describe()["vocab"] == 128


def test_calls_refuse_bad_pointers_and_sizes_before_they_touch_a_device(pkg):
    lib = pkg.lib()
    p, q, r = pkg.EmbeddingPlan(8, 16, 4, dtype=pkg.F32), pkg.VocabLossPlan(8, 4, 16), pkg.OrthogonalPlan(4, 6)
    a = 1 << 20  # an address that no call gets as far as using
    assert lib.tc_embedding_execute(q._h, a, 4, a, 4, a, pkg.I64, 8, None) == INVALID
    assert lib.tc_embedding_execute(p._h, None, 4, a, 4, a, pkg.I64, 8, None) == INVALID
    assert lib.tc_embedding_execute(p._h, a, 4, a, 4, a, pkg.F32, 8, None) == INVALID
    assert lib.tc_embedding_execute(p._h, a, 3, a, 4, a, pkg.I64, 8, None) == EXTENT
    assert lib.tc_embedding_execute(p._h, a, 4, a, 4, a, pkg.I64, 9, None) == EXTENT
    assert lib.tc_embedding_execute(p._h, a + 2, 4, a, 4, a, pkg.I64, 8, None) == ALIGNMENT
    assert lib.tc_embedding_execute_grad(p._h, a, 4, a, -1, a, pkg.I64, 8, 0, None, 0, None) == EXTENT
    assert lib.tc_vocab_loss_execute(p._h, a, a, a, 4, a, 4, a, pkg.I64, 8, None, 0, None) == INVALID
    assert lib.tc_vocab_loss_execute(q._h, a, None, a, 4, a, 4, a, pkg.I64, 8, None, 0, None) == INVALID
    assert lib.tc_vocab_loss_execute(q._h, a, a, a + 1, 4, a, 4, a, pkg.I64, 8, None, 0, None) == ALIGNMENT
    assert lib.tc_vocab_loss_execute(q._h, a, a, a, 4, a, 4, a, pkg.I64, 9, None, 0, None) == EXTENT
    assert lib.tc_vocab_loss_execute_grad(q._h, None, 4, None, 4, a, 4, a, 4, a, pkg.I64, a, a, 8, None, 0, None) == INVALID
    assert lib.tc_vocab_loss_execute_grad(q._h, a, 3, None, 4, a, 4, a, 4, a, pkg.I64, a, a, 8, None, 0, None) == EXTENT
    s = lambda *v: (ctypes.c_int64 * 3)(*v)  # noqa: E731
    assert lib.tc_orthogonal_execute(r._h, None, s(24, 6, 1), a, s(24, 6, 1), None, 0, None) == INVALID
    assert lib.tc_orthogonal_execute(r._h, a, s(24, 5, 1), a, s(24, 6, 1), None, 0, None) == EXTENT
    assert lib.tc_orthogonal_execute(r._h, a, s(24, 6, 1), a, s(24, 6, -1), None, 0, None) == EXTENT
    assert lib.tc_orthogonal_execute(r._h, a + 1, s(24, 6, 1), a, s(24, 6, 1), None, 0, None) == ALIGNMENT
    assert lib.tc_op_workspace_bytes(p._h, None) == INVALID and lib.tc_op_status(p._h, ctypes.byref(ctypes.c_int())) == STATE
    assert lib.tc_op_commit_in(p._h, None, 1 << 20) == INVALID
    assert lib.tc_op_set_test_fault(p._h, 1) == INVALID


# ---------------------------------------------------------------------------------------------------- embedding ----
LOOKUPS = [  # tokens, vocab, dim, type, extra elements per row, token type, scale
    (1, 1, 1, "f32", 0, torch.int64, 1.0), (7, 5, 8, "bf16", 0, torch.int32, 1.5), (33, 100, 129, "f16", 3, torch.int64, 0.25),
    (300, 1000, 64, "bf16", 8, torch.int64, 8.0), (1025, 50, 301, "f32", 1, torch.int64, 1.0), (64, 40, 2048, "bf16", 0, torch.int64, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,dim,kind,extra,index,scale", LOOKUPS)
def test_lookup(pkg, tokens, vocab, dim, kind, extra, index, scale):
    gen = new_gen(tokens)
    table = randn(gen, vocab, dim + extra).to(TYPES[kind])[:, :dim]
    ids = torch.randint(-2, vocab + 2, (tokens,), device="cuda", generator=gen).to(index)
    out = torch.full((tokens, dim + extra), 7.0, device="cuda").to(TYPES[kind])
    pkg.EmbeddingPlan(tokens, vocab, dim, dtype=code(pkg, kind), scale=scale).execute(out[:, :dim], table, ids)
    there = (ids >= 0) & (ids < vocab)
    ref = torch.where(there[:, None], table.double()[ids.clamp(0, vocab - 1).long()] * scale, 0.0)
    within(out[:, :dim], ref, 1.01 * unit(kind) * ref.abs(), "rows")
    assert bool((out[:, dim:] == 7.0).all())


def table_grad_reference(grad, ids, vocab, scale):
    keep = (ids >= 0) & (ids < vocab)
    ref = torch.zeros(vocab, grad.shape[1], dtype=torch.float64, device="cuda")
    size, n = torch.zeros_like(ref), torch.zeros(vocab, dtype=torch.float64, device="cuda")
    at = ids[keep].long()
    ref.index_add_(0, at, grad[keep].double() * scale)
    size.index_add_(0, at, grad[keep].double().abs() * abs(scale))
    n.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return ref, (n[:, None] + 2) * 2.0 ** -23 * size


GRADS = [  # tokens, vocab, dim, type, extra, how tokens are spread, accumulate
    (1, 1, 1, "f32", 0, "same", False), (5, 600, 8, "bf16", 0, "any", False), (31, 3, 129, "f16", 3, "any", False),
    (32, 7, 64, "bf16", 0, "same", False), (33, 7, 64, "bf16", 8, "same", True), (64, 1, 9, "f32", 0, "same", True),
    (2000, 511, 40, "bf16", 0, "few", False), (2000, 512, 301, "f32", 0, "few", False), (16384, 300000, 72, "f16", 0, "few", False),
    (16385, 1000, 33, "f32", 2, "few", False), (40000, 262144, 16, "bf16", 0, "few", True), (300000, 700, 8, "f32", 0, "few", False),
    (100, 50, 1100, "bf16", 0, "none", False)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,dim,kind,extra,spread,accumulate", GRADS)
def test_table_gradient(pkg, tokens, vocab, dim, kind, extra, spread, accumulate):
    gen = new_gen(tokens + dim)
    grad = randn(gen, tokens, dim + extra).to(TYPES[kind])[:, :dim]
    if spread == "same":
        ids = torch.full((tokens,), vocab - 1, device="cuda")
    elif spread == "none":
        ids = torch.full((tokens,), -1, device="cuda")
    elif spread == "any":
        ids = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    else:  # some numbers very often, some never, some outside
        ids = (torch.rand(tokens, device="cuda", generator=gen) ** 8 * (vocab + 2)).long() - 1
    table = randn(gen, vocab, dim + extra).to(TYPES[kind])
    old = table.clone()
    plan = pkg.EmbeddingPlan(tokens, vocab, dim, dtype=code(pkg, kind), scale=0.5)
    plan.execute_grad(table[:, :dim], grad, ids, accumulate=accumulate)
    ref, tol = table_grad_reference(grad, ids, vocab, 0.5)
    if accumulate:
        ref = ref + old[:, :dim].double()
        tol = tol + 2.0 ** -23 * old[:, :dim].double().abs()
    within(table[:, :dim], ref, tol + unit(kind) * (ref.abs() + tol) + tiny(kind), "table")
    assert torch.equal(table[:, dim:], old[:, dim:])
    again = old.clone()
    plan.execute_grad(again[:, :dim], grad, ids, accumulate=accumulate)
    assert torch.equal(again, table)  # the same bits


@pytest.mark.gpu
def test_rows_without_a_token_keep_infinities_out(pkg):
    ids = torch.tensor([2, -1, 2, 9], device="cuda")
    grad = torch.ones(4, 16, device="cuda")
    grad[1], grad[3] = float("nan"), float("inf")
    table = torch.full((4, 16), float("nan"), device="cuda")
    plan = pkg.EmbeddingPlan(8, 4, 16, dtype=pkg.F32)
    plan.execute_grad(table, grad, ids)
    ref = torch.zeros(4, 16, device="cuda")
    ref[2] = 2.0
    assert torch.equal(table, ref)
    plan.execute_grad(table, grad[:0], ids[:0])
    assert torch.equal(table, torch.zeros_like(ref))


@pytest.mark.gpu
def test_table_gradient_of_a_broadcast_row_and_against_differences(pkg):
    gen = new_gen(3)
    tokens, vocab, dim = 500, 70, 24
    ids = torch.randint(-1, vocab, (tokens,), device="cuda", generator=gen)
    row = randn(gen, 1, dim)
    plan = pkg.EmbeddingPlan(tokens, vocab, dim, dtype=pkg.F32, scale=2.0)
    got = torch.empty(vocab, dim, device="cuda")
    plan.execute_grad(got, row.expand(tokens, dim), ids)
    ref, tol = table_grad_reference(row.expand(tokens, dim), ids, vocab, 2.0)
    within(got, ref, tol + unit("f32") * ref.abs(), "broadcast")
    # the lookup is linear: the difference that a step makes is the gradient times the step
    table = torch.randint(-64, 64, (vocab, dim), device="cuda", generator=gen).float() / 64
    step = torch.randint(-64, 64, (vocab, dim), device="cuda", generator=gen).float() / 64
    out = [torch.empty(tokens, dim, device="cuda") for _ in range(2)]
    plan.execute(out[0], table, ids)
    plan.execute(out[1], table + step, ids)
    made = ((out[1] - out[0]).double() * row.double()).sum().item()
    assert abs(made - (got.double() * step.double()).sum().item()) <= 1e-5 * ref.abs().sum().item()


# ----------------------------------------------------------------------------------------------- vocabulary loss ----
def loss_reference(hidden, weight, targets, grad, kind):
    """Values and elementwise bounds in 64 bits."""
    (t, d), v, u = hidden.shape, weight.shape[0], unit(kind)
    part = (targets >= 0) & (targets < v)
    h = torch.where(part[:, None], hidden.double(), 0.0)
    w = weight.double()
    z = h @ w.T
    z_off = d * 2.0 ** -23 * (h.abs() @ w.abs().T)
    lse = torch.logsumexp(z, 1)
    at = targets.clamp(0, v - 1).long()[:, None]
    hit = z.gather(1, at)[:, 0]
    # logits, exponents rounded at the size of the largest logit, exponentials and sums of v terms in 32 bits
    e = z_off.amax(1) + 2.0 ** -20 * (1 + z.abs().amax(1)) + v * 2.0 ** -23 / 64
    zero = torch.zeros_like(lse)
    out = {"loss": torch.where(part, lse - hit, zero), "lse": torch.where(part, lse, zero)}
    tol = {"loss": 2 * e + 2.0 ** -22 * lse.abs(), "lse": e + 2.0 ** -22 * lse.abs()}
    g = torch.where(part, grad.double(), zero)
    p = (z - lse[:, None]).exp()
    onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
    G = g[:, None] * (p - onehot)
    G_off = u * G.abs() + (2 * e[:, None] + 2.0 ** -22) * g.abs()[:, None] * (p + onehot)
    if kind == "f16":
        G_off = G_off + g.abs().max() * 2.0 ** -38  # subnormals, with the largest weight at 2^14
    for name, x, y, xo, n in (("dhidden", G, w, G_off, v), ("dweight", G.T, h, G_off.T, t)):
        out[name] = x @ y
        raw = (xo + n * 2.0 ** -23 * (x.abs() + xo)) @ y.abs()
        tol[name] = raw + u * (out[name].abs() + raw) + tiny(kind)
    return out, tol


def loss_run(pkg, hidden, weight, targets, grad, kind, most=None, plan=None, want=("dhidden", "dweight"), stream=None, workspace=None):
    t, d = hidden.shape
    plan = plan or pkg.VocabLossPlan(most or max(t, 1), d, weight.shape[0], dtype=code(pkg, kind))
    nan = float("nan")
    new = lambda *s, dtype=TYPES[kind]: torch.full(s, nan, device="cuda", dtype=dtype)  # noqa: E731
    wide = [new(n, -(-d // 8) * 8 + 8) for n in (t, weight.shape[0])]  # rows further apart than they need to be
    out = {"loss": new(t, dtype=torch.float32), "lse": new(t, dtype=torch.float32), "dhidden": wide[0][:, :d], "dweight": wide[1][:, :d]}
    kw = dict(stream=stream, workspace=workspace)
    plan.execute(out["loss"], out["lse"], hidden, weight, targets, **kw)
    if want:
        plan.execute_grad(*(out[k] if k in want else None for k in ("dhidden", "dweight")), hidden, weight, targets, out["lse"], grad, **kw)
    assert plan.status() == 0
    assert all(bool(torch.isnan(x[:, d:]).all()) for x in wide)
    return out


def loss_inputs(seed, tokens, dim, vocab, kind, ignored, extra=0):
    gen = new_gen(seed)
    hidden = (randn(gen, tokens, dim + extra) * 2).to(TYPES[kind])[:, :dim]
    weight = (randn(gen, vocab, dim + extra) / dim ** 0.5).to(TYPES[kind])[:, :dim]
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    targets[torch.rand(tokens, device="cuda", generator=gen) < ignored] = -100
    grad = torch.rand(tokens, device="cuda", generator=gen) * (16.0 if kind == "f16" else 1.0 / max(1, tokens))
    return hidden, weight, targets, grad


LOSSES = [  # tokens, dim, vocab, type, share without a target, extra elements per row
    (1, 64, 128, "bf16", 0.0, 0), (1, 1, 1, "f16", 0.0, 0), (2, 7, 3, "bf16", 0.0, 0), (63, 64, 65, "f16", 0.3, 0), (64, 130, 1000, "bf16", 0.0, 0),
    (65, 72, 257, "bf16", 0.5, 8), (100, 33, 999, "f16", 0.2, 0), (128, 256, 128, "bf16", 0.0, 0), (129, 200, 131, "f16", 0.0, 3),
    (300, 512, 2000, "bf16", 0.1, 0), (257, 1000, 4097, "f16", 0.4, 0), (2048, 128, 20000, "bf16", 0.0, 0), (1500, 777, 3001, "bf16", 0.3, 0),
    (9000, 64, 1111, "bf16", 0.2, 0), (50, 640, 33, "bf16", 1.0, 0), (40000, 40, 300, "bf16", 0.3, 0),
    # up to four tokens: passes over the table
    (3, 131, 1001, "f16", 0.0, 0), (4, 256, 5000, "bf16", 0.3, 8), (5, 64, 70, "bf16", 0.0, 3), (8, 2048, 600, "bf16", 0.2, 0), (8, 77, 33, "f16", 0.0, 0),
    (2, 1000, 9000, "f16", 0.0, 0), (4, 2500, 400, "bf16", 0.0, 0), (4, 40, 300, "bf16", 1.0, 0), (9, 40, 300, "bf16", 0.3, 0), (1, 9, 1, "bf16", 0.0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,vocab,kind,ignored,extra", LOSSES)
def test_vocab_loss(pkg, tokens, dim, vocab, kind, ignored, extra):
    args = loss_inputs(tokens + vocab, tokens, dim, vocab, kind, ignored, extra)
    got = loss_run(pkg, *args, kind)
    ref, tol = loss_reference(*args, kind)
    for name in got:
        within(got[name], ref[name], tol[name], name)
    again = loss_run(pkg, *args, kind)
    assert all(torch.equal(got[k], again[k]) for k in got)  # the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,vocab,kind,extra", [(3, 1920, 11597, "f16", 0), (4, 256, 5000, "bf16", 8), (4, 2048, 3001, "f16", 0), (3, 101, 777, "bf16", 0)])
def test_few_tokens_gradients_are_rounded_once(pkg, tokens, dim, vocab, kind, extra):
    hidden, weight, targets, grad = loss_inputs(tokens + dim, tokens, dim, vocab, kind, 0.0, extra)
    got = loss_run(pkg, hidden, weight, targets, grad, kind)
    h, w, g = hidden.double(), weight.double(), grad.double()[:, None]
    z = h @ w.T
    p = torch.softmax(z, 1)
    onehot = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
    G = g * (p - onehot)
    # logits and exponents in 32 bits, as in loss_reference; nothing for a rounding of G
    e = (dim * 2.0 ** -23 * (h.abs() @ w.abs().T)).amax(1) + 2.0 ** -20 * (1 + z.abs().amax(1)) + vocab * 2.0 ** -23 / 64
    off = (2 * e[:, None] + 2.0 ** -22) * g * (p + onehot)
    for name, x, xo, y, n in (("dhidden", G, off, w, vocab), ("dweight", G.T, off.T, h, tokens)):
        want = x @ y
        raw = (xo + n * 2.0 ** -23 * (x.abs() + xo)) @ y.abs()
        within(got[name], want, raw + unit(kind) * (want.abs() + raw) + tiny(kind), name)


@pytest.mark.gpu
def test_vocab_loss_over_several_pieces(pkg):
    """A plan for many tokens takes the vocabulary in small pieces, whatever a call brings."""
    args = loss_inputs(5, 700, 96, 9001, "bf16", 0.1)
    plan = pkg.VocabLossPlan(65536, 96, 9001, dtype=pkg.BF16)
    assert plan.describe()["pieces"] >= 4
    got = loss_run(pkg, *args, "bf16", plan=plan)
    ref, tol = loss_reference(*args, "bf16")
    for name in got:
        within(got[name], ref[name], tol[name], name)
    odd = loss_inputs(6, 300, 95, 9001, "bf16", 0.1)  # and the table in pieces that have to be laid out
    plan = pkg.VocabLossPlan(65536, 95, 9001, dtype=pkg.BF16)
    got = loss_run(pkg, *odd, "bf16", plan=plan)
    ref, tol = loss_reference(*odd, "bf16")
    for name in got:
        within(got[name], ref[name], tol[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [4, 200])
def test_masked_rows_keep_infinities_and_nan_out(pkg, tokens):
    hidden, weight, targets, grad = loss_inputs(8, tokens, 128, 300, "bf16", 0.4)
    targets[1] = -1
    masked = targets < 0
    assert bool(masked.any())
    clean = loss_run(pkg, hidden, weight, targets, grad, "bf16")
    bad = hidden.clone()
    bad[masked] = torch.tensor([float("nan"), float("inf")], device="cuda").to(hidden.dtype).repeat(64)
    weights = torch.where(masked, float("nan"), grad)
    got = loss_run(pkg, bad, weight, targets, weights, "bf16")
    assert all(torch.equal(got[k], clean[k]) for k in got)
    over = torch.where(masked, 300, targets)  # at and above the vocabulary is no target either
    got = loss_run(pkg, bad, weight, over.int(), weights, "bf16")
    assert all(torch.equal(got[k], clean[k]) for k in got)


@pytest.mark.gpu
def test_large_and_infinite_logits(pkg):
    hidden, weight, targets, grad = loss_inputs(9, 80, 64, 500, "bf16", 0.0)
    args = (hidden * 64, weight * 16, targets, grad)  # logits of some thousands: one term carries the sum
    got = loss_run(pkg, *args, "bf16")
    ref, tol = loss_reference(*args, "bf16")
    for name in got:
        within(got[name], ref[name], tol[name], name)
    low = weight.clone()
    low[7:490] = 0
    low[7:490, 0] = float("-inf")  # most logits -inf: no share, and not NaN
    one = hidden.clone()
    one[:, 0] = 1.0
    plan = pkg.VocabLossPlan(80, 64, 500)
    loss, lse = (torch.empty(80, device="cuda") for _ in range(2))
    plan.execute(loss, lse, one, low, torch.zeros_like(targets))
    kept = torch.cat((low[:7], low[490:])).double()
    z = one.double() @ kept.T
    ref = torch.logsumexp(z, 1)
    off = 64 * 2.0 ** -23 * (one.double().abs() @ kept.abs().T).amax(1) + 2.0 ** -20 * (1 + z.abs().amax(1)) + 2.0 ** -22 * ref.abs()
    within(lse, ref, off, "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [4, 150])
def test_one_gradient_at_a_time_and_frozen_sides(pkg, tokens):
    args = loss_inputs(10, tokens, 96, 1000, "bf16", 0.1)
    both = loss_run(pkg, *args, "bf16")
    for name in ("dhidden", "dweight"):
        one = loss_run(pkg, *args, "bf16", want=(name,))
        assert torch.equal(one[name], both[name])
        assert bool(torch.isnan(one["dhidden" if name == "dweight" else "dweight"]).all())


@pytest.mark.gpu
def test_no_tokens(pkg):
    hidden, weight, targets, grad = loss_inputs(11, 4, 64, 100, "bf16", 0.0)
    got = loss_run(pkg, hidden[:0], weight, targets[:0], grad[:0], "bf16", most=4)
    assert bool((got["dweight"] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [4, 40])
def test_gradient_against_differences(pkg, t):
    gen = new_gen(12)
    d, v = 64, 300
    grid = lambda *s: torch.randint(-16, 17, s, device="cuda", generator=gen).to(torch.bfloat16) / 16  # noqa: E731
    hidden, weight = grid(t, d), grid(v, d) / 2
    targets = torch.randint(0, v, (t,), device="cuda", generator=gen)
    grad = torch.ones(t, device="cuda")
    base = loss_run(pkg, hidden, weight, targets, grad, "bf16")
    for name, x, step in (("dhidden", hidden, 2.0 ** -6), ("dweight", weight, 2.0 ** -7)):
        sign = (torch.randint(0, 2, x.shape, device="cuda", generator=gen) * 2 - 1).to(x.dtype) * step  # x +- step are exact
        total = []
        for s in (sign, -sign):
            a = (hidden + s, weight) if name == "dhidden" else (hidden, weight + s)
            total.append(loss_run(pkg, *a, targets, grad, "bf16", want=())["loss"].double().sum().item())
        made = (total[0] - total[1]) / 2
        said = (base[name].double() * sign.double()).sum().item()
        # the gradients' own roundings (two, each 2^-8 of the terms at most), and the third order: the logits' changes are
        # sums of d signs of size step * |other operand| (<= step * sqrt(d) in the mean), their cube times the softmax's third cumulant
        size = (base[name].double().abs() * step).norm().item()
        third = t * (step * d ** 0.5) ** 3
        assert abs(made - said) <= 2 * 2.0 ** -8 * size + third + 1e-4, (name, made, said)


@pytest.mark.gpu
def test_streams_workspaces_and_alignment(pkg):
    args = loss_inputs(13, 260, 128, 3000, "bf16", 0.1)
    plan = pkg.VocabLossPlan(260, 128, 3000).commit()
    ref = loss_run(pkg, *args, "bf16", plan=plan)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:  # one plan, three streams: calls share the plan's workspace one after the other
        with torch.cuda.stream(s):
            loss, lse = (torch.empty(260, device="cuda") for _ in range(2))
            dh, dw = torch.empty_like(args[0]), torch.empty_like(args[1])
            plan.execute(loss, lse, *args[:3])
            plan.execute_grad(dh, dw, *args[:3], lse, args[3])
            outs.append((loss, lse, dh, dw))  # and rows next to each other
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, ref[k]) for a, k in zip(o, ("loss", "lse", "dhidden", "dweight")))
    ws = torch.empty(plan.workspace_bytes() + 1024, dtype=torch.uint8, device="cuda")
    at = -ws.data_ptr() % 1024
    own = loss_run(pkg, *args, "bf16", plan=plan, workspace=ws[at:at + plan.workspace_bytes()])
    assert all(torch.equal(own[k], ref[k]) for k in own)
    with pytest.raises(pkg.TcError) as e:
        loss_run(pkg, *args, "bf16", plan=plan, workspace=ws[at:at + 1024])
    assert e.value.status == WORKSPACE
    # rows off 16 bytes, on either side
    shift = lambda x: torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)[1:].view_as(x).copy_(x)  # noqa: E731
    got = loss_run(pkg, shift(args[0]), shift(args[1]), *args[2:], "bf16", plan=plan)
    assert all(torch.equal(got[k], ref[k]) for k in got)


@pytest.mark.gpu
def test_memory_of_a_plan(pkg):
    """The caller's memory, the library's own, memory that is too small or not aligned."""
    args = loss_inputs(17, 64, 64, 500, "bf16", 0.1)
    ref = loss_run(pkg, *args, "bf16")
    lib, size = pkg.lib(), ctypes.c_size_t()
    plan = pkg.VocabLossPlan(64, 64, 500)
    pkg._check(lib.tc_op_workspace_bytes(plan._h, ctypes.byref(size)), "tc_op_workspace_bytes")
    memory = torch.full((size.value + 2048,), 255, dtype=torch.uint8, device="cuda")
    at = memory.data_ptr() + -memory.data_ptr() % 1024
    assert lib.tc_op_commit_in(plan._h, at + 16, size.value) == WORKSPACE
    assert lib.tc_op_commit_in(plan._h, at, size.value - 1) == WORKSPACE
    assert lib.tc_op_commit_in(plan._h, at, size.value) == 0 and lib.tc_op_commit_in(plan._h, at, size.value) == STATE
    plan._device = 0  # committed behind the wrapper's back
    got = loss_run(pkg, *args, "bf16", plan=plan)
    assert all(torch.equal(got[k], ref[k]) for k in ref)
    plan.close()
    plan = pkg.VocabLossPlan(64, 64, 500)
    assert lib.tc_op_commit(plan._h) == 0 and plan.workspace_bytes() == size.value
    plan._device = 0
    got = loss_run(pkg, *args, "bf16", plan=plan)
    assert all(torch.equal(got[k], ref[k]) for k in ref)


@pytest.mark.gpu
def test_python_checks_on_device_tensors(pkg):
    hidden, weight, targets, grad = loss_inputs(14, 16, 64, 50, "bf16", 0.0)
    plan = pkg.VocabLossPlan(16, 64, 50)
    loss = torch.empty(16, device="cuda")
    with pytest.raises(TypeError):
        plan.execute(loss, loss, hidden.half(), weight, targets)
    with pytest.raises(ValueError):
        plan.execute(loss, loss, hidden[:, :32], weight, targets)
    with pytest.raises(ValueError):
        plan.execute(loss, loss, hidden, weight.T.contiguous().T, targets)
    with pytest.raises(ValueError):
        plan.execute_grad(hidden[:1].expand(16, 64), None, hidden, weight, targets, loss, grad)
    with pytest.raises(pkg.TcError) as e:
        plan.execute(torch.empty(17, device="cuda"), torch.empty(17, device="cuda"), torch.cat((hidden, hidden[:1])), weight, torch.cat((targets, targets[:1])))
    assert e.value.status == EXTENT


# --------------------------------------------------------------------------------------------- orthogonalised updates ----
COEF = (3.4445, -4.7750, 2.0315)


def orthogonal_reference(x, coefficients, eps):
    x = x.double()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    for a, b, c in coefficients:
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * g @ g) @ x
    return x.transpose(1, 2) if tall else x


def orthogonal_bound(kind_in, kind_out, steps):
    """Three roundings to 11 bits per step and the input's (none for fp16), each at most 2^-11 of what it rounds, as if all
    added up; and the output's own."""
    return (3 * steps + 1) * 2.0 ** -11 + unit(kind_out)


ORTHS = [  # batch, rows, cols, type in, type out, steps
    (1, 1, 1, "f32", "bf16", 5), (1, 1, 100, "bf16", "bf16", 5), (3, 100, 1, "f16", "f16", 2), (2, 16, 24, "bf16", "f16", 5), (12, 128, 64, "f32", "bf16", 5),
    (1, 127, 129, "f32", "f16", 5), (1, 333, 200, "bf16", "bf16", 5), (2, 256, 256, "f16", "f16", 5), (1, 513, 1300, "bf16", "bf16", 5), (1, 1300, 515, "f32", "f16", 5),
    (5, 384, 768, "bf16", "bf16", 1), (1, 2000, 2048, "bf16", "bf16", 5),
    # up to 128 rows and 4096 columns: clusters of 1, 2, 4 and 8; beyond
    (7, 64, 256, "bf16", "bf16", 5), (40, 128, 257, "f16", "bf16", 5), (5, 300, 128, "f32", "bf16", 5), (2, 100, 700, "bf16", "bf16", 1),
    (1, 65, 1025, "bf16", "f16", 5), (3, 1100, 9, "f32", "f16", 3), (1, 128, 4096, "bf16", "bf16", 5), (1, 4095, 77, "f16", "bf16", 5),
    (1, 96, 4097, "bf16", "bf16", 5), (2, 129, 300, "bf16", "bf16", 5)]


def orthogonal_close(got, ref, tol):
    for g, r in zip(got.double(), ref):
        off = (g - r).norm().item() / max(r.norm().item(), 1e-300)
        assert off <= tol, "%.3e over %.3e" % (off, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols,kind,out_kind,steps", ORTHS)
def test_orthogonal(pkg, batch, rows, cols, kind, out_kind, steps):
    x = (randn(new_gen(rows + cols), batch, rows, cols) * 0.01).to(TYPES[kind])
    out = torch.full((batch, rows, cols), float("nan"), device="cuda", dtype=TYPES[out_kind])
    plan = pkg.OrthogonalPlan(rows, cols, batch=batch, dtype=code(pkg, kind), out_dtype=code(pkg, out_kind), steps=steps, coefficients=COEF)
    plan.execute(out, x)
    assert plan.status() == 0
    ref = orthogonal_reference(x, [COEF] * steps, 1e-7)
    orthogonal_close(out, ref, orthogonal_bound(kind, out_kind, steps))
    again = torch.empty_like(out)
    plan.execute(again, x)
    assert torch.equal(out, again)


@pytest.mark.gpu
def test_orthogonal_strides_and_own_coefficients(pkg):
    coefficients = [(4.0848, -6.8946, 2.9270), (3.9505, -6.3029, 2.6377), (1.875, -1.25, 0.375)]
    x = (randn(new_gen(2), 4, 90, 201)).to(torch.bfloat16)
    ref = orthogonal_reference(x, coefficients, 0.0)
    plan = pkg.OrthogonalPlan(90, 201, batch=4, steps=3, coefficients=coefficients, eps=0.0)
    tol = orthogonal_bound("bf16", "bf16", 3)
    padded = torch.full((4, 97, 208), 5.0, device="cuda", dtype=torch.bfloat16)
    plan.execute(padded[:, :90, :201], x)
    orthogonal_close(padded[:, :90, :201], ref, tol)
    assert bool((padded[:, 90:] == 5.0).all()) and bool((padded[:, :, 201:] == 5.0).all())
    turned = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # columns far apart
    out = torch.empty(201, 90, 4, device="cuda", dtype=torch.bfloat16).permute(2, 1, 0)
    plan.execute(out, turned)
    assert torch.equal(out, padded[:, :90, :201])
    columns = torch.empty(4, 201, 90, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    plan.execute(columns, x.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(columns, out)
    plan.execute(out, x[:1].expand(4, 90, 201))  # one matrix four times
    assert all(torch.equal(out[i], out[0]) for i in range(4)) and torch.equal(out[0], padded[0, :90, :201])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_orthogonal_extremes(pkg, kind):
    """Zeros stay zeros, scale does not matter, an infinity or a NaN shows everywhere, in its own matrix only."""
    x = randn(new_gen(4), 6, 48, 80).to(TYPES[kind])
    x[1] = 0
    x[2, 3, 5], x[3, 0, 0] = float("inf"), float("nan")
    x[4] = x[0] * 2.0 ** 8
    x[5] = x[0]
    x[5, 7] = 0  # an empty row
    plan = pkg.OrthogonalPlan(48, 80, batch=6, dtype=code(pkg, kind), out_dtype=pkg.BF16, eps=1e-7)
    out = torch.empty(6, 48, 80, device="cuda", dtype=torch.bfloat16)
    plan.execute(out, x)
    assert bool((out[1] == 0).all()) and bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[3]).all())
    ref = orthogonal_reference(x, [COEF] * 5, 1e-7)
    for i in (0, 4, 5):
        orthogonal_close(out[i:i + 1], ref[i:i + 1], orthogonal_bound(kind, "bf16", 5))
    assert bool((out[5, 7] == 0).all())


# -------------------------------------------------------------------------------------------------------- waits ----
@pytest.mark.gpu
def test_a_product_whose_operands_never_arrive_is_reported(pkg):
    """A stage that is left out makes the waits on it run out: the status word says so, the context stays usable."""
    args = loss_inputs(15, 200, 256, 400, "bf16", 0.0)
    plan = pkg.VocabLossPlan(200, 256, 400)
    pkg._check(pkg.lib().tc_op_set_test_fault(plan._h, 1), "tc_op_set_test_fault")
    loss, lse = (torch.empty(200, device="cuda") for _ in range(2))
    plan.execute(loss, lse, *args[:3])
    assert plan.status() in (20, 21, 22, 23)
    plan.status_reset()
    assert plan.status() == 0
    got = loss_run(pkg, *args, "bf16")
    ref, tol = loss_reference(*args, "bf16")
    within(got["loss"], ref["loss"], tol["loss"], "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(64, 700), (300, 400)])
def test_an_orthogonalisation_whose_products_never_end_is_reported(pkg, rows, cols):
    x = randn(new_gen(16), rows, cols).to(torch.bfloat16)
    out = torch.empty_like(x)
    plan = pkg.OrthogonalPlan(rows, cols)
    pkg._check(pkg.lib().tc_op_set_test_fault(plan._h, 1), "tc_op_set_test_fault")
    plan.execute(out, x)
    assert plan.status() in (20, 21, 22, 23, 24)
    plan = pkg.OrthogonalPlan(rows, cols)
    plan.execute(out, x)
    assert plan.status() == 0
    orthogonal_close(out[None], orthogonal_reference(x[None], [COEF] * 5, 1e-7), orthogonal_bound("bf16", "bf16", 5))


# ------------------------------------------------------------------------------------------------------- together ----
@pytest.mark.gpu
def test_the_example_learns():
    """The three operators and the engine's contractions in a training step (examples/train_step.py)."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_step.py")
    spec = importlib.util.spec_from_file_location("train_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    model = mod.Model(tokens=96, dim=64, vocab=300)
    ids = torch.arange(96, device="cuda") * 3
    targets = (ids * 7 + 3) % 300
    targets[::8] = -1
    # the first step's gradient of the mixing matrix, against autograd in 64 bits on the same bf16 table
    table, mixing = model.table.double(), model.mixing.double().requires_grad_()
    hidden = (table[ids] * 8.0) @ mixing
    part = targets >= 0
    wanted = torch.nn.functional.cross_entropy(hidden[part] @ table.T, targets[part])
    wanted.backward()
    first = model.step(ids, targets).item()
    # hidden is rounded to bf16 (2^-8 of each term of a logit at most, and logits are sums of 64), as are the gradients
    assert abs(first - wanted.item()) <= 2.0 ** -8 * (1 + wanted.item())
    off = (model.momentum.double() - mixing.grad).norm() / mixing.grad.norm()
    assert off <= 4 * 2.0 ** -8, off.item()
    losses = [model.step(ids, targets).item() for _ in range(30)]
    assert losses[-1] < 0.8 * first


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols,kind", [(3, 20, 50, "f16"), (2, 128, 190, "f32"), (1, 100, 193, "bf16"), (2, 1536, 77, "f32"), (1, 60, 1537, "f16"),
                                                  (2, 300, 200, "f32"), (1, 1000, 1333, "f16"), (1, 1300, 2100, "bf16"), (2, 64, 4096, "f16"), (1, 4097, 33, "f32"),
                                                  (1, 65, 1536, "bf16")])
def test_half_precision_results_keep_their_bits(pkg, batch, rows, cols, kind):
    """Two-term operands (at least 17 bits of what is rounded between the products) leave little but the result's own rounding."""
    gen = new_gen(rows * cols)
    few = max(1, min(rows, cols) // 16)  # some directions dominate: small ones are what roundings between the products would disturb
    x = randn(gen, batch, rows, few) @ randn(gen, batch, few, cols) * (2.0 / few ** 0.5) + randn(gen, batch, rows, cols)
    x = (x * 0.01).to(TYPES[kind])
    out = torch.empty(batch, rows, cols, device="cuda", dtype=torch.float16)
    plan = pkg.OrthogonalPlan(rows, cols, batch=batch, dtype=code(pkg, kind), out_dtype=pkg.F16)
    plan.execute(out, x)
    assert plan.status() == 0
    orthogonal_close(out, orthogonal_reference(x, [COEF] * 5, 1e-7), 16 * 2.0 ** -17 + 2.0 ** -11)


@pytest.mark.gpu
def test_a_plans_memory_is_free_of_earlier_work_on_its_stream(pkg):
    """torch's allocator hands out blocks that queued kernels of the same stream still write or read; the plan's first call may run
    on another stream, and its status word is cleared on a third."""
    args = loss_inputs(18, 260, 128, 3000, "bf16", 0.1)
    ref = loss_run(pkg, *args, "bf16")
    size = pkg.VocabLossPlan(260, 128, 3000).workspace_bytes() + 1024
    here, there = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for pending in ("writes", "reads"):
        plan = pkg.VocabLossPlan(260, 128, 3000)
        with torch.cuda.stream(here):
            block, copy = (torch.full((size,), 7, dtype=torch.uint8, device="cuda") for _ in range(2))
            at = block.data_ptr()
            torch.cuda._sleep(200_000_000)  # about a tenth of a second
            if pending == "writes":
                block.fill_(255)
            else:
                copy.copy_(block)
            del block
            plan.commit()
            assert plan._memory.data_ptr() == at
        with torch.cuda.stream(there):
            loss, lse = (torch.empty(260, device="cuda") for _ in range(2))
            dh, dw = torch.empty_like(args[0]), torch.empty_like(args[1])
            plan.execute(loss, lse, *args[:3])
            plan.execute_grad(dh, dw, *args[:3], lse, args[3])
        torch.cuda.synchronize()
        assert plan.status() == 0 and bool((copy == 7).all())
        assert all(torch.equal(a, ref[k]) for a, k in zip((loss, lse, dh, dw), ("loss", "lse", "dhidden", "dweight")))
        del plan, copy


@pytest.mark.gpu
def test_calls_of_two_threads_on_their_own_default_streams_follow_one_another(pkg):
    """Both threads pass the same handle, that of the per-thread default stream, which stands for two streams."""
    import threading
    import time
    args = loss_inputs(19, 260, 128, 3000, "bf16", 0.1)
    plan = pkg.VocabLossPlan(260, 128, 3000).commit()
    ref = loss_run(pkg, *args, "bf16", plan=plan)
    outs = [[torch.empty(260, device="cuda"), torch.empty(260, device="cuda"), torch.empty_like(args[0]), torch.empty_like(args[1])] for _ in range(2)]
    first_queued, failures, early = threading.Event(), [], []
    torch.cuda.synchronize()

    def work(i):
        try:
            mine, done = torch.cuda.ExternalStream(2), torch.cuda.Event()
            if i == 0:
                with torch.cuda.stream(mine):
                    torch.cuda._sleep(600_000_000)  # about a third of a second
            else:
                assert first_queued.wait(30)
            loss, lse, dh, dw = outs[i]
            plan.execute(loss, lse, *args[:3], stream=2)
            plan.execute_grad(dh, dw, *args[:3], lse, args[3], stream=2)
            done.record(mine)
            first_queued.set()
            if i == 1:
                time.sleep(0.05)  # far more than the calls take, far less than the first thread's sleep
                early.append(done.query())
            done.synchronize()
        except BaseException as e:  # noqa: B036 - the main thread reports it
            failures.append(e)
            first_queued.set()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures and early == [False], (failures, early)
    for o in outs:
        assert all(torch.equal(a, ref[k]) for a, k in zip(o, ("loss", "lse", "dhidden", "dweight")))


@pytest.mark.gpu
def test_closing_a_plan_waits_for_calls_with_workspaces_of_their_own(pkg):
    """They report to the plan's status word, whose memory goes back to the allocator."""
    args = loss_inputs(20, 64, 64, 500, "bf16", 0.1)
    ref = loss_run(pkg, *args, "bf16")
    plan = pkg.VocabLossPlan(64, 64, 500).commit()
    size = plan.workspace_bytes()
    streams = [torch.cuda.Stream() for _ in range(20)]
    spaces, outs, ends = [], [], []
    for _ in streams:
        ws = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
        spaces.append(ws[-ws.data_ptr() % 1024:][:size])
        outs.append((torch.empty(64, device="cuda"), torch.empty(64, device="cuda")))
    torch.cuda.synchronize()
    for round_ in range(2):  # the second on streams that the plan has seen
        for s, ws, (loss, lse) in zip(streams, spaces, outs):
            with torch.cuda.stream(s):
                torch.cuda._sleep(20_000_000 * (1 + len(ends) % 3))
                plan.execute(loss, lse, *args[:3], workspace=ws)
                ends.append(torch.cuda.Event())
                ends[-1].record()
    assert not ends[-1].query()
    plan.close()
    assert all(e.query() for e in ends)
    assert all(torch.equal(loss, ref["loss"]) and torch.equal(lse, ref["lse"]) for loss, lse in outs)


@pytest.mark.gpu
def test_captured_calls(pkg):
    """Calls recorded in a graph read what its replay finds; a plan that is not committed is refused and the capture goes on."""
    gen = new_gen(21)
    t, d, v = 300, 96, 2000
    rows, loss = pkg.EmbeddingPlan(t, v, d, scale=2.0).commit(), pkg.VocabLossPlan(t, d, v).commit()
    updates = [pkg.OrthogonalPlan(64, d).commit(), pkg.OrthogonalPlan(t, d + 64, out_dtype=pkg.F16).commit()]
    late = pkg.EmbeddingPlan(t, v, d), pkg.VocabLossPlan(t, d, v), pkg.OrthogonalPlan(64, d)
    half = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
    plans = [rows, loss] + updates
    spaces = []
    for plan in plans:
        ws = torch.empty(plan.workspace_bytes() + 1024, dtype=torch.uint8, device="cuda")
        spaces.append(ws[-ws.data_ptr() % 1024:][:plan.workspace_bytes()])

    def inputs():
        return dict(table=randn(gen, v, d).bfloat16() * 0.1, ids=torch.randint(-1, v, (t,), device="cuda", generator=gen),
                    grad=torch.rand(t, device="cuda", generator=gen), x=randn(gen, t, d + 64).bfloat16())

    def outputs():
        return dict(hidden=half(t, d), losses=half(t, dtype=torch.float32), lse=half(t, dtype=torch.float32), dhidden=half(t, d), dtable=half(v, d),
                    small=half(64, d), large=half(t, d + 64, dtype=torch.float16))

    def calls(i, o, own):
        ws = [dict(workspace=s) if own else {} for s in spaces]
        rows.execute(o["hidden"], i["table"], i["ids"])
        loss.execute(o["losses"], o["lse"], o["hidden"], i["table"], i["ids"], **ws[1])
        loss.execute_grad(o["dhidden"], o["dtable"], o["hidden"], i["table"], i["ids"], o["lse"], i["grad"], **ws[1])
        rows.execute_grad(o["dtable"], o["dhidden"], i["ids"], accumulate=True, **ws[0])
        updates[0].execute(o["small"], i["x"][:64, :d], **ws[2])
        updates[1].execute(o["large"], i["x"], **ws[3])

    for own in (True, False):
        fixed, got, graph = inputs(), outputs(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            for plan, args in zip(late, ((got["hidden"], fixed["table"], fixed["ids"]), (got["losses"], got["lse"], got["hidden"], fixed["table"], fixed["ids"]),
                                         (got["small"], fixed["x"][:64, :d]))):
                with pytest.raises(pkg.TcError) as e:
                    plan.execute(*args)
                assert e.value.status == STATE
            here = torch.cuda.current_stream().cuda_stream
            assert pkg.lib().tc_embedding_execute(late[0]._h, got["hidden"].data_ptr(), d, fixed["table"].data_ptr(), d, fixed["ids"].data_ptr(), pkg.I64, t,
                                                  here) == STATE
            assert pkg.lib().tc_embedding_execute_grad(late[0]._h, got["dtable"].data_ptr(), d, got["hidden"].data_ptr(), d, fixed["ids"].data_ptr(), pkg.I64,
                                                       t, 0, None, 0, here) == STATE
            calls(fixed, got, own)
        for _ in range(2):
            new, want = inputs(), outputs()
            calls(new, want, False)
            torch.cuda.synchronize()
            for k in fixed:
                fixed[k].copy_(new[k])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(got[k], want[k]) for k in got)
        assert all(plan.status() == 0 for plan in plans)
        del graph
    late[1].execute(got["losses"], got["lse"], got["hidden"], fixed["table"], fixed["ids"])
    assert torch.equal(got["losses"], want["losses"])


def test_threads_whose_first_calls_meet_commit_a_plan_once(pkg, monkeypatch):
    """No GPU: the allocator, the stream and the library's commit are stand-ins."""
    import threading
    import time
    plan, commits, failures = pkg.EmbeddingPlan(4, 4, 4), [], []

    class Stand:
        device = "cpu"
        synchronize = lambda self: None  # noqa: E731
        data_ptr = lambda self: 1024  # noqa: E731
        get_device = lambda self: 0  # noqa: E731

        def tc_op_commit_in(self, handle, memory, size):
            commits.append(memory)
            return 0 if len(commits) == 1 else STATE

    def empty(*args, **kw):
        time.sleep(0.05)
        return Stand()

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        m.setattr(torch.cuda, "current_stream", lambda device=None: Stand())
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        m.setattr(plan, "workspace_bytes", lambda: 1024, raising=False)
        m.setattr(pkg, "lib", lambda: Stand())
        gate = threading.Barrier(4)

        def work():
            try:
                gate.wait(10)
                plan._on(0)
            except Exception as e:
                failures.append(e)

        threads = [threading.Thread(target=work) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not failures and len(commits) == 1, failures


MEMORY = [(1, 8192, 262144), (4, 4096, 128256), (16, 2048, 131072), (16, 2047, 131072), (300, 999, 500001), (8192, 2048, 131072), (1, 70000, 262144), (4, 2048, 131072),
          (2, 64, 1000003)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,dim,vocab", MEMORY)
def test_the_loss_keeps_no_second_table(pkg, tokens, dim, vocab, kind):
    """What a plan takes: pieces of G, of partial gradients and of a table that has to be laid out, 256 MB each at most where a tile's
    rows or a token's gradient fit that; tokens' rows in tiles of 128; statistics; 16 bytes per row of the table for few tokens and their
    partial gradients, 16 KB per column of the table at most."""
    pkg_kind = code(pkg, kind)
    got = pkg.VocabLossPlan(tokens, dim, vocab, dtype=pkg_kind).describe()["workspace_bytes"]
    rows, pitch = -(-tokens // 128) * 128, -(-dim // 8) * 8
    packed = 2 * rows * pitch * 2 + rows * 64
    stats = 8 * (vocab // 64 + 2 * (vocab * pitch // (1 << 26)) + 64) * min(rows, 16384) + (1 << 17)
    slab = max(1 << 28, 4 * rows * pitch)
    few = vocab * 16 + (16384 * pitch if 16 * pitch <= 40960 else 0)
    if tokens <= 4 and 16 * pitch <= 40960:  # no pieces at all
        assert got <= packed + few + stats + (1 << 16), got
    assert got <= (2 << 28) + slab + packed + few + stats + 512 * pitch + (1 << 16), got


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,vocab,kind", [(20, 2047, 70001, "bf16"), (3, 8191, 17000, "f16")])
def test_a_table_laid_out_in_pieces(pkg, tokens, dim, vocab, kind):
    """Unaligned rows of a table whose aligned copy takes more than 256 MB; and more columns than few tokens are passed over."""
    args = loss_inputs(22, tokens, dim, vocab, kind, 0.0)
    got = loss_run(pkg, *args, kind)
    ref, tol = loss_reference(*args, kind)
    for name in got:
        within(got[name], ref[name], tol[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(48, 80), (200, 300)])  # one launch, and products
@pytest.mark.parametrize("kind,power", [("bf16", 80), ("bf16", -90), ("f32", 80), ("f32", -90), ("f32", 122), ("bf16", -110)])
def test_orthogonal_of_numbers_whose_squares_leave_32_bits(pkg, kind, power, rows, cols):
    """The norm of finite numbers is finite and not zero, so powers of two do not matter."""
    x = randn(new_gen(rows), 2, rows, cols).to(torch.bfloat16)
    scaled = (x.double() * 2.0 ** power).to(TYPES[kind])
    assert bool(torch.isfinite(scaled).all()) and torch.equal(scaled.double(), x.double() * 2.0 ** power)
    scaled[1, :, cols // 2:] = 0
    out = torch.empty(2, rows, cols, device="cuda", dtype=torch.bfloat16)
    pkg.OrthogonalPlan(rows, cols, batch=2, dtype=code(pkg, kind), out_dtype=pkg.BF16, eps=0.0).execute(out, scaled)
    orthogonal_close(out, orthogonal_reference(scaled, [COEF] * 5, 0.0), orthogonal_bound(kind, "bf16", 5))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,share,extra", [(40, 10000, 1e-6, 0), (300, 4099, 1e-7, 3)])
def test_half_precision_gradients_of_tokens_of_little_weight(pkg, tokens, vocab, share, extra):
    """G is rounded relative to each token's own weight, not to the largest of the call: rows of the gradient by hidden whose token
    weighs a millionth of another's, and rows of the table that only such tokens name, keep their bits."""
    d, u, gen = 64, unit("f16"), new_gen(tokens)
    weight = (1 + 0.1 * randn(gen, vocab, d + extra)).half()[:, :d]
    hidden = randn(gen, tokens, d + extra).half()[:, :d]
    targets = torch.arange(tokens, device="cuda") * 7
    light = torch.arange(tokens, device="cuda") % 2 == 1
    hidden[1::4] = 0  # as many equal probabilities as the table has rows
    hidden[:, 0] = torch.where(light, 0.0, 1.0).half()
    weight[targets[light], 0] = -60.0  # out of the others' reach
    grad = torch.where(light, share, 1.0) * 16384.0
    got = loss_run(pkg, hidden, weight, targets, grad, "f16")
    h, w, g = hidden.double(), weight.double(), grad.double()[:, None]
    z = h @ w.T
    p = torch.softmax(z, 1)
    onehot = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
    # logits and exponents as in loss_reference; a rounding of G relative to itself, or half of the smallest subnormal where the token's
    # weight (or up to half of it) is held at 2^14
    e = (d * 2.0 ** -23 * (h.abs() @ w.abs().T)).amax(1) + 2.0 ** -20 * (1 + z.abs().amax(1)) + vocab * 2.0 ** -23 / 64
    G = g * (p - onehot)
    off = u * G.abs() + (2 * e[:, None] + 2.0 ** -22) * g * (p + onehot) + g * 2.0 ** -38
    # the table's side: the same, and hidden times its share of the largest, whose smallest subnormal lies as far below
    low = 2.0 ** -38 * (g * h).abs().max() * (p - onehot).abs().sum(0)[:, None]
    for name, x, xo, y, n, more in (("dhidden", G, off, w, vocab, 0.0), ("dweight", G.T, off.T, h, tokens, low)):
        want = x @ y
        raw = (xo + n * 2.0 ** -23 * (x.abs() + xo)) @ y.abs() + more
        within(got[name], want, raw + u * (want.abs() + raw) + tiny("f16"), name)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols,out_kind", [(3, 64, 100, "bf16"), (2, 128, 4000, "bf16"), (2, 60, 2100, "f16"), (1, 100, 190, "f16")])
def test_an_orthogonalisation_that_gave_up_leaves_the_others_alone(pkg, batch, rows, cols, out_kind):
    """One CTA's first products are never announced.  It is reported, the batch's other matrices come out right, and so does the next
    call's work beside and behind it."""
    x = randn(new_gen(23), batch, rows, cols).to(torch.bfloat16)
    out = torch.empty(batch, rows, cols, device="cuda", dtype=TYPES[out_kind])
    new = lambda: pkg.OrthogonalPlan(rows, cols, batch=batch, out_dtype=code(pkg, out_kind))  # noqa: E731
    right, broken = new(), new()
    want = torch.empty_like(out)
    right.execute(want, x)
    orthogonal_close(want, orthogonal_reference(x, [COEF] * 5, 1e-7), orthogonal_bound("bf16", out_kind, 5))
    pkg._check(pkg.lib().tc_op_set_test_fault(broken._h, 1), "tc_op_set_test_fault")
    again = torch.empty_like(out)
    for _ in range(3):
        broken.execute(out, x)
        right.execute(again, x)
        assert broken.status() == 24 and right.status() == 0
        assert torch.equal(again, want) and torch.equal(out[1:], want[1:])
        broken.status_reset()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,vocab,extra", [(5, 33, 70, 0), (260, 96, 1000, 0), (2500, 40, 300, 3), (9000, 72, 1111, 0)])
def test_half_precision_gradients_of_weights_of_all_sizes(pkg, tokens, dim, vocab, extra):
    """Weights of either sign over twenty powers of two, zeros among them."""
    hidden, weight, targets, grad = loss_inputs(24 + tokens, tokens, dim, vocab, "f16", 0.2, extra)
    gen = new_gen(25)
    grad = grad * 256 * 2.0 ** -torch.randint(0, 20, (tokens,), device="cuda", generator=gen)
    grad = torch.where(torch.rand(tokens, device="cuda", generator=gen) < 0.1, 0.0, grad) * (torch.randint(0, 2, (tokens,), device="cuda", generator=gen) * 2 - 1)
    targets[2], grad[2] = -1, float("inf")  # takes no part
    args = hidden, weight, targets, grad
    got = loss_run(pkg, *args, "f16")
    clean = torch.where(targets < 0, 0.0, grad)
    ref, tol = loss_reference(hidden, weight, targets, clean, "f16")
    for name in got:
        within(got[name], ref[name], tol[name], name)
    for name in ("dhidden", "dweight"):  # by itself: in other slices of the sum
        within(loss_run(pkg, *args, "f16", want=(name,))[name], ref[name], tol[name], name)
    # a power of two on all weights is one on the gradients, as far as no result leaves its range
    less = loss_run(pkg, hidden, weight, targets, grad * 0.5, "f16")
    for name in ("dhidden", "dweight"):
        large = got[name].abs() > 2.0 ** -12
        assert torch.equal(less[name][large], got[name][large] * 0.5)
