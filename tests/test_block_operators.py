"""The operators inside of a model's block -- microscaled 4-bit numbers and their products, activations kept in 8 bits, norms on the
residual stream -- against plain 64-bit implementations.

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


def new_gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def spread(gen, rows, cols, kind):
    """Numbers whose columns' sizes differ by powers of two."""
    return (randn(gen, rows, cols) * torch.exp2(torch.randint(-6, 7, (cols,), device="cuda", generator=gen).float())).to(TYPES[kind])


def rows_apart(t, extra, fill=0.0):
    """The same matrix with `extra` elements behind each row."""
    out = torch.full((t.shape[0], t.shape[1] + extra), fill, device=t.device, dtype=t.dtype)
    out[:, :t.shape[1]] = t
    return out[:, :t.shape[1]]


def within(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), what
    off = torch.where(torch.isfinite(ref), (got - ref).abs() - tol, 0.0)
    assert off.numel() == 0 or bool((off <= 0).all()), "%s: %.3e over its bound" % (what, off.max().item())


# ------------------------------------------------------------------------------------- microscaled numbers in 64 bits ----
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
POWERS = [2.0 ** k for k in range(-127, 128)]


def micro(x, values):
    """Codes (whole numbers, the sign's bit above the magnitude's) and scales (e + 127) of a matrix's blocks, [rows, blocks, 32] and [rows, blocks]."""
    rows, cols = x.shape
    b = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x.double()
    b = b.view(rows, -1, 32)
    powers = torch.tensor(POWERS, dtype=torch.float64, device=x.device)
    top = b.abs().amax(dim=2)
    bad = ~torch.isfinite(b).all(dim=2)
    scale = torch.searchsorted(powers * values[-1], torch.where(bad, 1.0, top))  # the first that is no smaller
    v = torch.where(bad[:, :, None], 0.0, b) / powers[scale][:, :, None]
    table = torch.tensor(values, dtype=torch.float64, device=x.device)
    middle = (table[1:] + table[:-1]) / 2
    at = torch.searchsorted(middle, v.abs())
    tie = middle[at.clamp(max=len(values) - 2)] == v.abs()
    at = at + (tie & (at % 2 == 1)).long()
    bits = (len(values) - 1).bit_length()
    sign = torch.signbit(v) & ~bad[:, :, None]
    return at + (sign.long() << bits), torch.where(bad, 255, scale)


def micro_values(codes, scales, values, cols):
    bits = (len(values) - 1).bit_length()
    size = torch.tensor(values, dtype=torch.float64, device=codes.device)[codes & ((1 << bits) - 1)]
    v = torch.where(codes >> bits > 0, -size, size) * torch.tensor(POWERS + [float("nan")], dtype=torch.float64, device=codes.device)[scales][:, :, None]
    return v.flatten(1)[:, :cols]


def rounded(x, values):
    return micro_values(*micro(x, values), values, x.shape[1])


def pack4(codes, scales):
    """The bytes as the operators lay them out; bytes of scales that no row has are zeros."""
    flat = codes.flatten(1)
    rows, blocks = scales.shape
    out = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8, device=codes.device)
    out[:rows, :blocks] = scales.to(torch.uint8)
    out = out.view(-1, 4, 32, out.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return (flat[:, 0::2] + 16 * flat[:, 1::2]).to(torch.uint8), out


def quantised(pkg, x, kind, **kw):
    rows, cols = x.shape if not kw.get("transposed") else x.shape[::-1]
    plan = pkg.MicroscalePlan(rows, cols, dtype=code(pkg, kind))
    codes = torch.full(plan.codes_shape, 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(plan.scales_shape, dtype=torch.uint8, device="cuda")
    plan.execute(codes, scales, x, **kw)
    return plan, codes, scales


# ------------------------------------------------------------------------------------------------ refusals (no GPU) ----
def create(pkg, name, *args):
    h = ctypes.c_void_p()
    st = getattr(pkg.lib(), "tc_op_create_" + name)(*args, ctypes.byref(h))
    if st == 0:
        pkg.lib().tc_op_destroy(h)
    return st


def test_plans_refuse_what_they_cannot_do(pkg):
    assert create(pkg, "microscale", 4, 32, pkg.F32) == 0
    assert create(pkg, "microscale", 4, 32, pkg.F64) == INVALID
    assert create(pkg, "microscale", 0, 32, pkg.F32) == EXTENT
    assert create(pkg, "microscale", 4, 1 << 31, pkg.F32) == UNSUPPORTED
    assert create(pkg, "micro_product", 4, 4, 32, pkg.F32) == 0
    assert create(pkg, "micro_product", 4, 4, 32, pkg.I32) == INVALID
    assert create(pkg, "micro_product", 4, 0, 32, pkg.BF16) == EXTENT
    assert create(pkg, "micro_product", 4, 4, 1 << 31, pkg.BF16) == UNSUPPORTED
    assert create(pkg, "checkpoint", 4, 32, pkg.BF16, 2, 1, 1) == 0
    assert create(pkg, "checkpoint", 4, 32, pkg.F32, 2, 1, 0) == 0
    assert create(pkg, "checkpoint", 4, 32, pkg.F32, 2, 1, 1) == UNSUPPORTED
    assert create(pkg, "checkpoint", 4, 32, pkg.BF16, 3, 1, 1) == INVALID
    assert create(pkg, "checkpoint", 4, 32, pkg.BF16, -1, 1, 1) == INVALID
    assert create(pkg, "checkpoint", 4, 0, pkg.BF16, 0, 0, 0) == EXTENT
    assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F32, 1, 1.0, 1e-6) == 0
    assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F16, 1, 1.0, 1e-6) == INVALID
    assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F32, 3, 1.0, 1e-6) == INVALID
    assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F32, 1, float("nan"), 1e-6) == INVALID
    assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F32, 1, 1e39, 1e-6) == INVALID
    for eps in (0.0, -1.0, 1e-31, 1e31, float("nan")):
        assert create(pkg, "residual_norm", 4, 32, pkg.BF16, pkg.F32, 1, 1.0, eps) == INVALID
    assert create(pkg, "residual_norm", -1, 32, pkg.BF16, pkg.F32, 1, 1.0, 1e-6) == EXTENT
    lib = pkg.lib()
    assert lib.tc_op_create_microscale(4, 32, pkg.F32, None) == INVALID and lib.tc_op_create_residual_norm(4, 32, 1, 1, 0, 1.0, 1e-6, None) == INVALID


def test_python_plans_check_their_arguments(pkg):
    with pytest.raises(ValueError):
        pkg.CheckpointPlan(4, 4, activation="tanh")
    with pytest.raises(ValueError):
        pkg.ResidualNormPlan(4, 4, gate="row")
    with pytest.raises(pkg.TcError):
        pkg.ResidualNormPlan(4, 4, eps=0.0)
    with pytest.raises(pkg.TcError):
        pkg.MicroProductPlan(4, 4, 0)
    with pytest.raises(TypeError):
        pkg.MicroscalePlan(4, 32).execute(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8), torch.zeros(4, 32))
    with pytest.raises(TypeError):
        pkg.ResidualNormPlan(4, 4).execute(None, None, None, None)
    with pytest.raises(ValueError):
        pkg.CheckpointPlan(4, 4).restore(torch.zeros(4, 4), torch.zeros(4), torch.zeros(4))
    p = pkg.MicroscalePlan(129, 130)
    assert p.codes_shape == (129, 80) and p.scales_shape == (2, 2, 32, 4, 4) and p.describe()["bytes_per_row"] == 80
    c = pkg.CheckpointPlan(7, 33, gated=True, activation="silu")
    assert c.codes_shape == (7, 128) and c.scales_shape == (7, 4) and c.describe()["scales_per_row"] == 4
    assert not pkg.CheckpointPlan(7, 33, dtype=pkg.F32).products
    assert pkg.MicroProductPlan(8192, 8192, 4096).describe()["slices"] == 1
    assert pkg.ResidualNormPlan(8, 64, gate="token").describe()["gate"] == "token"


def test_calls_refuse_bad_pointers_and_sizes_before_they_touch_a_device(pkg):
    lib = pkg.lib()
    m, q, c, r = pkg.MicroscalePlan(8, 40), pkg.MicroProductPlan(8, 16, 40), pkg.CheckpointPlan(8, 40, gated=True), pkg.ResidualNormPlan(8, 40, gate="token")
    plain = pkg.ResidualNormPlan(8, 40)
    a = 1 << 20  # an address that no call gets as far as using
    assert lib.tc_microscale_execute(q._h, a, 32, a, a, 40, 0, 8, None) == INVALID
    assert lib.tc_microscale_execute(m._h, None, 32, a, a, 40, 0, 8, None) == INVALID
    assert lib.tc_microscale_execute(m._h, a, 16, a, a, 40, 0, 8, None) == EXTENT
    assert lib.tc_microscale_execute(m._h, a, 32, a, a, 40, 0, 9, None) == EXTENT
    assert lib.tc_microscale_execute(m._h, a, 40, a, a, 40, 0, 8, None) == ALIGNMENT
    assert lib.tc_microscale_execute(m._h, a + 8, 32, a, a, 40, 0, 8, None) == ALIGNMENT
    assert lib.tc_microscale_execute(m._h, a, 32, a + 4, a, 40, 0, 8, None) == ALIGNMENT
    assert lib.tc_microscale_execute(m._h, a, 32, a, a + 1, 40, 0, 8, None) == ALIGNMENT
    assert lib.tc_microscale_execute(m._h, a, 32, a, a, -1, 0, 8, None) == EXTENT
    assert lib.tc_microscale_restore(m._h, a, 39, a, 32, a, 8, None) == EXTENT
    assert lib.tc_microscale_restore(m._h, a, 40, a, 32, None, 8, None) == INVALID
    assert lib.tc_micro_product_execute(m._h, a, 16, a, 32, a, a, 32, a, 8, 0, None, 0, None) == INVALID
    assert lib.tc_micro_product_execute(q._h, a, 15, a, 32, a, a, 32, a, 8, 0, None, 0, None) == EXTENT
    assert lib.tc_micro_product_execute(q._h, a, 16, a, 31, a, a, 32, a, 8, 0, None, 0, None) == EXTENT
    assert lib.tc_micro_product_execute(q._h, a, 16, a, 32, a, a, 40, a, 8, 0, None, 0, None) == ALIGNMENT
    assert lib.tc_micro_product_execute(q._h, a + 1, 16, a, 32, a, a, 32, a, 8, 0, None, 0, None) == ALIGNMENT
    assert lib.tc_micro_product_execute(q._h, a, 16, a, 32, a, a, 32, None, 8, 0, None, 0, None) == INVALID
    assert lib.tc_checkpoint_execute(c._h, a, 39, a, a, a, 80, 8, None) == EXTENT
    assert lib.tc_checkpoint_execute(c._h, a, 40, a + 8, a, a, 80, 8, None) == ALIGNMENT
    assert lib.tc_checkpoint_execute(c._h, a, 40, a, a, None, 80, 8, None) == INVALID
    assert lib.tc_checkpoint_restore(c._h, None, 40, a, a, 8, None) == INVALID
    assert lib.tc_checkpoint_execute_grad(c._h, a, 79, a, 40, a, a, 8, None) == EXTENT
    assert lib.tc_checkpoint_execute_grad(c._h, a, 80, a, 40, a, None, 8, None) == INVALID
    assert lib.tc_checkpoint_execute_product(c._h, a, 40, pkg.F16, a, 5, a, a, 5, 8, 0, None, 0, None) == INVALID
    assert lib.tc_checkpoint_execute_product(c._h, a, 39, pkg.F32, a, 5, a, a, 5, 8, 0, None, 0, None) == EXTENT
    assert lib.tc_checkpoint_execute_product(c._h, a, 40, pkg.F32, a, 5, a, a, 0, 8, 0, None, 0, None) == EXTENT
    assert lib.tc_checkpoint_execute_product(c._h, a + 2, 40, pkg.F32, a, 5, a, a, 5, 8, 0, None, 0, None) == ALIGNMENT
    bare = pkg.CheckpointPlan(8, 40, products=False)
    assert lib.tc_checkpoint_execute_product(bare._h, a, 40, pkg.F32, a, 5, a, a, 5, 8, 0, None, 0, None) == UNSUPPORTED
    assert lib.tc_residual_norm_execute(r._h, a, 40, None, 0, a, 40, a, 40, None, None, None, 0, 8, None) == INVALID  # no gate
    assert lib.tc_residual_norm_execute(plain._h, a, 40, None, 0, a, 40, a, 40, None, None, a, 40, 8, None) == INVALID
    assert lib.tc_residual_norm_execute(r._h, a, 39, None, 0, a, 40, a, 40, None, None, a, 40, 8, None) == EXTENT
    assert lib.tc_residual_norm_execute(r._h, a, 40, None, 0, a, 40, a + 1, 40, None, None, a, 40, 8, None) == ALIGNMENT
    grad = lambda dx=a, dg=a, dh=a, dn=a, gate=a, plan=r, n=8, ld=40: lib.tc_residual_norm_execute_grad(  # noqa: E731
        plan._h, dx, ld, None, 0, dg, 40, None, None, dh, 40, dn, 40, a, 40, a, 40, None, None, gate, 40, n, None, 0, None)
    assert grad(dx=None, dg=None) == INVALID and grad(dh=None, dn=None) == INVALID and grad(gate=None) == INVALID
    assert grad(plan=plain, gate=None) == INVALID  # a gradient of no gate
    assert grad(n=9) == EXTENT and grad(ld=39) == EXTENT and grad(dx=a + 1) == ALIGNMENT
    fault = lambda plan: lib.tc_op_set_test_fault(plan._h, 1)  # noqa: E731
    assert fault(m) == INVALID and fault(r) == INVALID and fault(q) == 0 and fault(c) == 0


def test_results_over_arguments_are_refused(pkg):
    """Rows beyond what a block holds are read again once their result is written."""
    lib, a, b, c, d = pkg.lib(), 1 << 20, 1 << 21, 1 << 22, 1 << 23  # addresses that no call gets as far as using
    for dim in (40, 20000):
        r = pkg.ResidualNormPlan(8, dim, gate="token")
        call = lambda h, n, x, f, g: lib.tc_residual_norm_execute(r._h, h, dim, n, dim, x, dim, f, dim, None, None, g, dim, 8, None)  # noqa: E731
        assert [call(*at) for at in ((a, b, a, c, d), (a, b, c, a, d), (a, b, c, d, a), (a, a, b, c, d), (a, b, b, c, d), (a, None, a, c, d))] == [INVALID] * 6
        grad = lambda dx, df, dh, dn, h, f, g: lib.tc_residual_norm_execute_grad(  # noqa: E731
            r._h, dx, dim, df, dim, None, dim, None, None, dh, dim, dn, dim, h, dim, f, dim, None, None, g, dim, 8, None, 0, None)
        assert grad(a, b, a, c, d, d, d) == INVALID and grad(a, b, c, d, d, b, d) == INVALID and grad(a, a, b, c, d, d, d) == INVALID
    for gated in (False, True):
        k = pkg.CheckpointPlan(8, 40, gated=gated)
        assert lib.tc_checkpoint_execute(k._h, a, 80, b, c, a, 80, 8, None) == INVALID
        assert lib.tc_checkpoint_execute_grad(k._h, a, 80, a, 80, b, c, 8, None) == INVALID


# --------------------------------------------------------------------------------------------- microscaled numbers ----
MICROS = [  # rows, cols, type, elements behind each row, transposed
    (1, 1, "bf16", 0, False), (1, 32, "f32", 0, False), (3, 33, "f16", 0, False), (5, 127, "bf16", 1, False), (128, 128, "bf16", 0, False),
    (129, 136, "f16", 8, False), (300, 1000, "f32", 4, False), (257, 4104, "bf16", 0, False), (4000, 520, "bf16", 0, False),
    (1, 1, "bf16", 0, True), (33, 3, "f32", 0, True), (127, 129, "bf16", 1, True), (128, 128, "f16", 0, True), (1000, 70, "f32", 4, True), (264, 513, "bf16", 8, True),
    (65, 260, "f16", 0, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,kind,extra,transposed", MICROS)
def test_microscaled_numbers(pkg, rows, cols, kind, extra, transposed):
    gen = new_gen(rows * cols)
    x = spread(gen, rows, cols, kind)
    x[torch.rand(rows, cols, device="cuda", generator=gen) < 0.1] = 0
    given = rows_apart(x.T.contiguous() if transposed else x, extra, 3.0)
    plan = pkg.MicroscalePlan(rows, cols, dtype=code(pkg, kind))
    wide = torch.full((rows, plan.codes_shape[1] + 16), 0xA5, dtype=torch.uint8, device="cuda")
    codes, scales = wide[:, :plan.codes_shape[1]], torch.full(plan.scales_shape, 0x5A, dtype=torch.uint8, device="cuda")
    plan.execute(codes, scales, given, transposed=transposed)
    want, want_scales = micro(x, E2M1)
    want4, laid_out = pack4(want, want_scales)
    assert torch.equal(codes, want4) and bool((wide[:, plan.codes_shape[1]:] == 0xA5).all())
    # what no row has is left as it was, blocks behind the last are zeros
    row = torch.arange(scales.shape[0] * 128, device="cuda").view(-1, 1, 4, 32, 1).transpose(2, 3)
    there = (row < rows).expand(scales.shape)
    assert torch.equal(scales[there], laid_out[there]) and bool((scales[~there] == 0x5A).all())
    back = torch.full((rows, cols + extra), 7.0, device="cuda").to(TYPES[kind])
    plan.restore(back[:, :cols], codes, scales)
    assert torch.equal(back[:, :cols].double(), micro_values(want, want_scales, E2M1, cols)) and bool((back[:, cols:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_microscaled_borders_and_extremes(pkg, kind, transposed):
    info = torch.finfo(TYPES[kind])
    rows = []
    # every border between two codes, from both sides, below a largest element of 6 and of a little less or more than 6
    for top in (6.0, 6.0 * (1 - 2 * unit(kind)), 6.0 * (1 + 4 * unit(kind)), 4.0, 3.0, 1.0):
        values = [top]
        for a, b in zip(E2M1, E2M1[1:]):
            values += [(a + b) / 2 * s for s in (1.0, -1.0, 1 + 2 * unit(kind), 1 - 2 * unit(kind))]
        rows.append(values + [0.0] * (32 - len(values)))
    rows += [[0.0] * 32, [-0.0] * 32, [info.max] * 32, [info.max, -info.max] + [info.max * k / 32 for k in range(30)], [info.tiny] * 32,
             [info.smallest_normal * 2.0 ** -k for k in range(32)], [info.tiny * k / 8 for k in range(32)], [1.0, float("nan")] + [2.0] * 30,
             [float("inf")] + [1.0] * 31, [-float("inf")] * 32, [info.max] + [info.tiny] * 31]
    x = torch.tensor(rows, dtype=torch.float64, device="cuda").to(TYPES[kind]).repeat(1, 2)
    plan, codes, scales = quantised(pkg, x.T.contiguous() if transposed else x, kind, transposed=transposed)
    want, want_scales = micro(x, E2M1)
    want4, laid_out = pack4(want, want_scales)
    assert torch.equal(codes, want4) and torch.equal(scales, laid_out)
    back = torch.empty_like(x)
    plan.restore(back, codes, scales)
    ref = micro_values(want, want_scales, E2M1, 64)
    assert torch.equal(torch.isnan(back), torch.isnan(ref))
    assert torch.equal(back.double().nan_to_num(0.0), ref.clamp(-info.max, info.max).nan_to_num(0.0).to(TYPES[kind]).double())


PRODUCTS = [  # rows, cols, inner, result, elements behind each row of the result
    (1, 1, 1, "f32", 0), (1, 4096, 1024, "bf16", 0), (2, 130, 33, "f16", 1), (7, 129, 127, "f32", 3), (16, 512, 2048, "bf16", 0), (17, 300, 300, "f32", 0),
    (33, 257, 513, "bf16", 8), (64, 1000, 4097, "f16", 0), (65, 128, 128, "f32", 0), (100, 1100, 640, "bf16", 2), (129, 300, 1000, "f32", 0),
    (200, 4000, 90, "bf16", 0), (333, 1001, 777, "f32", 0), (1000, 2056, 1056, "bf16", 0), (1500, 3000, 520, "f16", 0), (2500, 4999, 257, "bf16", 0),
    (130, 200, 8200, "f32", 1), (256, 128, 16384, "bf16", 0)]


def product_case(pkg, gen, rows, cols, inner):
    a, b = spread(gen, rows, inner, "f32"), randn(gen, cols, inner)
    return quantised(pkg, a, "f32")[1:], quantised(pkg, b, "f32")[1:], rounded(a, E2M1), rounded(b, E2M1)


def product_bound(a, b, inner, kind, ref):
    return inner * 2.0 ** -23 * (a.abs() @ b.abs().T) + 1.01 * unit(kind) * ref.abs() + tiny(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,inner,kind,extra", PRODUCTS)
def test_micro_product(pkg, rows, cols, inner, kind, extra):
    gen = new_gen(rows + cols + inner)
    qa, qb, a, b = product_case(pkg, gen, rows, cols, inner)
    plan = pkg.MicroProductPlan(rows, cols, inner, out_dtype=code(pkg, kind))
    wide = torch.full((rows, cols + extra), 7.0, device="cuda").to(TYPES[kind])
    plan.execute(wide[:, :cols], *qa, *qb)
    ref = a @ b.T
    within(wide[:, :cols], ref, product_bound(a, b, inner, kind, ref), "product")
    assert bool((wide[:, cols:] == 7.0).all())
    again = wide.clone()
    plan.execute(again[:, :cols], *qa, *qb)
    assert torch.equal(again, wide)  # the same bits
    # added to what is there: once more rounded
    plan.execute(again[:, :cols], *qa, *qb, accumulate=True)
    old = wide[:, :cols].double()
    within(again[:, :cols], old + ref, inner * 2.0 ** -23 * (a.abs() @ b.abs().T) + 2.0 ** -23 * (old + ref).abs() + 1.01 * unit(kind) * (old + ref).abs() + tiny(kind), "sum")
    assert plan.status() == 0


@pytest.mark.gpu
def test_micro_product_tiles(pkg):
    """Every tile that the plans above and below may choose, sliced and not."""
    seen = {(tuple(d["tile"]), d["slices"] > 1) for d in (pkg.MicroProductPlan(*p[:3]).describe() for p in PRODUCTS + [(8192, 8192, 4096), (64, 64 * 1024, 512)])}
    assert {t for t, _ in seen} >= {(128, 256), (128, 128), (128, 64), (128, 32), (128, 16)}, seen
    assert {s for _, s in seen} == {True, False}


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 300])
def test_micro_product_of_nan_and_of_fewer_rows(pkg, rows):
    gen = new_gen(rows)
    cols, inner = 400, 700
    x = spread(gen, rows, inner, "bf16")
    x[rows // 2, inner - 1] = float("nan")
    x[0, 40] = float("inf")
    w = randn(gen, cols, inner).bfloat16()
    (_, *qa), (_, *qb) = quantised(pkg, x, "bf16"), quantised(pkg, w, "bf16")
    out = torch.empty(rows, cols, device="cuda")
    plan = pkg.MicroProductPlan(1000, cols, inner, out_dtype=pkg.F32)  # more rows than the call has
    plan.execute(out, *qa, *qb)
    a, b = rounded(x, E2M1), rounded(w, E2M1)
    ref = a @ b.T
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(out[rows // 2]).all())
    within(out, ref, inner * 2.0 ** -23 * (a.nan_to_num(0.0).abs() @ b.abs().T) + 2.0 ** -23 * ref.abs().nan_to_num(0.0), "other rows")
    plan.execute(out[:0], qa[0][:0], qa[1][:0], *qb)
    with pytest.raises(ValueError):
        plan.execute(out, qa[0][:, :16], qa[1], *qb)


@pytest.mark.gpu
def test_scales_of_the_whole_range(pkg):
    """Products of the largest and smallest scales, whose sum is in range or leaves it."""
    x = torch.zeros(3, 64, device="cuda")
    x[0, :32], x[1, 32:], x[2] = 2.0 ** 100, 2.0 ** -100, 2.0 ** 100
    w = torch.zeros(2, 64, device="cuda")
    w[0, :32], w[0, 32:], w[1] = 2.0 ** -110, 2.0 ** 90, 2.0 ** 40
    (_, *qa), (_, *qb) = quantised(pkg, x, "f32"), quantised(pkg, w, "f32")
    out = torch.empty(3, 2, device="cuda")
    pkg.MicroProductPlan(3, 2, 64, out_dtype=pkg.F32).execute(out, *qa, *qb)
    assert torch.equal(out.double(), torch.tensor([[2.0 ** -5, float("inf")], [2.0 ** -5, 2.0 ** -55], [float("inf"), float("inf")]], dtype=torch.float64, device="cuda"))


# -------------------------------------------------------------------------------------------------- kept activations ----
def activate(name, a):
    return a * torch.sigmoid(a) if name == "silu" else a * 0.5 * torch.erfc(a * -(0.5 ** 0.5)) if name == "gelu" else a


def function(name, gated, x):
    if not gated:
        return activate(name, x)
    a, b = x.chunk(2, dim=1)
    return activate(name, a) * b


def kept(x, gated):
    return torch.cat([rounded(p, E4M3) for p in x.chunk(2, dim=1)], dim=1) if gated else rounded(x, E4M3)


# fp32 arithmetic of a function of up to a dozen roundings and library functions of a few last places each
FUNCTION = 64 * 2.0 ** -24


def tail(x, gated):
    """Far out on the left the function is x times a share that is subnormal in fp32: rounded to a multiple of 2^-149, it is off by up to
    2^-150, and by as much again after the product by which it was made; times |x|, and times the other half's value."""
    a, b = x.double().abs().chunk(2, dim=1) if gated else (x.double().abs(), 1.0)
    return a * b * 2.0 ** -149


ACTS = [  # tokens, dim, type, activation, gated, elements behind each row
    (1, 1, "bf16", "silu", False, 0), (3, 33, "f32", "gelu", True, 0), (5, 32, "f16", "none", False, 1), (130, 127, "bf16", "gelu", False, 0),
    (64, 1000, "f16", "silu", True, 8), (257, 520, "bf16", "none", True, 0), (777, 301, "f32", "silu", False, 3), (2000, 2048, "bf16", "silu", True, 0),
    (1500, 1024, "f16", "gelu", False, 0), (5000, 264, "f32", "none", False, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,kind,name,gated,extra", ACTS)
def test_kept_activations(pkg, tokens, dim, kind, name, gated, extra):
    gen = new_gen(tokens + dim)
    parts = 2 if gated else 1
    x = spread(gen, tokens, parts * dim, kind)
    dy = randn(gen, tokens, dim).to(TYPES[kind])
    plan = pkg.CheckpointPlan(tokens, dim, dtype=code(pkg, kind), activation=name, gated=gated)
    codes, scales = (torch.full(s, 0xA5, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    y = torch.full((tokens, dim + extra), 7.0, device="cuda").to(TYPES[kind])
    plan.execute(codes, scales, rows_apart(x, extra, 3.0), y=y[:, :dim])
    parts_of = [micro(p, E4M3) for p in x.chunk(parts, dim=1)]
    assert torch.equal(codes, torch.cat([c.flatten(1) for c, _ in parts_of], dim=1).to(torch.uint8))
    assert torch.equal(scales, torch.cat([s for _, s in parts_of], dim=1).to(torch.uint8))
    size = function(name, gated, x.double()).abs()
    within(y[:, :dim], function(name, gated, x.double()), 1.01 * unit(kind) * size + FUNCTION * size + tiny(kind) + tail(x, gated), "result")
    assert bool((y[:, dim:] == 7.0).all())
    bare = torch.full_like(codes, 1)
    plan.execute(bare, scales, x)
    assert torch.equal(bare, codes)  # without a result

    v = kept(x, gated).requires_grad_()
    ref = function(name, gated, v)
    plan.restore(y[:, :dim], codes, scales)
    within(y[:, :dim], ref.detach(), (1.01 * unit(kind) + FUNCTION) * ref.detach().abs() + tiny(kind) + tail(v.detach(), gated), "restored")
    want, = torch.autograd.grad(ref, v, dy.double())
    dx = torch.full((tokens, parts * dim + extra), 7.0, device="cuda").to(TYPES[kind])
    plan.execute_grad(dx[:, :parts * dim], codes, scales, rows_apart(dy, extra))
    # the derivative is a sum of two terms of either sign: off by their sizes' share
    a = v.detach()[:, :dim]
    slope = (1.0 + a.abs() * torch.exp(-a.abs() / 2)) * (v.detach()[:, dim:].abs() if gated else 1.0)
    terms = torch.cat([slope, activate(name, a).abs()], dim=1) if gated else slope
    terms = terms * dy.double().abs().repeat(1, parts)
    # the second half's is dy times the function, which far out is off as in tail()
    far = torch.cat([torch.zeros_like(a), tail(a, False) * dy.double().abs()], dim=1) if gated else 0.0
    within(dx[:, :parts * dim], want, 1.01 * unit(kind) * want.abs() + FUNCTION * terms + far + tiny(kind), "gradient")
    assert bool((dx[:, parts * dim:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_kept_borders_and_extremes(pkg, kind):
    info = torch.finfo(TYPES[kind])
    middle = [(a + b) / 2 for a, b in zip(E4M3, E4M3[1:])]
    rows = [[448.0 * t] + middle[k:k + 31] for k in range(0, len(middle) - 30, 19) for t in (1.0, 1 - 2 * unit(kind), 1 + 4 * unit(kind))]
    rows += [[0.0] * 32, [-0.0] * 32, [info.max] * 32, [info.max] + [-info.max * k / 32 for k in range(31)], [info.tiny] * 32, [info.smallest_normal * 2.0 ** -k for k in range(32)],
             [1.0, float("nan")] + [2.0] * 30, [float("inf")] + [1.0] * 31, [info.max] + [info.tiny] * 31]
    x = torch.tensor(rows, dtype=torch.float64, device="cuda").to(TYPES[kind])
    plan = pkg.CheckpointPlan(len(rows), 32, dtype=code(pkg, kind))
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    plan.execute(codes, scales, x)
    want, want_scales = micro(x, E4M3)
    assert torch.equal(scales.long(), want_scales) and torch.equal(codes.long(), want.flatten(1))
    back = torch.empty_like(x)
    plan.restore(back, codes, scales)
    ref = micro_values(want, want_scales, E4M3, 32)
    assert torch.equal(torch.isnan(back), torch.isnan(ref))
    # a value that an f16 holds only as a subnormal is rounded to one
    assert torch.equal(back.double().nan_to_num(0.0), ref.clamp(-info.max, info.max).nan_to_num(0.0).to(TYPES[kind]).double())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_activations_far_out(pkg, name):
    x = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 88.0, -88.0, 104.0, -104.0, 1e4, -1e4, 3e38, -3e38, 1e-3, -1e-3]], device="cuda")
    plan = pkg.CheckpointPlan(1, 16, dtype=pkg.F32, activation=name)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    plan.execute(codes, scales, x, y=y)
    ref = activate(name, x.double())
    within(y, ref, FUNCTION * ref.abs() + 2.0 ** -100, "results")
    for value in x[0].tolist():  # alone in its block
        one = torch.tensor([[value] * 16], device="cuda")
        plan.execute(codes, scales, one)
        v = rounded(one, E4M3).requires_grad_()
        slope, = torch.autograd.grad(activate(name, v).sum(), v)
        plan.execute_grad(dx, codes, scales, torch.ones_like(x))
        within(dx, slope, FUNCTION * (slope.abs() + 1) if abs(value) < 100 else FUNCTION * slope.abs() + 2.0 ** -100, "slope at %g" % value)


WEIGHTS = [  # tokens, dim, outputs, type, activation, gated, elements behind each row, gradient's type
    (1, 1, 1, "bf16", "none", False, 0, "bf16"), (3, 33, 5, "f16", "silu", False, 0, "f32"), (130, 127, 300, "bf16", "gelu", True, 1, "f32"),
    (64, 256, 256, "f16", "none", False, 0, "f16"), (1000, 520, 136, "bf16", "silu", True, 8, "bf16"), (4100, 200, 1033, "f16", "none", False, 0, "f32"),
    (500, 2100, 1030, "bf16", "silu", False, 0, "bf16"), (8000, 64, 72, "bf16", "none", False, 0, "bf16"), (1500, 3000, 2504, "bf16", "none", False, 0, "f32"),
    (15000, 40, 2309, "bf16", "none", False, 0, "bf16"), (4096, 100, 130, "f16", "none", False, 0, "f16")]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,outputs,kind,name,gated,extra,out", WEIGHTS)
def test_weight_gradient_from_kept_activations(pkg, tokens, dim, outputs, kind, name, gated, extra, out):
    gen = new_gen(tokens + dim + outputs)
    x, dy = spread(gen, tokens, dim * (2 if gated else 1), kind), randn(gen, tokens, outputs).to(TYPES[kind])
    plan = pkg.CheckpointPlan(tokens, dim, dtype=code(pkg, kind), activation=name, gated=gated)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    plan.execute(codes, scales, x)
    f = function(name, gated, kept(x, gated))
    ref, size = dy.double().T @ f, dy.double().abs().T @ f.abs()
    # the function's value is rounded to the operands' type, unless it is what was kept (which bf16 and f16 hold)
    share = 0.0 if name == "none" and not gated else 1.01 * unit(kind) + FUNCTION
    tol = (tokens * 2.0 ** -23 + share) * size + (tokens * dy.double().abs().max() * tiny(kind))
    wide = torch.full((outputs, dim + extra), 7.0, device="cuda").to(TYPES[out])
    plan.execute_product(wide[:, :dim], rows_apart(dy, extra), codes, scales)
    within(wide[:, :dim], ref, tol + 1.01 * unit(out) * (ref.abs() + tol) + tiny(out), "weight")
    assert bool((wide[:, dim:] == 7.0).all())
    again = wide.clone()
    plan.execute_product(again[:, :dim], rows_apart(dy, extra), codes, scales)
    assert torch.equal(again, wide)  # the same bits
    plan.execute_product(again[:, :dim], dy, codes, scales, accumulate=True)
    both = wide[:, :dim].double() + ref
    within(again[:, :dim], both, tol + (1.01 * unit(out) + 2.0 ** -23) * (both.abs() + tol) + tiny(out), "added")
    assert plan.status() == 0


@pytest.mark.gpu
def test_weight_gradient_of_no_tokens_and_of_a_broadcast_row(pkg):
    gen = new_gen(5)
    plan = pkg.CheckpointPlan(40, 72, dtype=pkg.BF16)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    dw = torch.full((9, 72), 3.0, device="cuda")
    plan.execute_product(dw, torch.empty(0, 9, device="cuda").bfloat16(), codes[:0], scales[:0], accumulate=True)
    assert bool((dw == 3.0).all())
    plan.execute_product(dw, torch.empty(0, 9, device="cuda").bfloat16(), codes[:0], scales[:0])
    assert bool((dw == 0.0).all())
    row = randn(gen, 1, 72).bfloat16()
    plan.execute(codes, scales, row.expand(40, 72))
    dy = randn(gen, 1, 9).bfloat16()
    plan.execute_product(dw, dy.expand(40, 9), codes, scales)
    ref = 40 * dy.double().T @ rounded(row, E4M3)
    within(dw, ref, 41 * 2.0 ** -23 * ref.abs(), "broadcast")


# ------------------------------------------------------------------------------------------------------------- norms ----
NORMS = [  # tokens, dim, type, type of the weights, gate, elements behind each row
    (1, 1, "f32", "f32", "none", 0), (1, 4096, "bf16", "bf16", "channel", 0), (3, 7, "bf16", "f32", "token", 1), (33, 64, "f16", "f16", "channel", 0),
    (130, 257, "f32", "f32", "token", 0), (40, 520, "bf16", "bf16", "none", 8), (300, 1000, "bf16", "f32", "channel", 0), (777, 301, "f16", "f32", "token", 3),
    (1000, 2048, "bf16", "bf16", "token", 0), (50, 4104, "f16", "f16", "channel", 0), (20, 8192, "f32", "f32", "channel", 0), (9, 8200, "bf16", "bf16", "token", 0),
    (70, 16385, "f32", "f32", "channel", 0), (6, 16400, "bf16", "bf16", "channel", 0), (3000, 24, "bf16", "bf16", "channel", 0)]
EPS = 1e-5


def norm_inputs(gen, tokens, dim, kind, wkind, gate):
    s = {"x": spread(gen, tokens, dim, kind), "f": spread(gen, tokens, dim, kind), "dh": randn(gen, tokens, dim).to(TYPES[kind]), "dn": randn(gen, tokens, dim).to(TYPES[kind]),
         "post": (1 + 0.2 * randn(gen, dim)).to(TYPES[wkind]), "pre": (1 + 0.2 * randn(gen, dim)).to(TYPES[wkind]), "gate": None}
    if gate != "none":
        s["gate"] = torch.sigmoid(randn(gen, *((dim,) if gate == "channel" else (tokens, dim)))).to(TYPES[kind])
    return s


def norm_reference(s, scale, stored=None, eps=EPS):
    """h, n, and (h as it was stored) the gradients, with the sizes of what each is a sum of."""
    d = {k: None if v is None else v.double() for k, v in s.items()}
    g = 1.0 if d["gate"] is None else d["gate"]
    rms = lambda v: (v.square().mean(dim=1, keepdim=True) + eps).sqrt()  # noqa: E731
    u = d["f"] / rms(d["f"])
    h = scale * d["x"] + g * d["post"] * u
    out = {"h": (h, abs(scale) * d["x"].abs() + (g * d["post"] * u).abs()), "n": (d["pre"] * h / rms(h), None)}
    # h is off by a share of its terms: so is n, by what its row's norm makes of that
    out["n"] = (out["n"][0], out["n"][0].abs() + d["pre"].abs() * out["h"][1] / rms(h))
    if stored is not None:
        h = stored.double()
        r, q = 1 / rms(d["f"]), 1 / rms(h)
        v, w = h * q, d["dn"] * d["pre"]
        mean = lambda a: a.mean(dim=1, keepdim=True)  # noqa: E731
        dh = d["dh"] + q * (w - v * mean(w * v))
        dh_size = d["dh"].abs() + q * (w.abs() + v.abs() * mean((w * v).abs()))
        out["dx"] = (scale * dh, abs(scale) * dh_size)
        p, p_size = dh * g * d["post"], dh_size * abs(g) * d["post"].abs()
        out["df"] = (r * (p - u * mean(p * u)), r * (p_size + u.abs() * mean(p_size * u.abs())))
        out["dpost"] = ((dh * g * u).sum(dim=0), (dh_size * g * u.abs()).sum(dim=0))
        out["dpre"] = ((d["dn"] * v).sum(dim=0), (d["dn"] * v).abs().sum(dim=0))
        if d["gate"] is not None:
            a, b = dh * u * d["post"], dh_size * (u * d["post"]).abs()
            out["dgate"] = (a, b) if d["gate"].ndim == 2 else (a.sum(dim=0), b.sum(dim=0))
    return out


def norm_share(n):
    """Relative to the terms' sizes: fp32 sums over n and the roundings around them."""
    return (n + 32) * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,kind,wkind,gate,extra", NORMS)
def test_residual_norm(pkg, tokens, dim, kind, wkind, gate, extra):
    gen = new_gen(tokens + dim)
    s = norm_inputs(gen, tokens, dim, kind, wkind, gate)
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=code(pkg, kind), gate=gate, residual_scale=0.75, eps=EPS, weight_dtype=code(pkg, wkind))
    wide = {k: torch.full((tokens, dim + extra), 7.0, device="cuda").to(TYPES[kind]) for k in ("h", "n", "dx", "df", "dgate")}
    o = {k: v[:, :dim] for k, v in wide.items()}
    far = {k: v if v is None or v.ndim == 1 else rows_apart(v, extra, 5.0) for k, v in s.items()}
    plan.execute(o["h"], o["n"], far["x"], far["f"], s["post"], s["pre"], gate=far["gate"])
    vectors = {k: torch.full((dim,), 7.0, device="cuda").to(TYPES[wkind]) for k in ("dpost", "dpre")}
    if gate == "none":
        o["dgate"] = None
    elif gate == "channel":
        o["dgate"] = torch.full((dim,), 7.0, device="cuda").to(TYPES[kind])
    call = lambda o, v: plan.execute_grad(o["dx"], o["df"], v["dpost"], v["dpre"], far["dh"], far["dn"], o["h"], far["f"], s["post"], s["pre"],  # noqa: E731
                                          gate=far["gate"], dgate=o["dgate"])
    call(o, vectors)
    ref = norm_reference(s, 0.75, stored=o["h"])
    for k, (want, size) in ref.items():
        got = vectors[k] if k in vectors else o[k]
        n = dim + (tokens if k in ("dpost", "dpre") or (k == "dgate" and gate == "channel") else 0)
        rounding = unit(wkind if k in vectors else kind)
        within(got, want, norm_share(n) * size + 1.01 * rounding * want.abs() + tiny(wkind if k in vectors else kind), k)
    assert all(bool((w[:, dim:] == 7.0).all()) for w in wide.values())
    twice = {k: None if v is None else v.clone() for k, v in o.items()}
    again = {k: torch.empty_like(v) for k, v in vectors.items()}
    call(twice, again)
    assert all(torch.equal(twice[k], o[k]) for k in o if o[k] is not None) and all(torch.equal(again[k], vectors[k]) for k in vectors)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 9000])
def test_parts_of_a_norm(pkg, dim):
    """Without weights, without a second norm, and one gradient at a time: the same numbers."""
    gen = new_gen(dim)
    tokens = 50
    s = norm_inputs(gen, tokens, dim, "f32", "f32", "channel")
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=pkg.F32, gate="channel", eps=EPS)
    ones = torch.ones(dim, device="cuda")
    h, n, h2, n2 = (torch.empty(tokens, dim, device="cuda") for _ in range(4))
    plan.execute(h, n, s["x"], s["f"], gate=s["gate"])
    plan.execute(h2, n2, s["x"], s["f"], ones, ones, gate=s["gate"])
    assert torch.equal(h, h2) and torch.equal(n, n2)
    plan.execute(h2.zero_(), None, s["x"], s["f"], gate=s["gate"])
    assert torch.equal(h, h2)
    new = lambda: {"dx": torch.empty_like(h), "df": torch.empty_like(h), "dpost": torch.empty(dim, device="cuda"), "dpre": torch.empty(dim, device="cuda"),  # noqa: E731
                   "dgate": torch.empty(dim, device="cuda")}

    def grad(o, dh, dn):
        plan.execute_grad(o.get("dx"), o.get("df"), o.get("dpost"), o.get("dpre"), dh, dn, h, s["f"], s["post"], s["pre"], gate=s["gate"], dgate=o.get("dgate"))
        return o

    every = grad(new(), s["dh"], s["dn"])
    for k in every:
        assert torch.equal(grad({k: torch.empty_like(every[k])}, s["dh"], s["dn"])[k], every[k]), k
    zero = torch.zeros_like(h)
    for dh, dn in ((s["dh"], None), (None, s["dn"])):
        a, b = grad(new(), dh, dn), grad(new(), zero if dh is None else dh, zero if dn is None else dn)
        assert all(torch.equal(a[k], b[k]) for k in a)
    empty = grad({"dpost": every["dpost"], "dpre": every["dpre"], "dgate": every["dgate"]}, s["dh"], s["dn"])
    plan.execute_grad(None, None, empty["dpost"], empty["dpre"], zero[:0], zero[:0], h[:0], s["f"][:0], gate=s["gate"], dgate=empty["dgate"])
    assert all(bool((v == 0).all()) for v in empty.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 2000, 17000])
@pytest.mark.parametrize("kind,power", [("f32", 90), ("bf16", 90), ("f32", -90), ("bf16", 0)])
def test_norms_whose_squares_leave_32_bits(pkg, kind, power, dim):
    """Among rows of zeros; with a large or a small eps beside them."""
    gen = new_gen(dim + power)
    tokens, eps = 12, 1e-30 if power < 0 else 1e-6
    s = norm_inputs(gen, tokens, dim, kind, kind, "none")
    for k in ("x", "f"):
        s[k] = (s[k].double() * 2.0 ** power).to(TYPES[kind])
        s[k][3::4] = 0
    s["dh"] = (s["dh"].double() * 2.0 ** (-20 if power > 0 else 20)).to(TYPES[kind])
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=code(pkg, kind), eps=eps)
    o = {k: torch.empty(tokens, dim, device="cuda", dtype=TYPES[kind]) for k in ("h", "n", "dx", "df")}
    o.update({k: torch.empty(dim, device="cuda", dtype=TYPES[kind]) for k in ("dpost", "dpre")})
    plan.execute(o["h"], o["n"], s["x"], s["f"], s["post"], s["pre"])
    plan.execute_grad(o["dx"], o["df"], o["dpost"], o["dpre"], s["dh"], s["dn"], o["h"], s["f"], s["post"], s["pre"])
    for k, (want, size) in norm_reference(s, 1.0, stored=o["h"], eps=eps).items():
        # 2^-120: what products with a norm's inverse near the smallest numbers lose
        within(o[k], want, norm_share(dim + tokens) * size + 1.01 * unit(kind) * want.abs() + 2.0 ** -120, k)


@pytest.mark.gpu
def test_a_token_with_nan_keeps_to_itself(pkg):
    gen = new_gen(11)
    tokens, dim = 20, 200
    s = norm_inputs(gen, tokens, dim, "bf16", "bf16", "token")
    plan = pkg.ResidualNormPlan(tokens, dim, gate="token")
    clean, dirty = ([torch.empty(tokens, dim, device="cuda").bfloat16() for _ in range(5)] for _ in range(2))
    for o, bad in ((clean, 1.0), (dirty, float("nan"))):
        s["f"][7, 3] = bad
        plan.execute(o[0], o[1], s["x"], s["f"], s["post"], s["pre"], gate=s["gate"])
        plan.execute_grad(o[2], o[3], None, None, s["dh"], s["dn"], o[0], s["f"], s["post"], s["pre"], gate=s["gate"], dgate=o[4])
    others = torch.arange(tokens, device="cuda") != 7
    assert all(torch.equal(a[others], b[others]) for a, b in zip(clean, dirty))
    assert all(bool(torch.isnan(b[7]).all()) for b in dirty)


@pytest.mark.gpu
def test_norm_gradient_against_differences(pkg):
    gen = new_gen(21)
    tokens, dim, step = 6, 48, 2.0 ** -10
    s = norm_inputs(gen, tokens, dim, "f32", "f32", "channel")
    s["x"], s["f"] = randn(gen, tokens, dim), randn(gen, tokens, dim)
    plan = pkg.ResidualNormPlan(tokens, dim, dtype=pkg.F32, gate="channel", residual_scale=0.5, eps=EPS)

    def forward(t):
        h, n = torch.empty(tokens, dim, device="cuda"), torch.empty(tokens, dim, device="cuda")
        plan.execute(h, n, t["x"], t["f"], t["post"], t["pre"], gate=t["gate"])
        return h, n

    h, _ = forward(s)
    got = {"x": torch.empty_like(h), "f": torch.empty_like(h), "post": torch.empty(dim, device="cuda"), "pre": torch.empty(dim, device="cuda"), "gate": torch.empty(dim, device="cuda")}
    plan.execute_grad(got["x"], got["f"], got["post"], got["pre"], s["dh"], s["dn"], h, s["f"], s["post"], s["pre"], gate=s["gate"], dgate=got["gate"])
    for k, g in got.items():
        towards = torch.randint(0, 2, s[k].shape, device="cuda", generator=gen).float() * 2 - 1
        up, down = (forward({**s, k: s[k] + sign * step * towards}) for sign in (1, -1))
        made = sum(((a - b).double() * w.double()).sum() for a, b, w in zip(up, down, (s["dh"], s["dn"]))) / (2 * step)
        want = (g.double() * towards.double()).sum()
        size = (g.double().abs()).sum()
        # third order terms of a step of 2^-10 relative to numbers around one, and fp32 results over it
        assert abs(made - want) <= (64 * step ** 2 + 2.0 ** -22 / step) * (size + tokens * dim), k


@pytest.mark.gpu
@pytest.mark.parametrize("name,gated", [("silu", True), ("gelu", False)])
def test_activation_gradient_against_differences(pkg, name, gated):
    """At inputs that eight bits hold, where what is kept is the input."""
    gen = new_gen(22)
    tokens, dim, step = 5, 64, 2.0 ** -9
    x = rounded(randn(gen, tokens, dim * (2 if gated else 1)), E4M3).float()
    dy = randn(gen, tokens, dim)
    plan = pkg.CheckpointPlan(tokens, dim, dtype=pkg.F32, activation=name, gated=gated)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
    y, dx = [torch.empty(tokens, dim, device="cuda") for _ in range(2)], torch.empty_like(x)
    towards = torch.randint(0, 2, x.shape, device="cuda", generator=gen).float() * 2 - 1
    for out, sign in zip(y, (1, -1)):
        plan.execute(codes, scales, x + sign * step * towards, y=out)
    plan.execute(codes, scales, x)
    plan.execute_grad(dx, codes, scales, dy)
    made = ((y[0] - y[1]).double() * dy.double()).sum() / (2 * step)
    want = (dx.double() * towards.double()).sum()
    assert abs(made - want) <= (8 * step ** 2 + 2.0 ** -21 / step) * (dx.double().abs().sum() + tokens * dim)


# ------------------------------------------------------------------------------------- together, streams, captures ----
class Block:
    """norm -> 4-bit product -> gated activation, kept in 8 bits -> 4-bit product -> norm, and back; weights [out, in] in bf16."""

    def __init__(self, pkg, tokens, dim, hidden, seed=0):
        gen = new_gen(seed)
        self.tokens, self.dim, self.hidden = tokens, dim, hidden
        self.up, self.down = (randn(gen, 2 * hidden, dim) * dim ** -0.5).bfloat16(), (randn(gen, dim, hidden) * hidden ** -0.5).bfloat16()
        self.post, self.pre, self.gate = ((1 + 0.1 * randn(gen, dim)).bfloat16() for _ in range(3))
        self.norm = pkg.ResidualNormPlan(tokens, dim, gate="channel", residual_scale=0.9)
        self.act = pkg.CheckpointPlan(tokens, hidden, activation="silu", gated=True)
        self.micro = {k: pkg.MicroscalePlan(*k) for k in {(tokens, dim), (2 * hidden, dim), (tokens, hidden), (dim, hidden), (tokens, 2 * hidden), (hidden, dim), (dim, 2 * hidden)}}
        self.product = {k: pkg.MicroProductPlan(*k) for k in {(tokens, 2 * hidden, dim), (tokens, dim, hidden), (tokens, hidden, dim), (tokens, dim, 2 * hidden)}}
        self.weight = pkg.CheckpointPlan(tokens, dim)
        self.plans = [self.norm, self.act, self.weight, *self.micro.values(), *self.product.values()]
        for p in self.plans:
            p.commit()
        half = lambda *shape: torch.empty(*shape, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        small = lambda p: [torch.zeros(s, device="cuda", dtype=torch.uint8) for s in (p.codes_shape, p.scales_shape)]  # noqa: E731
        t, d, h = tokens, dim, hidden
        self.kept, self.kept_in = small(self.act), small(self.weight)
        self.q = {name: small(self.micro[k]) for name, k in (("n", (t, d)), ("up", (2 * h, d)), ("y", (t, h)), ("down", (d, h)), ("df", (t, d)), ("downT", (h, d)),
                                                            ("da", (t, 2 * h)), ("upT", (d, 2 * h)))}
        self.o = {"h": half(t, d), "n": half(t, d), "a": half(t, 2 * h), "y": half(t, h), "f": half(t, d), "h2": half(t, d), "n2": half(t, d), "df": half(t, d), "dy": half(t, h),
                  "da": half(t, 2 * h), "dn": half(t, d), "dh": half(t, d), "dx": half(t, d), "df0": half(t, d), "dpost": half(d), "dpre": half(d), "dgate": half(d),
                  "dup": torch.empty(2 * h, d, device="cuda"), "ddown": half(d, h)}

    def matmul(self, out, name, x, wname, w, transposed=False):
        t, k = x.shape
        n = out.shape[1]
        self.micro[(t, k)].execute(*self.q[name], x)
        self.micro[(n, k)].execute(*self.q[wname], w, transposed=transposed)
        self.product[(t, n, k)].execute(out, *self.q[name], *self.q[wname])

    def run(self, x, f0, dh2, dn2):
        o = self.o
        self.norm.execute(o["h"], o["n"], x, f0, self.post, self.pre, gate=self.gate)
        self.weight.execute(*self.kept_in, o["n"])
        self.matmul(o["a"], "n", o["n"], "up", self.up)
        self.act.execute(*self.kept, o["a"], y=o["y"])
        self.matmul(o["f"], "y", o["y"], "down", self.down)
        self.norm.execute(o["h2"], o["n2"], o["h"], o["f"], self.post, self.pre, gate=self.gate)
        # back: by the second norm, the projections and the first norm
        self.norm.execute_grad(o["dh"], o["df"], None, None, dh2, dn2, o["h2"], o["f"], self.post, self.pre, gate=self.gate)
        self.act.execute_product(o["ddown"], o["df"], *self.kept)
        self.matmul(o["dy"], "df", o["df"], "downT", self.down, transposed=True)
        self.act.execute_grad(o["da"], *self.kept, o["dy"])
        self.weight.execute_product(o["dup"], o["da"], *self.kept_in)
        self.matmul(o["dn"], "da", o["da"], "upT", self.up, transposed=True)
        self.norm.execute_grad(o["dx"], o["df0"], o["dpost"], o["dpre"], o["dh"], o["dn"], o["h"], f0, self.post, self.pre, gate=self.gate, dgate=o["dgate"])
        return o


def block_inputs(tokens, dim, seed=1):
    gen = new_gen(seed)
    return [randn(gen, tokens, dim).bfloat16() for _ in range(4)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim,hidden", [(1, 64, 96), (200, 256, 392), (333, 129, 200)])
def test_a_block_of_all_of_them(pkg, tokens, dim, hidden):
    """Each step against its own definition, on what the step before it gave."""
    block, (x, f0, dh2, dn2) = Block(pkg, tokens, dim, hidden), block_inputs(tokens, dim)
    o = block.run(x, f0, dh2, dn2)
    assert all(p.status() == 0 for p in block.plans)
    kind = "bf16"

    def product(got, x, w):
        a, b = rounded(x, E2M1), rounded(w, E2M1)
        ref = a @ b.T
        within(got, ref, product_bound(a, b, x.shape[1], kind, ref), "product")

    def norm(s, got, stored):
        for k, (want, size) in norm_reference(s, 0.9, stored=stored, eps=1e-6).items():
            if got.get(k) is not None:
                within(got[k], want, norm_share(dim + tokens) * size + 1.01 * unit(kind) * want.abs() + tiny(kind), k)

    s = {"post": block.post, "pre": block.pre, "gate": block.gate}
    norm({**s, "x": x, "f": f0, "dh": o["dh"], "dn": o["dn"]}, {"h": o["h"], "n": o["n"], "dx": o["dx"], "df": o["df0"], "dpost": o["dpost"], "dpre": o["dpre"], "dgate": o["dgate"]},
         o["h"])
    product(o["a"], o["n"], block.up)
    y = function("silu", True, o["a"].double())
    within(o["y"], y, (1.01 * unit(kind) + FUNCTION) * y.abs() + tiny(kind), "y")
    product(o["f"], o["y"], block.down)
    norm({**s, "x": o["h"], "f": o["f"], "dh": dh2, "dn": dn2}, {"h": o["h2"], "n": o["n2"], "df": o["df"]}, o["h2"])
    v = kept(o["a"], True).requires_grad_()
    f = function("silu", True, v)
    size = o["df"].double().abs().T @ f.detach().abs()
    ref = o["df"].double().T @ f.detach()
    within(o["ddown"], ref, (tokens * 2.0 ** -23 + 1.02 * unit(kind)) * size + 1.02 * unit(kind) * ref.abs() + 1e-30, "down")
    product(o["dy"], o["df"], block.down.T)
    da, = torch.autograd.grad(f, v, o["dy"].double())
    within(o["da"], da, 1.01 * unit(kind) * da.abs() + FUNCTION * (1 + v.detach().abs().amax()) ** 2 * o["dy"].double().abs().repeat(1, 2), "da")
    ref, size = o["da"].double().T @ rounded(o["n"], E4M3), o["da"].double().abs().T @ rounded(o["n"], E4M3).abs()
    within(o["dup"], ref, (tokens + 2) * 2.0 ** -23 * size, "up")
    product(o["dn"], o["da"], block.up.T)


@pytest.mark.gpu
def test_a_captured_block(pkg):
    tokens, dim, hidden = 150, 128, 160
    block, inputs = Block(pkg, tokens, dim, hidden), block_inputs(tokens, dim)
    want = {k: v.clone() for k, v in block.run(*inputs).items()}
    torch.cuda.synchronize()
    given = [torch.zeros_like(t) for t in inputs]
    for v in block.o.values():
        v.fill_(5.0)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        block.run(*given)
    for _ in range(2):
        for a, b in zip(given, inputs):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(block.o[k], want[k]) for k in want)
        for a in given:
            a.zero_()
        graph.replay()
    del graph


@pytest.mark.gpu
def test_calls_on_several_streams(pkg):
    """Calls in the plan's own workspace follow one another; calls with workspaces of their own may overlap."""
    gen = new_gen(31)
    tokens, dim, outputs = 3000, 1000, 520
    plan = pkg.CheckpointPlan(tokens, dim, activation="gelu")
    norm = pkg.ResidualNormPlan(tokens, dim, gate="none")
    product = pkg.MicroProductPlan(40, outputs, dim).commit()
    sets = []
    for _ in range(4):
        x, dy, h, f = (randn(gen, tokens, n).bfloat16() for n in (dim, outputs, dim, dim))
        codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (plan.codes_shape, plan.scales_shape))
        plan.execute(codes, scales, x)
        (_, *qa), (_, *qb) = quantised(pkg, x[:40], "bf16"), quantised(pkg, randn(gen, outputs, dim).bfloat16(), "bf16")
        sets.append(dict(codes=codes, scales=scales, dy=dy, h=h, f=f, dh=x, qa=qa, qb=qb, ws=[torch.empty(p.workspace_bytes() + 1024, dtype=torch.uint8, device="cuda")
                                                                                            for p in (plan, norm, product)]))
    aligned = lambda w: w[-w.data_ptr() % 1024:][:w.numel() - 1024]  # noqa: E731

    def calls(s, own):
        ws = [aligned(w) if own else None for w in s["ws"]]
        o = [torch.empty(outputs, dim, device="cuda").bfloat16(), torch.empty(tokens, dim, device="cuda").bfloat16(), torch.empty(dim, device="cuda").bfloat16(),
             torch.empty(40, outputs, device="cuda").bfloat16()]
        plan.execute_product(o[0], s["dy"], s["codes"], s["scales"], workspace=ws[0])
        norm.execute_grad(None, o[1], o[2], None, s["dh"], None, s["h"], s["f"], workspace=ws[1])
        product.execute(o[3], *s["qa"], *s["qb"], workspace=ws[2])
        return o

    want = [calls(s, False) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for own in (False, True):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(calls(s, own))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    with pytest.raises(pkg.TcError) as e:
        product.execute(want[0][3], *sets[0]["qa"], *sets[0]["qb"], workspace=aligned(sets[0]["ws"][2])[:512])
    assert e.value.status == WORKSPACE


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [8, 600])
def test_products_whose_operands_never_arrive_are_reported(pkg, rows):
    gen = new_gen(rows)
    x, w = randn(gen, rows, 4096).bfloat16(), randn(gen, 300, 4096).bfloat16()
    (_, *qa), (_, *qb) = quantised(pkg, x, "bf16"), quantised(pkg, w, "bf16")
    out = torch.empty(rows, 300, device="cuda").bfloat16()
    plan = pkg.MicroProductPlan(rows, 300, 4096)
    assert pkg.lib().tc_op_set_test_fault(plan._h, 1) == 0
    plan.execute(out, *qa, *qb)
    assert plan.status() in range(30, 36)
    plan.status_reset()
    assert plan.status() == 0
    kept_plan = pkg.CheckpointPlan(rows, 4096)
    assert pkg.lib().tc_op_set_test_fault(kept_plan._h, 1) == 0
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="cuda") for s in (kept_plan.codes_shape, kept_plan.scales_shape))
    kept_plan.execute(codes, scales, x)
    assert kept_plan.status() == 0
    if rows > 200:  # more than one stage
        kept_plan.execute_product(torch.empty(300, 4096, device="cuda"), randn(gen, rows, 300).bfloat16(), codes, scales)
        assert kept_plan.status() in (20, 21, 22, 23)
    good = pkg.MicroProductPlan(rows, 300, 4096)
    good.execute(out, *qa, *qb)
    a, b = rounded(x, E2M1), rounded(w, E2M1)
    within(out, a @ b.T, product_bound(a, b, 4096, "bf16", a @ b.T), "another plan")


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [256, 251])
def test_rows_more_than_32_bits_apart(pkg, cols):
    """Inputs and outputs whose rows lie 2^30 + 8 elements apart: the same results as those of compact ones."""
    gen = new_gen(cols)
    rows, apart = 4, (1 << 30) + 8
    memory = torch.empty(3 * apart + 4096, device="cuda", dtype=torch.bfloat16)
    place = lambda k: torch.as_strided(memory, (rows, cols), (apart, 1), 512 * k + (0 if cols % 8 == 0 else 1))  # noqa: E731
    x, f, dh = (randn(gen, rows, cols).bfloat16() for _ in range(3))
    far = [place(k) for k in range(5)]
    for t, v in zip(far, (x, f, dh)):
        t.copy_(v)
    out = lambda *shape: torch.empty(*(shape or (rows, cols)), device="cuda", dtype=torch.bfloat16)  # noqa: E731
    plan = pkg.MicroscalePlan(rows, cols)
    pairs = [[torch.zeros(s, device="cuda", dtype=torch.uint8) for s in (plan.codes_shape, plan.scales_shape)] for _ in range(2)]
    plan.execute(*pairs[0], x)
    plan.execute(*pairs[1], far[0])
    assert all(torch.equal(a, b) for a, b in zip(*pairs))
    plan.restore(far[3], *pairs[0])
    assert torch.equal(far[3], rounded(x, E2M1).bfloat16())
    weights = quantised(pkg, randn(gen, cols, cols).bfloat16(), "bf16")[1:]
    product, near = pkg.MicroProductPlan(rows, cols, cols), out()
    product.execute(near, *pairs[0], *weights)
    product.execute(far[3], *pairs[0], *weights)
    assert torch.equal(far[3], near)
    act, y, dx = pkg.CheckpointPlan(rows, cols, activation="gelu"), out(), out()
    kept_pairs = [[torch.zeros(s, device="cuda", dtype=torch.uint8) for s in (act.codes_shape, act.scales_shape)] for _ in range(2)]
    act.execute(*kept_pairs[0], x, y=y)
    act.execute(*kept_pairs[1], far[0], y=far[3])
    assert all(torch.equal(a, b) for a, b in zip(*kept_pairs)) and torch.equal(far[3], y)
    act.execute_grad(dx, *kept_pairs[0], dh)
    act.execute_grad(far[3], *kept_pairs[0], far[2])
    assert torch.equal(far[3], dx)
    dw = [out(cols, cols) for _ in range(2)]
    for d, dy in zip(dw, (dh, far[2])):
        act.execute_product(d, dy, *kept_pairs[0])
    assert torch.equal(*dw)
    some = out(rows, cols)
    act.execute_product(some, dh[:, :rows].contiguous(), *kept_pairs[0])
    act.execute_product(far[3], dh[:, :rows].contiguous(), *kept_pairs[0])
    assert torch.equal(far[3], some)
    norm, h, n, df = pkg.ResidualNormPlan(rows, cols), out(), out(), out()
    norm.execute(h, n, x, f)
    norm.execute(far[3], far[4], far[0], far[1])
    assert torch.equal(far[3], h) and torch.equal(far[4], n)
    norm.execute_grad(dx, df, None, None, dh, None, h, f)
    norm.execute_grad(far[4], None, None, None, far[2], None, far[3], far[1])
    assert torch.equal(far[4], dx)
    norm.execute_grad(None, far[4], None, None, far[2], None, far[3], far[1])
    assert torch.equal(far[4], df)


@pytest.mark.gpu
def test_python_checks_on_device_tensors(pkg):
    x = torch.zeros(4, 40, device="cuda").bfloat16()
    m, c, r = pkg.MicroscalePlan(4, 40), pkg.CheckpointPlan(4, 40, gated=True, activation="silu"), pkg.ResidualNormPlan(4, 40, gate="channel")
    codes, scales = (torch.zeros(s, device="cuda", dtype=torch.uint8) for s in (m.codes_shape, m.scales_shape))
    with pytest.raises(ValueError):
        m.execute(codes, scales, x, transposed=True)
    with pytest.raises(ValueError):
        m.execute(codes, scales[:, :0], x)
    with pytest.raises(TypeError):
        m.execute(codes, scales, x.float())
    with pytest.raises(TypeError):
        m.execute(codes.char(), scales, x)
    with pytest.raises(ValueError):
        m.restore(x[:1].expand(4, 40), codes, scales)
    with pytest.raises(pkg.TcError) as e:
        pkg.MicroscalePlan(3, 40).execute(codes, scales, x)
    assert e.value.status == EXTENT
    kc, ks = (torch.zeros(s, device="cuda", dtype=torch.uint8) for s in (c.codes_shape, c.scales_shape))
    with pytest.raises(ValueError):
        c.execute(kc, ks, x)  # half of its columns
    with pytest.raises(ValueError):
        c.execute(torch.zeros(4, 256, device="cuda", dtype=torch.uint8)[:, :128], ks, x.repeat(1, 2))
    with pytest.raises(TypeError):
        c.execute_product(torch.zeros(5, 40, device="cuda", dtype=torch.float64), torch.zeros(4, 5, device="cuda").bfloat16(), kc, ks)
    with pytest.raises(ValueError):
        r.execute(x, None, x.clone(), x.clone())  # no gate
    with pytest.raises(ValueError):
        r.execute(x, None, x.clone(), x.clone(), gate=x.clone())
    with pytest.raises(TypeError):
        r.execute(x, None, x.clone(), x.clone(), torch.ones(40, device="cuda"), gate=x[0].clone())
