"""ResidualRmsNormQuant against its formula in 64 bits.

Tolerances.  With u = 2^-24 (half a step of fp32) and n elements a row: h = x + r is off by u; a sum of n squares, each
folded into one of the partial sums, by at most (n + 1) u relative (all terms positive), which halves under the square
root; the square root, the division by n, the addition of epsilon, the products with gamma and rstd add u each.  y is therefore within
(n / 2 + 8) u of the formula, and so is amax.  Codes: q = RINT(y 127 / amax) with both at most (n + 20) u off in all: where the exact quotient is
within 127 (n + 20) u of a half integer the neighbour is as good; everywhere else the code is the exact one.  The MX codes likewise: the
value has to be one of the two that the grid offers for y within (n + 20) u."""

import pytest
import torch

from asc_devkit_b200 import _lib as L
from asc_devkit_b200 import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
EMAX = {L.DT_FP8_E4M3: 8, L.DT_FP8_E5M2: 15, L.DT_FP4X2_E2M1: 2}
TOP = {L.DT_FP8_E4M3: 448.0, L.DT_FP8_E5M2: 57344.0, L.DT_FP4X2_E2M1: 6.0}
DIGITS = {L.DT_FP8_E4M3: (3, -6), L.DT_FP8_E5M2: (2, -14), L.DT_FP4X2_E2M1: (1, 0)}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}


def formula(x, r, g, eps):
    h = x.double().cpu()
    if r is not None:
        h = h + r.double().cpu()
    y = h * g.double().cpu() / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, y


def decode(dst, dt):
    """Codes -> the values they stand for, in 64 bits on the host."""
    if dt == L.DT_FP4X2_E2M1:
        b = dst.cpu()
        codes = torch.stack([b & 15, b >> 4], -1).reshape(b.shape[0], -1).long()
        mags = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        return mags[codes & 7] * torch.where(codes >= 8, -1.0, 1.0)
    kind = torch.float8_e4m3fn if dt == L.DT_FP8_E4M3 else torch.float8_e5m2
    return dst.cpu().view(kind).double()


def to_grid(v, dt):
    """Nearest value of the element type to v (ties to even, saturating), in 64 bits."""
    digits, lowest = DIGITS[dt]
    v = v.clamp(-TOP[dt], TOP[dt])
    grain = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** lowest))) - digits)
    return torch.round(v / grain) * grain


def inputs(m, n, dt, residual=True, gdt=None, seed=0, pitch=0):
    g = torch.Generator().manual_seed(seed + 1000 * m + n)
    def mat(scale):
        t = torch.zeros(m, n + pitch, dtype=dt, device=DEV)
        t[:, :n] = (torch.randn(m, n, generator=g) * scale).to(DEV)
        return t[:, :n]
    x, r = mat(0.7), mat(1.5) if residual else None
    gamma = (1 + 0.2 * torch.randn(n, generator=g)).to(gdt or dt).to(DEV)
    return x, r, gamma


def run(x, r, gamma, dt, eps=1e-6, in_place=None, **kw):
    m, n = x.shape
    dst = torch.full((m, n // (2 if dt == L.DT_FP4X2_E2M1 else 1)), 0x55, dtype=torch.int8 if dt == L.DT_I8 else torch.uint8, device=DEV)
    scale = torch.full((m,), 7.0, device=DEV) if dt == L.DT_I8 else torch.full((m, n // 32), 0x55, dtype=torch.uint8, device=DEV)
    total = in_place if in_place is not None else torch.empty(m, n, dtype=x.dtype, device=DEV)
    norm = torch.empty(m, n, dtype=x.dtype, device=DEV)
    ops.ResidualRmsNormQuant(dst, scale, x, gamma, eps, residual=r, residualOut=total, normOut=norm, dst_dtype=dt, **kw)
    torch.cuda.synchronize()
    return dst, scale, total, norm


def check(x, r, gamma, dt, got, eps=1e-6):
    dst, scale, total, norm = got
    n = x.shape[1]
    h, y = formula(x, r, gamma, eps)
    tol = (n + 20) * U
    half = HALF_STEP[x.dtype]
    tiny = float(torch.finfo(x.dtype).smallest_normal) * 2 * half  # half a step among the subnormals
    assert torch.all((total.cpu().double() - h).abs() <= h.abs() * (half + 2 * U) + tiny)
    assert torch.all((norm.cpu().double() - y).abs() <= y.abs() * (half + tol) + tiny)
    if dt == L.DT_I8:
        amax = y.abs().amax(-1)
        want = torch.where(amax > 0, amax / 127, 1.0)
        assert torch.all((scale.cpu().double() - want).abs() <= want * tol)
        q = y / want[:, None]
        assert torch.all((dst.cpu().double() - q).abs() <= 0.5 + 127 * tol)
        return
    unit = torch.exp2(scale.cpu().double() - 127)
    blocks = y.reshape(y.shape[0], -1, 32)
    amax = blocks.abs().amax(-1)
    lo, hi = (torch.floor(torch.log2((amax * s).clamp(min=1e-300))) - EMAX[dt] for s in (1 - tol, 1 + tol))
    e = scale.cpu().double() - 127
    assert torch.all((amax == 0) & (e == 0) | (amax > 0) & (e >= lo.clamp(-127, 127)) & (e <= hi.clamp(-127, 127)))
    v = blocks / unit[..., None]
    got_v = decode(dst, dt).reshape(blocks.shape)
    slack = 2.0 ** -8 if dt == L.DT_FP4X2_E2M1 else 0.0  # fp4 is rounded to bfloat16 first: half a step of that beside tol
    low, high = to_grid(v - v.abs() * (tol + slack), dt), to_grid(v + v.abs() * (tol + slack), dt)
    assert torch.all((got_v >= low) & (got_v <= high))


@gpu
@pytest.mark.parametrize("out", [L.DT_I8, L.DT_FP8_E4M3, L.DT_FP8_E5M2, L.DT_FP4X2_E2M1])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 32), (1, 4096), (3, 64), (5, 416), (300, 1024), (2, 7168), (7, 8224), (2, 16384)])
def test_vector_kernel(m, n, dt, out):
    x, r, g = inputs(m, n, dt)
    check(x, r, g, out, run(x, r, g, out))


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 1), (4, 7), (3, 255), (2, 4097), (5, 20000), (1, 2), (40, 1022), (3, 2049), (2, 8191), (2, 8194), (3, 16382), (1, 16385)])
def test_odd_widths_to_int8(m, n, dt):
    x, r, g = inputs(m, n, dt)
    check(x, r, g, L.DT_I8, run(x, r, g, L.DT_I8))


@gpu
@pytest.mark.parametrize("out", [L.DT_I8, L.DT_FP8_E4M3, L.DT_FP8_E5M2, L.DT_FP4X2_E2M1])
@pytest.mark.parametrize("pitch", [8, 5])
def test_row_pitches(out, pitch):
    """A pitch of 8 elements keeps 16-byte vectors, 5 elements do not."""
    x, r, g = inputs(9, 2048, torch.bfloat16, pitch=pitch)
    check(x, r, g, out, run(x, r, g, out))


@gpu
@pytest.mark.parametrize("n", [256, 255])
def test_slices_of_one_buffer(n):
    """Source, residual, sum and norm as column slices of one matrix: they lie in each other's gaps."""
    x, r, g = inputs(17, n, torch.bfloat16)
    want = run(x, r, g, L.DT_I8)
    wide = torch.zeros(17, 4 * n + 8, dtype=torch.bfloat16, device=DEV)
    xs, rs, total, norm = (wide[:, i * n:(i + 1) * n] for i in range(4))
    xs.copy_(x)
    rs.copy_(r)
    dst, scale = torch.empty_like(want[0]), torch.empty_like(want[1])
    ops.ResidualRmsNormQuant(dst, scale, xs, g, 1e-6, residual=rs, residualOut=total, normOut=norm)
    for a, b in zip(want, (dst, scale, total, norm)):
        assert torch.equal(a, b)
    assert torch.equal(xs, x) and torch.equal(rs, r) and (wide[:, 4 * n:] == 0).all()


@gpu
@pytest.mark.parametrize("out", [L.DT_I8, L.DT_FP8_E4M3])
def test_rows_beyond_the_registers(out):
    x, r, g = inputs(3, 16384 + 32, torch.float16)
    check(x, r, g, out, run(x, r, g, out))


@gpu
@pytest.mark.parametrize("out", [L.DT_I8, L.DT_FP8_E5M2])
def test_float_gamma_no_residual_and_optional_outputs(out):
    x, _, g = inputs(33, 4096, torch.bfloat16, residual=False, gdt=torch.float32)
    full = run(x, None, g, out)
    check(x, None, g, out, full)
    dst, scale = torch.empty_like(full[0]), torch.empty_like(full[1])
    ops.ResidualRmsNormQuant(dst, scale, x, g, 1e-6, dst_dtype=out)
    assert torch.equal(dst, full[0]) and torch.equal(scale, full[1])


@gpu
@pytest.mark.parametrize("n", [4096, 4097])
def test_in_place_residual(n):
    """residualOut may be the residual or the source; same bits as with a tensor of its own."""
    x, r, g = inputs(200, n, torch.bfloat16)
    want = run(x, r, g, L.DT_I8)
    r2 = r.clone()
    got = run(x, r2, g, L.DT_I8, in_place=r2)
    x2 = x.clone()
    got2 = run(x2, r, g, L.DT_I8, in_place=x2)
    for a, b, c in zip(want, got, got2):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
@pytest.mark.parametrize("place", ["own", "src", "residual", "unaligned"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out", [L.DT_FP8_E4M3, L.DT_FP8_E5M2])
def test_mx_codes_next_to_a_tie(out, dt, place):
    """Whole numbers: h and its sum of squares are exact and n is a power of two, so rstd is known to 2^-44 and the code has to be the exact one for
    every element further than 2^-40 from the middle between two codes (three roundings to fp32 would reach 2^-23)."""
    m, n, eps = 4096, 1024, 2.0 ** -20
    g = torch.Generator().manual_seed(5)
    x, r = ((torch.randint(1, 9, (m, n), generator=g) * (1 - 2 * torch.randint(0, 2, (m, n), generator=g))).to(dt).to(DEV) for _ in range(2))
    gamma = (1 + 0.2 * torch.randn(n, generator=g)).to(DEV)
    h = x.double() + r.double()
    y = h * gamma.double() / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    dst, scale = torch.empty(m, n, dtype=torch.uint8, device=DEV), torch.empty(m, n // 32, dtype=torch.uint8, device=DEV)
    if place == "unaligned":
        wide = torch.empty(m, n + 1, dtype=dt, device=DEV)
        wide[:, 1:] = x
        x = wide[:, 1:]
    total = {"own": torch.empty_like(r), "src": x, "residual": r, "unaligned": None}[place]
    ops.ResidualRmsNormQuant(dst, scale, x, gamma, eps, residual=r, residualOut=total, dst_dtype=out)
    v = (y.reshape(m, -1, 32) / torch.exp2(scale.double() - 127)[..., None]).reshape(m, n)
    got = dst.view(torch.float8_e4m3fn if out == L.DT_FP8_E4M3 else torch.float8_e5m2).double()
    low, high = to_grid(v * (1 - 2.0 ** -40), out), to_grid(v * (1 + 2.0 ** -40), out)
    wrong = (got != low) & (got != high)
    assert not wrong.any(), f"{int(wrong.sum())} codes on the wrong side"
    assert total is None or torch.equal(total.double(), h)


@gpu
@pytest.mark.parametrize("place", ["own", "none", "src", "residual", "unaligned", "alone"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out", [L.DT_FP8_E4M3, L.DT_FP8_E5M2, L.DT_FP4X2_E2M1])
def test_block_exponents_next_to_a_power_of_two(out, dt, place):
    """One element of a block decides its exponent, and gamma puts it within a few of its own steps of a power of two.  Whole numbers, n a power of
    two: h and the sum are exact and rstd is known to 2^-44, so what is left is the rounding of h * gamma, half a step of fp32: the exponent has
    to be the exact one wherever |y| is further than 2^-24 + 2^-40 from the power."""
    n, eps, calls = 1024, 2.0 ** -20, 60
    rng = torch.Generator().manual_seed(31)
    wrong = sided = 0
    for call in range(calls):
        def whole(low, high, *shape):
            return torch.randint(low, high + 1, shape, generator=rng) * (1 - 2 * torch.randint(0, 2, shape, generator=rng))
        x, r = whole(1, 8, 1, n), whole(1, 8, 1, n)
        at = torch.arange(32) * 32 + torch.randint(0, 32, (32,), generator=rng)
        x[0, at], r[0, at] = 20 + whole(1, 9, 32), 9 + whole(1, 6, 32)   # h from 14 to 44
        if place == "alone":
            x, r = x + r, torch.zeros_like(r)
        h = (x + r).double()
        rstd = 1 / torch.sqrt((h * h).mean() + eps)
        power = 2.0 ** torch.randint(-3, 4, (32,), generator=rng)
        gamma = torch.full((n,), 2.0 ** -9)
        near = (power / (h[0, at] * rstd)).float()
        gamma[at] = near + torch.randint(-2, 3, (32,), generator=rng) * (torch.nextafter(near, 2 * near) - near)
        xs, rs, gs = x.to(dt).to(DEV), r.to(dt).to(DEV), gamma.to(DEV)
        if place == "unaligned":
            wide = torch.empty(1, n + 1, dtype=dt, device=DEV)
            wide[:, 1:] = xs
            xs = wide[:, 1:]
        total = {"own": torch.empty_like(rs), "src": xs, "residual": rs}.get(place)
        dst = torch.empty(1, n // (2 if out == L.DT_FP4X2_E2M1 else 1), dtype=torch.uint8, device=DEV)
        scale = torch.empty(1, 32, dtype=torch.uint8, device=DEV)
        ops.ResidualRmsNormQuant(dst, scale, xs, gs, eps, residual=None if place == "alone" else rs, residualOut=total, dst_dtype=out)
        y = (h * gamma.double() * rstd).reshape(32, 32).abs().amax(-1)
        clear = (y / power - 1).abs() > 2.0 ** -24 + 2.0 ** -40
        want = torch.floor(torch.log2(power)) - (y < power).double() - EMAX[out]
        wrong += int(((scale[0].cpu().double() - 127 != want) & clear).sum())
        sided += int((y < power).sum())
    assert 32 * calls / 4 < sided < 32 * calls * 3 / 4   # both sides are met
    assert wrong == 0, f"{wrong} exponents on the wrong side"


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("out", [L.DT_FP8_E4M3, L.DT_FP8_E5M2])
@pytest.mark.parametrize("small", [False, True])
def test_mx_codes_do_not_depend_on_the_outputs_or_the_alignment(small, out, dt):
    """The same values with residualOut, without it, in the place of either operand and from unaligned rows: the same codes, also where one
    operand is 0 or far below the other.  Whole numbers, whose squares add up exactly in any order; with small operands (2^-13 of whole
    numbers) only the calls of one kernel are compared."""
    m, n = 16384, 2048
    g = torch.Generator(device=DEV).manual_seed(9)
    def whole():
        return torch.randint(1, 17, (m, n), generator=g, device=DEV) * (1 - 2 * torch.randint(0, 2, (m, n), generator=g, device=DEV))
    x, r = whole().to(dt), whole().to(dt)
    r *= 2.0 ** -13 if small else 1.0
    r[torch.rand(m, n, generator=g, device=DEV) < 0.5] = 0
    x[:, ::7] = 0
    gamma = 1 + 0.2 * torch.randn(n, generator=g, device=DEV)
    seen = {}
    for place in ("own", "none", "src", "residual") + (() if small else ("unaligned",)):
        dst, scale = torch.empty(m, n, dtype=torch.uint8, device=DEV), torch.empty(m, n // 32, dtype=torch.uint8, device=DEV)
        xs, rs = x.clone(), r.clone()
        if place == "unaligned":
            wide = torch.empty(m, n + 1, dtype=dt, device=DEV)
            wide[:, 1:] = x
            xs = wide[:, 1:]
        total = {"own": torch.empty_like(r), "src": xs, "residual": rs}.get(place)
        ops.ResidualRmsNormQuant(dst, scale, xs, gamma, 2.0 ** -20, residual=rs, residualOut=total, dst_dtype=out)
        seen[place] = dst, scale
    for place, (dst, scale) in seen.items():
        assert torch.equal(scale, seen["own"][1]), place
        assert torch.equal(dst, seen["own"][0]), f"{place}: {int((dst != seen['own'][0]).sum())} other codes"


@gpu
@pytest.mark.parametrize("pitch", [0, 5])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("out", [L.DT_FP8_E4M3, L.DT_FP8_E5M2, L.DT_FP4X2_E2M1])
def test_small_epsilon_and_blocks_far_below_the_row(out, dt, pitch):
    """Rows of 1e-20 with blocks down to fp32's last normal numbers (and zeros) under an epsilon of 1e-36: rstd is 2^59.8, and for the smaller
    blocks rstd * 2^-e alone would be beyond fp32."""
    x, _, g = inputs(6, 512, dt, residual=False, pitch=pitch)
    factor = torch.exp2(-111.0 - torch.arange(16, device=DEV)).repeat(6, 1)
    factor[:, 0] = 1e-20
    x.copy_((x.float().reshape(6, 16, 32) * factor[..., None]).reshape(6, 512))
    x[:, 5::32] = 0
    check(x, None, g, out, run(x, None, g, out, eps=1e-36), eps=1e-36)


@gpu
@pytest.mark.parametrize("pitch", [0, 5])
@pytest.mark.parametrize("out", [L.DT_FP8_E4M3, L.DT_FP8_E5M2])
def test_codes_next_to_a_tie_under_a_subnormal_epsilon(out, pitch):
    """epsilon 2^-148, squares below 2^-196: rstd is 2^74 to 2^-49, and its remainder has to be a number."""
    m, n = 4096, 1024
    rng = torch.Generator().manual_seed(6)
    wide = torch.zeros(m, n + pitch, device=DEV)
    x = wide[:, :n]
    x.copy_(torch.randint(1, 4097, (m, n), generator=rng).double() * 2.0 ** -110)
    gamma = (2.0 ** 30 * (1 + 0.2 * torch.randn(n, generator=rng))).to(DEV)
    dst, scale = torch.empty(m, n, dtype=torch.uint8, device=DEV), torch.empty(m, n // 32, dtype=torch.uint8, device=DEV)
    ops.ResidualRmsNormQuant(dst, scale, x, gamma, 2.0 ** -148, dst_dtype=out)
    y = x.double() * gamma.double() * 2.0 ** 74
    v = (y.reshape(m, -1, 32) / torch.exp2(scale.double() - 127)[..., None]).reshape(m, n)
    got = dst.view(torch.float8_e4m3fn if out == L.DT_FP8_E4M3 else torch.float8_e5m2).double()
    low, high = to_grid(v * (1 - 2.0 ** -40), out), to_grid(v * (1 + 2.0 ** -40), out)
    wrong = (got != low) & (got != high)
    assert not wrong.any(), f"{int(wrong.sum())} codes on the wrong side"


@gpu
@pytest.mark.parametrize("n", [512, 511])
def test_special_rows_int8(n):
    x, r, g = inputs(8, n, torch.bfloat16, residual=False)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, n - 1] = float("-inf")
    x[4] = 1e30       # its square overflows fp32
    x[5] *= 1e-36     # far below epsilon; the codes still use the whole range
    dst, scale, total, _ = run(x, None, g, L.DT_I8)
    assert torch.equal(torch.isnan(total), torch.isnan(x))  # the conversion to bfloat16 makes every NaN the canonical one
    assert torch.equal(total[~torch.isnan(x)], x[~torch.isnan(x)])
    assert (dst[1] == 0).all() and scale[1] == 1
    for i in (2, 3, 4):
        assert torch.isnan(scale[i]) and (dst[i] == 0).all()
    keep = torch.tensor([0, 5, 6, 7], device=DEV)
    _, y = formula(x[keep], None, g, 1e-6)
    want = y.abs().amax(-1) / 127
    tol = (n + 20) * U
    # row 5's scale is among fp32's subnormals: half a step there is 2^-150
    assert torch.all((scale[keep].cpu().double() - want).abs() <= want * tol + 2.0 ** -149)
    assert torch.all((dst[keep].cpu().double() - y / want[:, None]).abs() <= 0.5 + 127 * tol)


@gpu
def test_special_blocks_mx():
    x, _, g = inputs(4, 128, torch.float32, residual=False)
    x[0, :32] = 0
    x[1, 40] = float("inf")
    x[2] = 0
    x[3] *= 1e-37
    dst, scale, _, _ = run(x, None, g, L.DT_FP8_E4M3)
    assert scale[0, 0] == 127 and (dst[0, :32] & 0x7F == 0).all()
    assert (scale[1] == 0xFF).all() and (dst[1] == 0).all()
    assert (scale[2] == 127).all() and (dst[2] & 0x7F == 0).all()
    rows = torch.tensor([0, 3], device=DEV)
    check(x[rows], None, g, L.DT_FP8_E4M3, (dst[rows], scale[rows], x[rows], formula(x[rows], None, g, 1e-6)[1].float()))


@gpu
def test_saturating_residual_sum():
    x = torch.full((1, 64), 60000.0, dtype=torch.float16, device=DEV)
    g = torch.ones(64, dtype=torch.float16, device=DEV)
    dst, _, total, _ = run(x, x.clone(), g, L.DT_I8)
    assert (total == 65504).all() and (dst == 127).all()


@gpu
def test_other_stream_capture_and_two_launches():
    x, r, g = inputs(64, 1024, torch.bfloat16)
    want = run(x, r, g, L.DT_I8)
    s = torch.cuda.Stream()
    dst, scale = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    s.wait_stream(torch.cuda.current_stream())
    ops.ResidualRmsNormQuant(dst, scale, x, g, 1e-6, residual=r, stream=s)
    s.synchronize()
    assert torch.equal(dst, want[0]) and torch.equal(scale, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.ResidualRmsNormQuant(dst, scale, x, g, 1e-6, residual=r)
        ops.ResidualRmsNormQuant(dst, scale, x, g, 1e-6, residual=r)
    for _ in range(3):
        dst.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dst, want[0]) and torch.equal(scale, want[1])


@gpu
def test_empty():
    x = torch.empty(0, 64, dtype=torch.float16, device=DEV)
    ops.ResidualRmsNormQuant(torch.empty(0, 64, dtype=torch.int8, device=DEV), torch.empty(0, device=DEV), x,
                             torch.ones(64, dtype=torch.float16, device=DEV), 1e-6)


@gpu
def test_feeds_the_w8a8_matmul():
    """norm + quantisation -> W8A8 matmul against the product in 64 bits of the codes' values."""
    m, n, out = 48, 512, 256
    x, r, g = inputs(m, n, torch.bfloat16)
    q, scale, _, _ = run(x, r, g, L.DT_I8)
    rng = torch.Generator().manual_seed(5)
    w = torch.randint(-127, 128, (out, n), generator=rng, dtype=torch.int8).to(DEV)
    ws = (0.01 * torch.rand(out, generator=rng)).to(DEV)
    c = torch.empty(m, out, dtype=torch.bfloat16, device=DEV)
    ops.MatmulW8A8(c, q, w, scale, ws)
    # whole numbers first: they add up exactly, also to 0
    want = (q.double() @ w.double().T) * scale.double()[:, None] * ws.double()
    assert torch.all((c.double() - want).abs() <= want.abs() * (2.0 ** -8 + 8 * U))


# ---- refusals: argument checks come before any CUDA work ---------------------------------------------------------
def refuse(status, dst=0x10000, dstT=L.DT_I8, scale=0x20000, total=None, norm=None, src=0x30000, res=None, gamma=0x40000, srcT=L.DT_BF16,
           gT=L.DT_BF16, m=2, n=64, eps=1e-6, lds=0, ldr=0, ldo=0):
    import ctypes as C
    p = L.RmsNormParam(m, n, eps, lds, ldr, ldo, 0)
    v = lambda a: None if a is None else C.c_void_p(a)  # noqa: E731
    rc = L.lib().ascq_residual_rms_norm_quant(v(dst), dstT, v(scale), v(total), v(norm), v(src), v(res), v(gamma), srcT, gT, C.byref(p), None)
    assert rc == status, (rc, L.lib().ascq_last_error())


def test_refusals():
    refuse(L.ERR_INVALID_ARG, dst=None)
    refuse(L.ERR_INVALID_ARG, src=None)
    refuse(L.ERR_INVALID_ARG, gamma=None)
    refuse(L.ERR_INVALID_ARG, scale=None)
    refuse(L.ERR_UNSUPPORTED, srcT=L.DT_I8)
    refuse(L.ERR_UNSUPPORTED, gT=L.DT_F16)
    refuse(L.ERR_UNSUPPORTED, dstT=L.DT_HIF8)
    refuse(L.ERR_INVALID_ARG, eps=0.0)
    refuse(L.ERR_INVALID_ARG, eps=float("nan"))
    refuse(L.ERR_INVALID_ARG, eps=float("inf"))
    refuse(L.ERR_INVALID_ARG, dstT=L.DT_FP8_E4M3, n=48)
    refuse(L.ERR_INVALID_ARG, lds=63)
    refuse(L.ERR_INVALID_ARG, ldr=-1)
    refuse(L.ERR_ALIGNMENT, src=0x30001)
    refuse(L.ERR_ALIGNMENT, scale=0x20002)
    refuse(L.ERR_INVALID_ARG, dst=0x30000)                       # dst on src
    refuse(L.ERR_INVALID_ARG, total=0x30010)                     # residualOut partly on src
    refuse(L.ERR_INVALID_ARG, total=0x30000, ldo=128)            # residualOut on src with another pitch
    refuse(L.ERR_INVALID_ARG, norm=0x30000)                      # normOut on src
    refuse(L.ERR_INVALID_ARG, total=0x50000, norm=0x50080)       # two outputs
    refuse(L.ERR_INVALID_ARG, total=0x40000)                     # residualOut on gamma
    refuse(L.ERR_INVALID_ARG, total=0x30070, lds=128, ldo=128)   # rows of 128 bytes, 256 apart: the last 16 bytes of src's
    refuse(L.ERR_INVALID_ARG, total=0x300F0, lds=128, ldo=128)   # the first 112 of its next row
    refuse(L.ERR_INVALID_ARG, total=0x2FF90, lds=128, ldo=128, m=300)  # begins before src, reaches into it
    refuse(L.ERR_INVALID_ARG, total=0x30080, lds=128, ldo=192)   # another pitch


def test_python_refusals_name_the_reason():
    cpu = torch.zeros(2, 64, dtype=torch.bfloat16)
    g = torch.zeros(64, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.ResidualRmsNormQuant(q, s, cpu, g, 1e-6)
    with pytest.raises(ValueError, match="one element per column"):
        ops.ResidualRmsNormQuant(q, s, cpu, g[:63], 1e-6)
    with pytest.raises(ValueError, match="shape and dtype"):
        ops.ResidualRmsNormQuant(q, s, cpu, g, 1e-6, residual=cpu.float())
    with pytest.raises(ValueError, match="one float per row"):
        ops.ResidualRmsNormQuant(q, s[:1], cpu, g, 1e-6)
