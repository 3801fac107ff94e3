"""ExpertSort, ExpertDispatch, ExpertCombine and ExpertCombineGrad against plain implementations in 64 bits.

Sorting and dispatching copy: exact.  Tolerances of the sums, with u = 2^-24 and s the half step of the output's type: a sum of k
products in fp32, each added with one rounding, is within k u of its terms' absolute sum; the result's own rounding adds s of the value.  A
dot product over h elements has h roundings at most on any of its partial sums' paths: h u of the absolute sum."""
import ctypes as C

import pytest
import torch

from asc_devkit_b200 import _lib as L
from asc_devkit_b200 import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half a step among the subnormals that the values reach


def plain_sort(ids, experts):
    flat = ids.reshape(-1).cpu().long()
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices
    kept = int(valid.sum())
    slot_of_row = torch.full((flat.numel(),), -1, dtype=torch.int32)
    slot_of_row[:kept] = order[:kept].int()
    row_of_slot = torch.full((flat.numel(),), -1, dtype=torch.int32)
    row_of_slot[order[:kept]] = torch.arange(kept, dtype=torch.int32)
    return torch.bincount(flat[valid], minlength=experts), row_of_slot.reshape(ids.shape), slot_of_row


def sort(ids, experts, **kw):
    counts = torch.full((experts,), 77, dtype=torch.int64, device=DEV)
    row_of_slot = torch.full(ids.shape, 77, dtype=torch.int32, device=DEV)
    slot_of_row = torch.full((ids.numel(),), 77, dtype=torch.int32, device=DEV)
    ops.ExpertSort(counts, row_of_slot, ids, slotOfRow=slot_of_row, **kw)
    torch.cuda.synchronize()
    return counts, row_of_slot, slot_of_row


def check_sort(ids, experts):
    got = sort(ids.to(DEV), experts)
    for a, b in zip(got, plain_sort(ids, experts)):
        assert torch.equal(a.cpu(), b)
    return got


def route(t, k, e, seed=0, outside=0.0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + 131 * t + 7 * k + e)
    ids = torch.stack([torch.randperm(max(e, k), generator=g)[:k] for _ in range(t)]) if t else torch.zeros(0, k, dtype=torch.int64)
    if outside:
        drop = torch.rand(ids.shape, generator=g) < outside
        ids = torch.where(drop, torch.tensor([-1, e, -(2 ** 31), 2 ** 31 - 1])[torch.randint(0, 4, ids.shape, generator=g)], ids)
    return ids.to(dtype)


# ---- sort ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t,k,e", [(1, 1, 1), (1, 8, 256), (3, 2, 5), (33, 3, 7), (100, 8, 60), (1021, 4, 64), (257, 6, 1024), (2500, 8, 128), (9001, 8, 256), (129, 8, 9), (4097, 4, 30), (20000, 8, 64)])
def test_sort(t, k, e, dtype):
    check_sort(route(t, k, e, dtype=dtype), e)


@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t,k,e", [(64, 4, 16), (5000, 8, 32)])
def test_sort_with_slots_that_have_no_expert_here(t, k, e, dtype):
    check_sort(route(t, k, e, outside=0.6, dtype=dtype), e)


@gpu
@pytest.mark.parametrize("slots", [1, 31, 4096, 70001])
@pytest.mark.parametrize("value", [0, 4, -1])
def test_sort_with_one_expert_for_all(slots, value):
    check_sort(torch.full((slots, 1), value, dtype=torch.int32), 5)


@gpu
def test_sort_wide_numbers_do_not_wrap():
    ids = torch.tensor([[2 ** 32 + 1, 1, -(2 ** 32) + 2]], dtype=torch.int64)
    check_sort(ids, 3)


@gpu
def test_sort_many_slots():
    g = torch.Generator().manual_seed(3)
    check_sort(torch.randint(-1, 1024, (1 << 20, 2), generator=g, dtype=torch.int32), 1024)


@gpu
def test_sort_of_nothing_and_without_slot_of_row():
    counts = torch.full((9,), 5, dtype=torch.int64, device=DEV)
    ops.ExpertSort(counts, torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, dtype=torch.int64, device=DEV))
    assert (counts == 0).all()
    ids = route(50, 4, 9).to(DEV)
    rows = torch.empty(50, 4, dtype=torch.int32, device=DEV)
    ops.ExpertSort(counts, rows, ids)
    want = plain_sort(ids, 9)
    assert torch.equal(counts.cpu(), want[0]) and torch.equal(rows.cpu(), want[1])


# ---- dispatch -----------------------------------------------------------------------------------------------------
def check_dispatch(src, ids, experts, scale=None, rows=None):
    counts, row_of_slot, _ = sort(ids.to(DEV), experts)
    t, k = ids.shape
    rows = t * k if rows is None else rows
    fill = torch.full((rows, src.shape[1]), 3, device=DEV).to(src.dtype)
    dst = fill.clone()
    ds = torch.full((rows,) + tuple(scale.shape[1:]), 9, device=DEV).to(scale.dtype) if scale is not None else None
    ops.ExpertDispatch(dst, src, row_of_slot, dstScale=ds, srcScale=scale)
    torch.cuda.synchronize()
    want, ws = fill.cpu(), torch.full_like(ds, 9).cpu() if ds is not None else None
    ros, s, sc = row_of_slot.cpu(), src.cpu(), scale.cpu() if scale is not None else None
    for j in range(k):
        at = ((ros[:, j] >= 0) & (ros[:, j] < rows)).nonzero()[:, 0]
        want[ros[at, j].long()] = s[at]
        if sc is not None:
            ws[ros[at, j].long()] = sc[at]
    assert torch.equal(dst.cpu(), want)
    assert ds is None or torch.equal(ds.cpu(), ws)


@gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("t,k,e,h", [(1, 1, 1, 1), (1, 8, 256, 7168), (16, 8, 256, 2048), (33, 3, 7, 77), (5, 40, 64, 130), (700, 4, 16, 1026), (300, 2, 8, 4100)])
def test_dispatch(t, k, e, h, dtype):
    src = torch.randint(0, 100, (t, h), device=DEV).to(dtype)
    check_dispatch(src, route(t, k, e), e, torch.rand(t, device=DEV))


@gpu
def test_dispatch_pitched_rows_block_scales_and_outside_slots():
    src = torch.randint(0, 255, (90, 1024 + 64), device=DEV, dtype=torch.uint8)[:, :1024]
    scales = torch.randint(0, 255, (90, 32), device=DEV, dtype=torch.uint8)
    check_dispatch(src, route(90, 6, 12, outside=0.5), 12, scales)
    check_dispatch(torch.randint(0, 255, (90, 1030), device=DEV, dtype=torch.uint8)[:, 1:1025], route(90, 6, 12, outside=0.5), 12, scales)


@gpu
def test_dispatch_into_fewer_rows_than_the_slots_name():
    """A row number behind dst's last row is skipped, not written."""
    src = torch.randint(0, 100, (40, 512), device=DEV).to(torch.int8)
    check_dispatch(src, route(40, 4, 8), 8, torch.rand(40, device=DEV), rows=100)


# ---- combine and its gradient -----------------------------------------------------------------------------------------
@gpu
def test_dispatch_of_scales_beside_empty_rows():
    ids = route(37, 3, 8, outside=0.2, dtype=torch.int32).to(DEV)
    counts, ros, _ = sort(ids, 8)
    scale, got = torch.rand(37, device=DEV), torch.full((37 * 3,), 5.0, device=DEV)
    ops.ExpertDispatch(torch.zeros(37 * 3, 0, dtype=torch.int8, device=DEV), torch.zeros(37, 0, dtype=torch.int8, device=DEV), ros, dstScale=got, srcScale=scale)
    want = torch.full_like(got, 5.0)
    named = ros >= 0
    want[ros[named].long()] = scale[:, None].expand(37, 3)[named]
    assert torch.equal(got, want)


def test_dispatch_rows_whose_span_would_not_fit_64_bits():
    st = L.lib().ascq_expert_dispatch(P(0x100000), P(0x200000), 1 << 34, 0, None, None, 0, P(0x300000), 4, 2, (1 << 31) - 1, None)
    assert st == L.ERR_INVALID_ARG
    assert b"2^32" in L.lib().ascq_last_error()


def experts_case(t, k, e, h, dt, outside=0.0, seed=0):
    g = torch.Generator().manual_seed(seed + t + h)
    ids = route(t, k, e, outside=outside)
    _, ros, _ = sort(ids.to(DEV), e)
    w = torch.softmax(torch.randn(t, k, generator=g), -1).to(DEV)
    rows = torch.randn(t * k, h, generator=g).to(dt).to(DEV)
    d_out = (0.1 * torch.randn(t, h, generator=g)).to(dt).to(DEV)
    return ros, w, rows, d_out


def plain_combine(rows, ros, w):
    """(sum, sum of absolute terms) in 64 bits."""
    t, k = ros.shape
    out = torch.zeros(t, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    rows, ros = rows.double().cpu(), ros.cpu()
    w = w.double().cpu() if w is not None else torch.ones(t, k, dtype=torch.float64)
    for j in range(k):
        at = ((ros[:, j] >= 0) & (ros[:, j] < rows.shape[0])).nonzero()[:, 0]
        term = w[at, j, None] * rows[ros[at, j].long()]
        out[at] += term
        mag[at] += term.abs()
    return out, mag


SHAPES = [(1, 1, 1, 1), (50, 4, 8, 2046), (9, 3, 5, 34), (1, 8, 256, 7168), (16, 8, 64, 2048), (33, 3, 7, 77), (6, 40, 64, 264), (500, 4, 16, 1032), (130, 9, 20, 4104), (20, 2, 4, 9000)]


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("outside", [0.0, 0.7])
@pytest.mark.parametrize("t,k,e,h", SHAPES)
def test_combine(t, k, e, h, outside, dt):
    ros, w, rows, _ = experts_case(t, k, e, h, dt, outside)
    for weights in (w, None):
        out = torch.full((t, h), 5.0, dtype=dt, device=DEV)
        ops.ExpertCombine(out, rows, ros, weights)
        want, mag = plain_combine(rows, ros, weights)
        tol = mag * k * U * (1 + HALF_STEP[dt]) + want.abs() * HALF_STEP[dt] + TINY[dt]
        assert torch.all((out.cpu().double() - want).abs() <= tol)


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("outside", [0.0, 0.7])
@pytest.mark.parametrize("t,k,e,h", SHAPES)
def test_combine_grad(t, k, e, h, outside, dt):
    ros, w, rows, d_out = experts_case(t, k, e, h, dt, outside)
    d_rows, d_w = torch.full_like(rows, 5.0), torch.full((t, k), 5.0, device=DEV)
    ops.ExpertCombineGrad(d_rows, d_w, d_out, rows, ros, w)
    torch.cuda.synchronize()
    want = torch.full(rows.shape, 5.0, dtype=torch.float64)
    want_w, mag_w = torch.zeros(t, k, dtype=torch.float64), torch.zeros(t, k, dtype=torch.float64)
    r, c, d, wh = ros.cpu(), rows.double().cpu(), d_out.double().cpu(), w.double().cpu()
    for j in range(k):
        at = (r[:, j] >= 0).nonzero()[:, 0]
        row = r[at, j].long()
        want[row] = wh[at, j, None] * d[at]
        want_w[at, j] = (c[row] * d[at]).sum(-1)
        mag_w[at, j] = (c[row] * d[at]).abs().sum(-1)
    assert torch.all((d_rows.cpu().double() - want).abs() <= want.abs() * (HALF_STEP[dt] + 2 * U) + TINY[dt])
    assert torch.all((d_w.cpu().double() - want_w).abs() <= mag_w * (h + 2) * U)
    # each output alone gives the same bits; without weights they count as 1
    only_rows, only_w = torch.full_like(rows, 5.0), torch.full((t, k), 5.0, device=DEV)
    ops.ExpertCombineGrad(only_rows, None, d_out, rows, ros, w)
    ops.ExpertCombineGrad(None, only_w, d_out, rows, ros, w)
    assert torch.equal(only_rows, d_rows) and torch.equal(only_w, d_w)
    ops.ExpertCombineGrad(only_rows, None, d_out, rows, ros)
    ones = torch.full_like(rows, 5.0)
    ops.ExpertCombineGrad(ones, None, d_out, rows, ros, torch.ones_like(w))
    assert torch.equal(only_rows, ones)


@gpu
def test_gradients_against_differences():
    """A central difference of the combined sum (linear in the rows and in the weights, so exact up to fp32 rounding): with
    step d, values of at most m and sums of n terms, n m u / d on each side."""
    t, k, e, h = 5, 3, 6, 40
    ros, w, rows, d_out = experts_case(t, k, e, h, torch.float32, outside=0.3)
    d_rows, d_w = torch.zeros_like(rows), torch.zeros(t, k, device=DEV)
    ops.ExpertCombineGrad(d_rows, d_w, d_out, rows, ros, w)

    def loss(rows, w):
        out = torch.empty(t, h, device=DEV)
        ops.ExpertCombine(out, rows, ros, w)
        return float((out.double() * d_out.double()).sum())

    step = 0.5
    bound = 2 * (k + 1) * U / step * float((rows.abs().max() + step) * w.max() * d_out.abs().double().sum())
    for i, c in [(0, 0), (3, 17), (7, 39), (14, 5)]:
        up, down = rows.clone(), rows.clone()
        up[i, c] += step
        down[i, c] -= step
        assert abs((loss(up, w) - loss(down, w)) / (2 * step) - float(d_rows[i, c])) <= bound
    bound = 2 * (k + h) * U / step * float(rows.abs().max() * (w.max() + step) * d_out.abs().double().sum())
    for i in range(t):
        for j in range(k):
            up, down = w.clone(), w.clone()
            up[i, j] += step
            down[i, j] -= step
            assert abs((loss(rows, up) - loss(rows, down)) / (2 * step) - float(d_w[i, j])) <= bound


@gpu
def test_nothing_of_a_dropped_slot_reaches_the_result():
    """NaN in the weight of a slot without a row, and in rows that no slot names."""
    ros, w, rows, d_out = experts_case(40, 4, 8, 256, torch.bfloat16, outside=0.5)
    kept = int((ros >= 0).sum())
    out, d_w = torch.empty(40, 256, dtype=torch.bfloat16, device=DEV), torch.empty(40, 4, device=DEV)
    ops.ExpertCombine(out, rows, ros, w)
    rows2, w2 = rows.clone(), torch.where(ros >= 0, w, float("nan"))
    rows2[kept:] = float("nan")
    out2 = torch.empty_like(out)
    ops.ExpertCombine(out2, rows2, ros, w2)
    assert torch.equal(out, out2)
    ops.ExpertCombineGrad(None, d_w, d_out, rows2, ros, w2)
    assert torch.isfinite(d_w).all() and (d_w[ros < 0] == 0).all()
    none = torch.full_like(ros, -1)
    ops.ExpertCombine(out, rows2, none, w2)
    assert (out == 0).all()


@gpu
def test_dispatch_then_combine_is_the_gradient_of_dispatch():
    """<dispatch(x), g> = <x, combine(g)> in integers that fp32 holds exactly."""
    t, k, e, h = 37, 4, 9, 128
    ros, _, _, _ = experts_case(t, k, e, h, torch.float32, outside=0.4)
    x = torch.randint(-8, 9, (t, h), device=DEV).float()
    g = torch.randint(-8, 9, (t * k, h), device=DEV).float()
    rows, dx = torch.zeros(t * k, h, device=DEV), torch.empty(t, h, device=DEV)
    ops.ExpertDispatch(rows, x, ros)
    ops.ExpertCombine(dx, g, ros)
    assert float((rows.double() * g.double()).sum()) == float((x.double() * dx.double()).sum())


@gpu
def test_layer_from_residual_stream_to_combined_experts():
    """The operators as a serving loop uses them: norm + int8, sort, dispatch, grouped W8A8 matmul, combine; against the same
    steps in 64 bits on the quantised values."""
    t, k, e, h, n = 60, 4, 12, 256, 128
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(t, h, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    gamma = torch.ones(h, dtype=torch.bfloat16, device=DEV)
    q, s = torch.empty(t, h, dtype=torch.int8, device=DEV), torch.empty(t, device=DEV)
    ops.ResidualRmsNormQuant(q, s, x, gamma, 1e-6, residual=r, residualOut=r)
    ids = route(t, k, e, outside=0.3)
    counts, ros, _ = sort(ids.to(DEV), e)
    groups = counts.tolist()
    rows, rs = torch.empty(sum(groups), h, dtype=torch.int8, device=DEV), torch.empty(sum(groups), device=DEV)
    ops.ExpertDispatch(rows, q, ros, dstScale=rs, srcScale=s)
    w8 = torch.randint(-127, 128, (e, n, h), generator=g, dtype=torch.int8).to(DEV)
    ws = (0.001 * torch.rand(e, n, generator=g)).to(DEV)
    y = torch.empty(sum(groups), n, dtype=torch.bfloat16, device=DEV)
    ops.GroupMatmulW8A8(y, rows, w8, rs, ws, groups)
    weights = torch.softmax(torch.randn(t, k, generator=g), -1).to(DEV)
    out = torch.empty(t, n, dtype=torch.bfloat16, device=DEV)
    ops.ExpertCombine(out, y, ros, weights)
    ops.MatmulStatus()
    xq = q.double().cpu() * s.double().cpu()[:, None]
    want, mag = torch.zeros(t, n, dtype=torch.float64), torch.zeros(t, n, dtype=torch.float64)
    for i in range(t):
        for j in range(k):
            a = int(ids[i, j])
            if 0 <= a < e:
                v = float(weights[i, j]) * ((w8[a].double().cpu() * ws[a].double().cpu()[:, None]) @ xq[i])
                want[i] += v
                mag[i] += v.abs()
    # the grouped matmul's bf16 result is off by 2^-8 of each term, the sum by k u, its own rounding by 2^-8
    assert torch.all((out.double().cpu() - want).abs() <= mag * (2.0 ** -8 + (k + 4) * U) + (want.abs() + mag * 2.0 ** -8) * 2.0 ** -8)


@gpu
def test_capture_replay_and_other_stream():
    ids = route(200, 4, 16, outside=0.2).to(DEV)
    want = [v.clone() for v in sort(ids, 16)]
    x = torch.randint(-100, 100, (200, 512), device=DEV).to(torch.int8)
    counts, ros, sor = (torch.zeros_like(v) for v in want)
    rows = torch.zeros(800, 512, dtype=torch.int8, device=DEV)
    ref = torch.zeros_like(rows)
    ops.ExpertDispatch(ref, x, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.ExpertSort(counts, ros, ids, slotOfRow=sor)
        ops.ExpertDispatch(rows, x, ros)
    for _ in range(2):
        ros.fill_(-1)
        rows.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ros, want[1]) and torch.equal(counts, want[0]) and torch.equal(rows, ref)
    s = torch.cuda.Stream()
    rows.zero_()
    s.wait_stream(torch.cuda.current_stream())
    ops.ExpertSort(counts, ros, ids, slotOfRow=sor, stream=s)
    ops.ExpertDispatch(rows, x, ros, stream=s)
    s.synchronize()
    assert torch.equal(sor, want[2]) and torch.equal(rows, ref)


@gpu
def test_empty_calls():
    f = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    none = torch.empty(0, 2, dtype=torch.int32, device=DEV)
    ops.ExpertDispatch(f(0, 8), f(0, 8), none)
    ops.ExpertCombine(f(0, 8), f(0, 8), none)
    ops.ExpertCombineGrad(f(0, 8), f(0, 2), f(0, 8), f(0, 8), none)
    out, ros = torch.full((3, 8), 4.0, device=DEV), torch.full((3, 2), 5, dtype=torch.int32, device=DEV)
    ops.ExpertCombine(out, f(0, 8), ros)     # no rows: nothing to add up
    assert (out == 0).all()


# ---- refusals ---------------------------------------------------------------------------------------------------------
P = lambda a: None if a is None else C.c_void_p(a)  # noqa: E731


def test_sort_refusals():
    def call(counts=0x1000, ros=0x20000, sor=None, ids=0x40000, idt=L.DT_I32, slots=8, e=4):
        return L.lib().ascq_expert_sort(P(counts), P(ros), P(sor), P(ids), idt, slots, e, None)
    assert call(idt=L.DT_F32) == L.ERR_UNSUPPORTED
    assert call(e=0) == L.ERR_INVALID_ARG
    assert call(e=1025) == L.ERR_INVALID_ARG
    assert call(slots=-1) == L.ERR_INVALID_ARG
    assert call(slots=1 << 31) == L.ERR_INVALID_ARG
    assert call(counts=None) == L.ERR_INVALID_ARG
    assert call(ros=None) == L.ERR_INVALID_ARG
    assert call(ids=None) == L.ERR_INVALID_ARG
    assert call(counts=0x1004) == L.ERR_ALIGNMENT
    assert call(ids=0x40004, idt=L.DT_I64) == L.ERR_ALIGNMENT
    assert call(ros=0x20002) == L.ERR_ALIGNMENT
    assert call(ros=0x40000) == L.ERR_INVALID_ARG
    assert call(sor=0x20010) == L.ERR_INVALID_ARG


def test_dispatch_refusals():
    def call(dst=0x100000, src=0x200000, width=64, ld=0, ds=None, ss=None, sb=0, ros=0x300000, t=4, k=2, rows=8):
        return L.lib().ascq_expert_dispatch(P(dst), P(src), width, ld, P(ds), P(ss), sb, P(ros), t, k, rows, None)
    assert call(k=0) == L.ERR_INVALID_ARG
    assert call(t=-1) == L.ERR_INVALID_ARG
    assert call(rows=-1) == L.ERR_INVALID_ARG
    assert call(t=1 << 30, k=2) == L.ERR_INVALID_ARG
    assert call(ld=63) == L.ERR_INVALID_ARG
    assert call(ds=0x400000) == L.ERR_INVALID_ARG
    assert call(ds=0x400000, ss=0x500000) == L.ERR_INVALID_ARG
    assert call(dst=None) == L.ERR_INVALID_ARG
    assert call(src=None) == L.ERR_INVALID_ARG
    assert call(ros=None) == L.ERR_INVALID_ARG
    assert call(ros=0x300002) == L.ERR_ALIGNMENT
    assert call(dst=0x200010) == L.ERR_INVALID_ARG
    assert call(ds=0x500000, ss=0x500000, sb=4) == L.ERR_INVALID_ARG
    assert call(width=1 << 41) == L.ERR_INVALID_ARG


def test_combine_refusals():
    def call(dst=0x100000, rows=0x200000, dt=L.DT_BF16, ros=0x300000, w=0x400000, t=4, k=2, r=8, h=64):
        return L.lib().ascq_expert_combine(P(dst), P(rows), dt, P(ros), P(w), t, k, r, h, None)
    assert call(dt=L.DT_I8) == L.ERR_UNSUPPORTED
    assert call(k=0) == L.ERR_INVALID_ARG
    assert call(h=-1) == L.ERR_INVALID_ARG
    assert call(dst=None) == L.ERR_INVALID_ARG
    assert call(rows=None) == L.ERR_INVALID_ARG
    assert call(dst=0x100001) == L.ERR_ALIGNMENT
    assert call(w=0x400002) == L.ERR_ALIGNMENT
    assert call(dst=0x200000) == L.ERR_INVALID_ARG
    assert call(dst=0x400000) == L.ERR_INVALID_ARG


def test_combine_grad_refusals():
    def call(dr=0x100000, dw=0x200000, do=0x300000, rows=0x400000, dt=L.DT_F16, ros=0x500000, w=0x600000, t=4, k=2, r=8, h=64):
        return L.lib().ascq_expert_combine_grad(P(dr), P(dw), P(do), P(rows), dt, P(ros), P(w), t, k, r, h, None)
    assert call(dr=None, dw=None) == L.ERR_INVALID_ARG
    assert call(dt=L.DT_I32) == L.ERR_UNSUPPORTED
    assert call(do=None) == L.ERR_INVALID_ARG
    assert call(rows=None) == L.ERR_INVALID_ARG
    assert call(dr=0x400000) == L.ERR_INVALID_ARG
    assert call(dw=0x600000) == L.ERR_INVALID_ARG
    assert call(dr=0x300000) == L.ERR_INVALID_ARG
    assert call(dw=0x200001) == L.ERR_ALIGNMENT


def test_combine_grad_of_empty_rows_is_no_error():
    """Rows of no elements: nothing to write, and torch gives such tensors no address.  (No CUDA work: this runs without a GPU.)"""
    grad = L.lib().ascq_expert_combine_grad
    assert grad(None, None, None, None, L.DT_F16, P(0x500000), P(0x600000), 4, 2, 8, 0, None) == L.OK
    assert grad(None, None, None, None, L.DT_F16, P(0x500000), P(0x600000), 4, 2, 0, 64, None) == L.OK


def test_python_refusals():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.ExpertSort(torch.zeros(4, dtype=torch.int64), i32(3, 2), torch.zeros(3, 2))
    with pytest.raises(ValueError, match="one element per slot"):
        ops.ExpertSort(torch.zeros(4, dtype=torch.int64), i32(3), i32(3, 2))
    with pytest.raises(ValueError, match="rowOfSlot"):
        ops.ExpertDispatch(torch.zeros(6, 8), torch.zeros(3, 8), i32(2, 2))
    with pytest.raises(ValueError, match="go together"):
        ops.ExpertDispatch(torch.zeros(6, 8), torch.zeros(3, 8), i32(3, 2), srcScale=torch.zeros(3))
    with pytest.raises(ValueError, match="weights"):
        ops.ExpertCombine(torch.zeros(3, 8), torch.zeros(6, 8), i32(3, 2), torch.zeros(3, 2).half())
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.ExpertCombine(torch.zeros(3, 8), torch.zeros(6, 8), i32(3, 2))
    with pytest.raises(ValueError, match="gradRows"):
        ops.ExpertCombineGrad(torch.zeros(5, 8), None, torch.zeros(3, 8), torch.zeros(6, 8), i32(3, 2))
