"""LowRankAdd against its formula in 64 bits.

Tolerance, with u = 2^-24 and s the half step of the output's type.  The inner product of K terms and the second one of r terms run in the
tensor cores' fp32 accumulators, which may truncate where fp32 arithmetic rounds: at most 2 u of the terms' absolute sum
per addition.  The inner product enters the second as two 16-bit values: what they leave out is s^2 of it, and no more than
2^-35 of the row's largest where fp16's subnormals end.  The scale and the addition of base add a few u, the result's rounding s of it."""
import ctypes as C

import pytest
import torch

from asc_devkit_b200 import _lib as L
from asc_devkit_b200 import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def case(m, n, k, r, lo, dt, span=1, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed + 7 * m + n + 3 * k + r + lo)
    x = torch.randn(m, k, generator=g).to(dt)
    base = torch.randn(m, n, generator=g).to(dt)
    a = (torch.randn(lo, r, k, generator=g) * k ** -0.5).to(dt)
    b = (torch.randn(lo, n, r, generator=g) * r ** -0.5).to(dt)
    scale = 0.5 + torch.rand(lo, generator=g)
    if ids is None:
        ids = torch.randint(-1, lo, (-(-m // span),), generator=g).repeat_interleave(span)[:m]
    return [t.to(DEV) for t in (x, base, a, b, scale, ids.to(torch.int32))]


def check(got, x, base, a, b, scale, ids):
    dt, k, r = x.dtype, x.shape[1], a.shape[1]
    want = base.double() if base is not None else torch.zeros(got.shape, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(want)
    for e in range(a.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if not len(at):
            continue
        s = float(scale[e]) if scale is not None else 1.0
        xa, aa, ba = x[at].double(), a[e].double(), b[e].double()
        inner, mag = xa @ aa.T, xa.abs() @ aa.abs().T
        want[at] += s * (inner @ ba.T)
        off = mag * (2 * (k + 2 * r + 8) * U) + inner.abs() * HALF_STEP[dt] ** 2 + inner.abs().amax(-1, keepdim=True) * 2.0 ** -35
        tol[at] += abs(s) * (off @ ba.abs().T)
    tol += (want.abs() + tol) * (HALF_STEP[dt] + 4 * U) + (2.0 ** -25 if dt == torch.float16 else 0.0)  # half a step among fp16's subnormals
    none = (ids < 0) | (ids >= a.shape[0])
    if base is not None:
        assert torch.equal(got[none], base[none])
    else:
        assert (got[none] == 0).all()
    worst = ((got.double() - want).abs() - tol).max() if got.numel() else 0
    assert worst <= 0, f"{float(worst)} beyond the bound"


SHAPES = [  # m, n, k, r, adapters, tokens of a request
    (1, 8, 8, 8, 1, 1), (1, 4096, 4096, 16, 16, 1), (32, 4096, 4096, 16, 16, 1), (5, 264, 520, 8, 3, 1), (17, 1000, 72, 24, 2, 1), (16, 96, 2048, 40, 40, 1),
    (64, 512, 1024, 64, 64, 1), (200, 2048, 512, 128, 5, 33), (1024, 256, 512, 16, 1000, 1), (1025, 256, 512, 32, 1023, 1), (1337, 640, 1376, 32, 8, 97),
    (2500, 264, 136, 64, 3, 700), (3000, 520, 1032, 104, 7, 1), (1100, 4096, 256, 128, 4, 300), (4096, 1024, 1024, 64, 16, 256),
    # tiles of 128 tokens: more than 20 million of m (n + k), a third of that for ranks above 64
    (1700, 4104, 8200, 16, 3, 1), (2500, 8200, 72, 32, 5, 130), (4700, 4096, 264, 64, 16, 300), (1400, 200, 5000, 128, 2, 1030), (700, 5000, 5000, 104, 2, 7), (8000, 8, 2760, 8, 20, 1),
    (2600, 8000, 8, 24, 1, 2100), (3500, 3000, 3000, 48, 4, 129), (1500, 8200, 6000, 40, 8, 1500)]


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,r,lo,span", SHAPES)
def test_against_the_formula(m, n, k, r, lo, span, dt):
    x, base, a, b, scale, ids = case(m, n, k, r, lo, dt, span)
    for bs, sc, i in ((base, scale, ids), (None, None, ids.long())):
        got = torch.full((m, n), 3.0, dtype=dt, device=DEV)
        ops.LowRankAdd(got, bs, x, a, b, i, scale=sc)
        check(got, x, bs, a, b, sc, ids)


@gpu
@pytest.mark.parametrize("m,n", [(1, 136), (16, 136), (40, 136), (1500, 136), (1500, 14000)])
def test_one_adapter_or_none_for_all(m, n):
    for value in (0, 2, -1, 3, 2 ** 31 - 1):
        x, base, a, b, scale, ids = case(m, n, 264, 16, 3, torch.bfloat16, ids=torch.full((m,), value))
        got = torch.empty_like(base)
        ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
        check(got, x, base, a, b, scale, ids)


@gpu
@pytest.mark.parametrize("m", [48, 1200, 27000])
def test_in_place_pitched_rows_and_repeated_calls(m):
    x, base, a, b, scale, ids = case(m, 256, 512, 32, 6, torch.float16)
    want = torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    wide = torch.full((m, 256 + 24), 5.0, dtype=torch.float16, device=DEV)
    wide[:, 8:264] = base
    xw = torch.full((m, 512 + 16), 9.0, dtype=torch.float16, device=DEV)
    xw[:, 16:] = x
    ops.LowRankAdd(wide[:, 8:264], wide[:, 8:264], xw[:, 16:], a, b, ids, scale=scale)
    assert torch.equal(wide[:, 8:264], want) and (wide[:, :8] == 5).all() and (wide[:, 264:] == 5).all()
    for _ in range(3):
        again = torch.empty_like(base)
        ops.LowRankAdd(again, base, x, a, b, ids, scale=scale)
        assert torch.equal(again, want)


@gpu
@pytest.mark.parametrize("m", [33, 3000])
def test_slices_of_one_buffer(m):
    """x, base and dst as column slices of one matrix."""
    n, k = 1024, 6144
    x, base, a, b, scale, ids = case(m, n, k, 16, 3, torch.bfloat16)
    want = torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    wide = torch.zeros(m, k + 2 * n + 8, dtype=torch.bfloat16, device=DEV)
    xs, bs, ds = wide[:, :k], wide[:, k:k + n], wide[:, k + n:k + 2 * n]
    xs.copy_(x)
    bs.copy_(base)
    ops.LowRankAdd(ds, bs, xs, a, b, ids, scale=scale)
    assert torch.equal(ds, want) and torch.equal(xs, x) and torch.equal(bs, base) and (wide[:, -8:] == 0).all()


@gpu
@pytest.mark.parametrize("m,n", [(40, 128), (1200, 20000)])
def test_large_and_small_inner_products(m, n):
    """Inner products beyond fp16's range and among its subnormals: the second product brings them back."""
    x, base, a, b, scale, ids = case(m, n, 256, 16, 2, torch.float16, ids=torch.zeros(m))
    for fx, fb in ((2000.0, 2.0 ** -14), (2.0 ** -14, 1000.0)):
        xs, bs = (x.float() * fx).to(torch.float16), (b.float() * fb).to(torch.float16)
        got = torch.empty_like(base)
        ops.LowRankAdd(got, None, xs, a, bs, ids, scale=scale)
        check(got, xs, None, a, bs, scale, ids)


@gpu
@pytest.mark.parametrize("m,n", [(40, 128), (1200, 20000)])
@pytest.mark.parametrize("ex,eb", [(-7, 119), (-100, 122), (-100, 100), (-60, 20), (100, -100), (119, -122), (110, 10)])
def test_bfloat16_over_its_whole_range(m, n, ex, eb):
    """Inner products near 2^ex, B near 2^eb: their products are in range, so is every step towards them."""
    x, base, a, b, scale, ids = case(m, n, 256, 16, 2, torch.bfloat16, ids=torch.zeros(m))
    xs, bs = (x.double() * 2.0 ** ex).to(torch.bfloat16), (b.double() * 2.0 ** eb).to(torch.bfloat16)
    for own in (base, None):
        got = torch.empty_like(base)
        ops.LowRankAdd(got, own, xs, a, bs, ids, scale=scale)
        assert torch.isfinite(got).all()
        check(got, xs, own, a, bs, scale, ids)


@gpu
@pytest.mark.parametrize("m,n", [(20, 64), (1300, 16384)])
def test_bfloat16_inner_product_next_to_the_end_of_fp32(m, n):
    """1.9921875 * 2^127 * 1.003 lies between bfloat16's largest value and fp32's."""
    x = torch.zeros(m, 64, dtype=torch.bfloat16, device=DEV)
    x[:, 3] = 2.0 ** 64
    a = torch.zeros(1, 16, 64, dtype=torch.bfloat16, device=DEV)
    a[0, 5, 3] = 1.9921875 * 2.0 ** 63
    b = torch.full((1, n, 16), 2.0 ** -20, dtype=torch.bfloat16, device=DEV)
    scale = torch.tensor([1.003], device=DEV)
    got = torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(m, dtype=torch.int32, device=DEV)
    ops.LowRankAdd(got, None, x, a, b, ids, scale=scale)
    check(got, x, None, a, b, scale, ids)


@gpu
@pytest.mark.parametrize("m,n", [(60, 64), (1300, 16384)])
def test_values_that_are_not_finite_stay_in_their_token(m, n):
    x, base, a, b, scale, ids = case(m, n, 128, 16, 3, torch.bfloat16)
    want = torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    t = int((ids >= 0).nonzero()[3])
    x2 = x.clone()
    x2[t, 5] = float("nan")
    got = torch.empty_like(base)
    ops.LowRankAdd(got, base, x2, a, b, ids, scale=scale)
    rest = torch.arange(m, device=DEV) != t
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[t]).all()
    # NaN in the input of a token without an adapter, and in an adapter that no token uses
    none = int((ids < 0).nonzero()[0])
    x2 = x.clone()
    x2[none] = float("nan")
    ops.LowRankAdd(got, base, x2, a, b, ids, scale=scale)
    assert torch.equal(got, want)
    a2, b2 = torch.cat([a, torch.full_like(a[:1], float("nan"))]), torch.cat([b, torch.full_like(b[:1], float("nan"))])
    ops.LowRankAdd(got, base, x, a2, b2, ids, scale=torch.cat([scale, scale[:1]]))
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("m,n", [(20, 64), (1300, 16384)])
def test_infinite_inner_product_beside_large_finite_ones(m, n):
    x = torch.zeros(m, 64, dtype=torch.float16, device=DEV)
    x[:, :2], x[:, 5] = 30000.0, 1.0
    a = torch.zeros(1, 16, 64, dtype=torch.float16, device=DEV)
    a[0, 0, 5] = float("inf")
    a[0, 1, :2] = -60000.0  # an inner product of -3.6e9
    b = torch.ones(1, n, 16, dtype=torch.float16, device=DEV)
    got = torch.zeros(m, n, dtype=torch.float16, device=DEV)
    ops.LowRankAdd(got, None, x, a, b, torch.zeros(m, dtype=torch.int32, device=DEV))
    assert (got == float("inf")).all()


@gpu
@pytest.mark.parametrize("m,n,k", [(40, 136, 264), (2000, 8200, 3000)])
def test_ranks_beyond_one_call(m, n, k):
    """As the header says: a rank of 4 padded with zeros, one of 256 in two calls (each of which rounds its result)."""
    x, base, a, b, scale, ids = case(m, n, k, 256, 3, torch.float16)
    four, padded = (a[:, :4].contiguous(), b[:, :, :4].contiguous()), (torch.zeros_like(a[:, :8]), torch.zeros_like(b[:, :, :8]))
    padded[0][:, :4], padded[1][:, :, :4] = four
    got = torch.empty_like(base)
    ops.LowRankAdd(got, base, x, padded[0].contiguous(), padded[1].contiguous(), ids, scale=scale)
    check(got, x, base, *four, scale, ids)
    first = torch.empty_like(base)
    ops.LowRankAdd(first, base, x, a[:, :128].contiguous(), b[:, :, :128].contiguous(), ids, scale=scale)
    check(first, x, base, a[:, :128], b[:, :, :128], scale, ids)
    got.copy_(first)
    ops.LowRankAdd(got, got, x, a[:, 128:].contiguous(), b[:, :, 128:].contiguous(), ids, scale=scale)
    check(got, x, first, a[:, 128:], b[:, :, 128:], scale, ids)


@gpu
def test_result_that_overflows_saturates():
    x = torch.full((2, 8), 100.0, dtype=torch.float16, device=DEV)
    a, b = torch.full((1, 8, 8), 10.0, dtype=torch.float16, device=DEV), torch.full((1, 8, 8), 10.0, dtype=torch.float16, device=DEV)
    got = torch.empty(2, 8, dtype=torch.float16, device=DEV)
    ops.LowRankAdd(got, None, x, a, b, torch.tensor([0, -1], dtype=torch.int32, device=DEV))
    assert (got[0] == 65504).all() and (got[1] == 0).all()


@gpu
@pytest.mark.parametrize("m", [64, 1100, 27000])
def test_other_stream_and_capture(m):
    x, base, a, b, scale, ids = case(m, 256, 512, 16, 8, torch.bfloat16)
    want = torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    s = torch.cuda.Stream()
    got = torch.zeros_like(base)
    s.wait_stream(torch.cuda.current_stream())
    ops.LowRankAdd(got, base, x, a, b, ids, scale=scale, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
        ops.LowRankAdd(got, got, x, a, b, ids, scale=scale)
    twice = torch.empty_like(base)
    ops.LowRankAdd(twice, want, x, a, b, ids, scale=scale)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, twice)


@gpu
@pytest.mark.parametrize("m,n,k", [(24, 512, 1024), (3100, 4096, 2560)])
def test_beside_the_w8a8_projection(m, n, k):
    """A projection with adapters, for a decode step and for prompts: int8 matmul, then the adapters on its result in place; the
    launches of several layers follow each other without a wait."""
    r, lo = 16, 5
    x, _, a, b, scale, ids = case(m, n, k, r, lo, torch.bfloat16)
    g = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    q, qs, y = torch.empty(m, k, dtype=torch.int8, device=DEV), torch.empty(m, device=DEV), torch.empty_like(x)
    ops.ResidualRmsNormQuant(q, qs, x, g, 1e-6, normOut=y)
    rng = torch.Generator().manual_seed(5)
    w = torch.randint(-127, 128, (n, k), generator=rng, dtype=torch.int8).to(DEV)
    ws = (0.001 * torch.rand(n, generator=rng)).to(DEV)
    c = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    ops.MatmulW8A8(c, q, w, qs, ws)
    base = c.clone()
    ops.LowRankAdd(c, c, y, a, b, ids, scale=scale)
    check(c, y, base, a, b, scale, ids)
    layers = [torch.empty_like(c) for _ in range(6)]
    for t in layers:
        ops.MatmulW8A8(t, q, w, qs, ws)
        ops.LowRankAdd(t, t, y, a, b, ids, scale=scale)
    ops.MatmulStatus()
    assert all(torch.equal(t, c) for t in layers)


@gpu
def test_two_calls_at_once_on_two_streams():
    """Each call has its own workspace: two long ones and two short ones in flight together."""
    big = case(3000, 4096, 3000, 32, 4, torch.float16, span=200)
    small = case(100, 512, 1024, 16, 8, torch.float16)
    want = []
    for x, base, a, b, scale, ids in (big, small):
        want.append(torch.empty_like(base))
        ops.LowRankAdd(want[-1], base, x, a, b, ids, scale=scale)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.zeros_like(w) for w in want] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, outs in zip(streams, got):
            for out, (x, base, a, b, scale, ids) in zip(outs, (big, small)):
                ops.LowRankAdd(out, base, x, a, b, ids, scale=scale, stream=s)
    torch.cuda.synchronize()
    for outs in got:
        for out, w in zip(outs, want):
            assert torch.equal(out, w)


@gpu
@pytest.mark.parametrize("size", [4096, 3 << 20, 40 << 20])
def test_workspaces_of_two_streams_are_never_the_same_block(size):
    """What one stream's call gave back may still be read by its kernels: a call on another stream must not get it, in either
    direction.  (Nothing runs here: only the addresses count.)"""
    dev, other = torch.device(DEV), torch.cuda.Stream()
    mine = ops._workspace(size, dev, None)
    at = mine.data_ptr()
    del mine
    theirs = ops._workspace(size, dev, other)
    assert theirs.data_ptr() != at
    back = theirs.data_ptr()
    del theirs
    mine = ops._workspace(size, dev, None)
    assert mine.data_ptr() != back
    del mine
    assert ops._workspace(size, dev, other).data_ptr() == back  # the same stream's next call may have it


@gpu
@pytest.mark.parametrize("m,n,k", [(1500, 256, 512), (3000, 4096, 3000)])
def test_a_call_on_another_stream_takes_its_own_workspace(m, n, k, monkeypatch):
    """The public call's workspace: taken while `stream` is torch's current stream."""
    x, base, a, b, scale, ids = case(m, n, k, 16, 4, torch.bfloat16)
    want, got, s, seen = torch.empty_like(base), torch.empty_like(base), torch.cuda.Stream(), []
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    s.wait_stream(torch.cuda.current_stream())
    empty = torch.empty

    def note(*args, **kw):
        seen.append(torch.cuda.current_stream())
        return empty(*args, **kw)
    monkeypatch.setattr(torch, "empty", note)
    ops.LowRankAdd(got, base, x, a, b, ids, scale=scale, stream=s)
    monkeypatch.undo()
    s.synchronize()
    assert seen == [s] and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("m,n,k,r,lo,span", [(1700, 4104, 8200, 16, 3, 1), (4700, 4096, 264, 64, 16, 300), (1400, 4096, 5000, 128, 2, 1030), (8192, 4096, 4096, 64, 16, 700)])
@pytest.mark.parametrize("chunks,blocks", [(0, -1), (3, -1), (-1, 0), (-1, 2)])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_exact(m, n, k, r, lo, span, chunks, blocks):
    """Loads of A (first launch) or B (second) that are never made, a wait limit of about ten milliseconds: every role leaves
    its loop, what was issued has ended before shared and tensor memory are given back, and the status names the timeout once."""
    x, base, a, b, scale, ids = case(m, n, k, r, lo, torch.float16, span)
    want, got = torch.empty_like(base), torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    ops.MatmulStatus()
    if chunks > 0 and k < 4096:
        return  # (too few chunks in a CTA for the third to be missed)
    ops.SetWaitLimitCycles(20_000_000)
    try:
        L.check(L.lib().ascq_test_withhold_low_rank(chunks, blocks))
        ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
        with pytest.raises(ops.AscqError) as e:
            ops.MatmulStatus()
        assert e.value.status == L.ERR_TIMEOUT and "low-rank" in e.value.message
    finally:
        ops.SetWaitLimitCycles(0)
    ops.MatmulStatus()  # the status word was cleared
    for _ in range(2):
        got.fill_(3.0)
        ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
        ops.MatmulStatus()
        assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("m,n,k,r,lo,span", [(1700, 4104, 8200, 16, 3, 1), (1400, 4096, 5000, 128, 2, 1030), (8192, 4096, 4096, 64, 16, 700)])
@pytest.mark.parametrize("limit", [1, 3000, 30000])
def test_a_limit_shorter_than_ordinary_waits(m, n, k, r, lo, span, limit):
    """CTAs give up with their own copies and MMAs under way, at any point of their loops; the call after it, with the ordinary limit, is exact."""
    x, base, a, b, scale, ids = case(m, n, k, r, lo, torch.bfloat16, span)
    want, got = torch.empty_like(base), torch.empty_like(base)
    ops.LowRankAdd(want, base, x, a, b, ids, scale=scale)
    ops.MatmulStatus()
    ops.SetWaitLimitCycles(limit)
    try:
        for _ in range(3):
            ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
            try:
                ops.MatmulStatus()
                assert torch.equal(got, want)  # nobody gave up
            except ops.AscqError as e:
                assert e.status == L.ERR_TIMEOUT
    finally:
        ops.SetWaitLimitCycles(0)
    got.fill_(3.0)
    ops.LowRankAdd(got, base, x, a, b, ids, scale=scale)
    ops.MatmulStatus()
    assert torch.equal(got, want)


STATUS_COPIES = """
import torch
from torch.profiler import ProfilerActivity, profile
from asc_devkit_b200 import ops

def copies():
    ops.MatmulStatus()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        for _ in range(5):
            ops.MatmulStatus()
    return sum(e.count for e in p.key_averages() if "Memcpy" in e.key and "DtoH" in e.key.replace(" ", "")) / 5

torch.zeros(1, device="cuda:0")
z = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda:0")
before = copies()
ops.LowRankAdd(z(4, 16), None, z(4, 8), z(2, 8, 8), z(2, 16, 8), torch.zeros(4, dtype=torch.int32, device="cuda:0"))
few = copies()
ops.LowRankAdd(z(2000, 8192), None, z(2000, 4096), z(2, 16, 4096), z(2, 8192, 16), torch.zeros(2000, dtype=torch.int32, device="cuda:0"))
print("copies", before, few, copies())
"""


@gpu
def test_status_of_a_program_without_adapters_costs_what_it_did():
    """ascq_matmul_status reads the status word of the adapters' kernels (a copy and a wait of its own) only after a call that launched them."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", STATUS_COPIES], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    before, few, after = (float(v) for v in out.stdout.split("copies")[1].split())
    if after == 0:
        pytest.skip("the profiler records no copies here")
    assert before == 3 and few == 3 and after == 4, out.stdout   # int8 / half matmuls, MX matmuls, exchange; then the adapters


@gpu
def test_empty():
    e = lambda *s: torch.empty(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    ops.LowRankAdd(e(0, 16), e(0, 16), e(0, 8), e(2, 8, 8), e(2, 16, 8), torch.empty(0, dtype=torch.int32, device=DEV))


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_refusals():
    P = lambda v: None if v is None else C.c_void_p(v)  # noqa: E731

    def call(dst=0x1000000, ldd=0, base=0x2000000, ldb=0, x=0x3000000, ldx=0, a=0x4000000, b=0x5000000, dt=L.DT_BF16, ids=0x6000000, idt=L.DT_I32, sc=None, m=4,
             n=64, k=64, r=16, lo=3, ws=None, wsb=0):
        return L.lib().ascq_low_rank_add(P(dst), ldd, P(base), ldb, P(x), ldx, P(a), P(b), dt, P(ids), idt, P(sc), m, n, k, r, lo, P(ws), wsb, None)
    assert call(dt=L.DT_F32) == L.ERR_UNSUPPORTED
    assert call(idt=L.DT_I8) == L.ERR_UNSUPPORTED
    for bad in (dict(m=-1), dict(n=-8), dict(k=0), dict(n=60), dict(k=60), dict(r=0), dict(r=12), dict(r=136), dict(lo=0), dict(lo=1024), dict(ldd=56), dict(ldx=8), dict(ldb=8),
                dict(dst=None), dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(dst=0x3000000), dict(dst=0x5000010), dict(dst=0x2000010),
                dict(dst=0x2000000, ldd=72), dict(m=2000), dict(m=2000, ws=0x7000000, wsb=1000), dict(m=2000, ws=0x3000000, wsb=1 << 20)):
        assert call(**bad) == L.ERR_INVALID_ARG, bad
    for bad in (dict(dst=0x1000008), dict(x=0x3000002), dict(ldd=68), dict(ldx=68), dict(ids=0x6000002), dict(ids=0x6000004, idt=L.DT_I64), dict(sc=0x8000001),
                dict(m=2000, ws=0x7000008, wsb=1 << 20)):
        assert call(**bad) == L.ERR_ALIGNMENT, bad
    size = L.lib().ascq_low_rank_add_workspace_size
    assert size(1024, 4096, 4096, 16, 8) == 0
    assert size(2000, 4096, 4096, 16, 1000) == 8016 + 2000 * 4                    # counts and order
    # many tokens of few adapters: tiles (and their number), units and the inner products too
    assert size(2000, 8192, 4096, 64, 3) == 32 + 8000 + (2000 // 128 + 5) * 16 + 8000 + 2000 * 2 * 64 * 2
    assert size(512, 11008, 4096, 128, 3) > 0 and size(512, 11008, 4096, 64, 3) == 0


@pytest.mark.parametrize("n,k", [((1 << 30) + 8, 64), (64, (1 << 30) + 8), ((1 << 31) - 8, (1 << 31) - 8)])
def test_widths_whose_indices_would_wrap(n, k):
    # the second check that such a call meets is the one of dst: NULL here, so that no build launches it
    st = L.lib().ascq_low_rank_add(None, 0, None, 0, None, 0, None, None, L.DT_BF16, None, L.DT_I32, None, 4, n, k, 16, 3, None, 0, None)
    assert st == L.ERR_INVALID_ARG
    assert b"2^30" in L.lib().ascq_last_error()


def test_python_refusals():
    z = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    ids = torch.zeros(4, dtype=torch.int32)
    good = [z(4, 16), z(4, 16), z(4, 8), z(2, 8, 8), z(2, 16, 8), ids]
    for i, bad, text in ((0, z(4, 8), "base and dst"), (1, z(3, 16), "base and dst"), (3, z(2, 8, 16), "A must be"), (4, z(1, 16, 8), "A must be"),
                         (4, z(2, 16, 8).float(), "one dtype"), (5, ids[:3], "adapterIds")):
        args = list(good)
        args[i] = bad
        with pytest.raises(ValueError, match=text):
            ops.LowRankAdd(*args)
    with pytest.raises(ValueError, match="scale"):
        ops.LowRankAdd(*good, scale=torch.zeros(3))
    with pytest.raises(TypeError):
        ops.LowRankAdd(*good[:5], ids.float())
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.LowRankAdd(*good)
