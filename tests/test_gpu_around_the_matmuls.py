"""The operators around the matmuls as a serving loop runs them: norm with MX output, dispatch of rows and their E8M0 scales, grouped MX matmul, combine, the
adapters beside a projection; and each operator's first call of a process made inside a captured graph.

Tolerance of the layer, U = 2^-24: the grouped matmul adds K terms up in fp32 accumulators that may truncate (2 U of the terms' absolute sum per addition) and
rounds to bfloat16 (2^-8); combine adds k terms (U each) and rounds once more."""
import os
import subprocess
import sys

import pytest
import torch

from asc_devkit_b200 import _lib as L
from asc_devkit_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def values(codes, scales, dt):
    """Codes [rows, ...] with their E8M0 scales -> what they stand for, in 64 bits on the host."""
    codes, scales = codes.cpu(), scales.cpu()
    if dt == L.DT_FP4X2_E2M1:
        v = E2M1[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(codes.shape[0], -1)
    else:
        v = codes.view(torch.float8_e4m3fn if dt == L.DT_FP8_E4M3 else torch.float8_e5m2).double()
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


@pytest.mark.parametrize("held", [12, 5])
@pytest.mark.parametrize("dt", [L.DT_FP8_E4M3, L.DT_FP8_E5M2, L.DT_FP4X2_E2M1])
def test_mx_layer_from_residual_stream_to_combined_experts(dt, held):
    t, k, e, h, n = 75, 4, 12, 512, 256
    g = torch.Generator().manual_seed(dt + held)
    x, r = (torch.randn(t, h, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    gamma = (1 + 0.2 * torch.randn(h, generator=g)).to(torch.bfloat16).to(DEV)
    width = h // 2 if dt == L.DT_FP4X2_E2M1 else h
    q, s = torch.empty(t, width, dtype=torch.uint8, device=DEV), torch.empty(t, h // 32, dtype=torch.uint8, device=DEV)
    ops.ResidualRmsNormQuant(q, s, x, gamma, 1e-6, residual=r, residualOut=r, dst_dtype=dt)
    ids = torch.argsort(torch.rand(t, e, generator=g), -1)[:, :k].to(torch.int32).to(DEV)
    counts, ros = torch.empty(held, dtype=torch.int64, device=DEV), torch.empty(t, k, dtype=torch.int32, device=DEV)
    ops.ExpertSort(counts, ros, ids)
    groups = counts.tolist()
    rows, rs = torch.empty(sum(groups), width, dtype=torch.uint8, device=DEV), torch.empty(sum(groups), h // 32, dtype=torch.uint8, device=DEV)
    ops.ExpertDispatch(rows, q, ros, dstScale=rs, srcScale=s)
    # every row and its scales went together
    for slot in range(k):
        at = (ros[:, slot] >= 0).nonzero()[:, 0]
        assert torch.equal(rows[ros[at, slot].long()], q[at]) and torch.equal(rs[ros[at, slot].long()], s[at])
    w = torch.randint(0, 256, (held, n, width), generator=g, dtype=torch.uint8)
    if dt != L.DT_FP4X2_E2M1:
        w &= 0x3F  # finite, at most 1.875
        w |= (torch.randint(0, 2, w.shape, generator=g) * 0x80).to(torch.uint8)
    ws = (127 + torch.randint(-4, 2, (held, n, h // 32), generator=g)).to(torch.uint8)
    w, ws = w.to(DEV), ws.to(DEV)
    y = torch.empty(sum(groups), n, dtype=torch.bfloat16, device=DEV)
    if dt == L.DT_FP4X2_E2M1:
        ops.GroupMatmulMxfp4(y, rows, rs, w, ws, groups, h, n)
    else:
        ops.GroupMatmulMxfp8(y, rows, dt, rs, w, dt, ws, groups, h, n)
    weights = torch.softmax(torch.randn(t, k, generator=g), -1).to(DEV)
    out = torch.empty(t, n, dtype=torch.bfloat16, device=DEV)
    ops.ExpertCombine(out, y, ros, weights)
    ops.MatmulStatus()
    xv, want, mag = values(q, s, dt), torch.zeros(t, n, dtype=torch.float64), torch.zeros(t, n, dtype=torch.float64)
    wv = values(w.reshape(held * n, width), ws.reshape(held * n, h // 32), dt).reshape(held, n, h)
    total = torch.zeros_like(mag)  # of the products' magnitudes
    for i in range(t):
        for j in range(k):
            a = int(ids[i, j])
            if a < held:
                c = float(weights[i, j])
                want[i] += c * (wv[a] @ xv[i])
                mag[i] += c * (wv[a] @ xv[i]).abs()
                total[i] += c * (wv[a].abs() @ xv[i].abs())
    off = total * (2 * h * U) * (1 + 2.0 ** -8) + mag * (2.0 ** -8 + (k + 4) * U)
    assert torch.all((out.double().cpu() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8)


FIRST_CALL = """
import torch
from asc_devkit_b200 import _lib as L
from asc_devkit_b200 import ops
dev = "cuda:0"
g = torch.Generator().manual_seed(3)
r = lambda *s, dt=torch.bfloat16: torch.randn(*s, generator=g).to(dt).to(dev)
what = "{what}"
if what.startswith("norm"):
    n = {{"norm_rows": 1024, "norm_odd": 1023, "norm_any": 20001}}[what]
    x, gamma, dst, scale = r(9, n), r(n), torch.zeros(9, n, dtype=torch.int8, device=dev), torch.zeros(9, device=dev)
    outs = [dst, scale]
    call = lambda: ops.ResidualRmsNormQuant(dst, scale, x, gamma, 1e-6)
elif what.startswith("sort"):
    t = {{"sort_one": 16, "sort_cluster": 9000}}[what]
    ids = torch.randint(-1, 16, (t, 4), generator=g).to(dev)
    outs = [torch.zeros(16, dtype=torch.int64, device=dev), torch.zeros(t, 4, dtype=torch.int32, device=dev)]
    call = lambda: ops.ExpertSort(*outs, ids)
elif what in ("dispatch", "combine", "grad"):
    ros = torch.randperm(200, generator=g).to(torch.int32).reshape(50, 4).to(dev)
    w = torch.rand(50, 4, generator=g).to(dev)
    if what == "dispatch":
        outs, x = [torch.zeros(200, 512, dtype=torch.bfloat16, device=dev)], r(50, 512)
        call = lambda: ops.ExpertDispatch(outs[0], x, ros)
    elif what == "combine":
        outs, x = [torch.zeros(50, 512, dtype=torch.bfloat16, device=dev)], r(200, 512)
        call = lambda: ops.ExpertCombine(outs[0], x, ros, w)
    else:
        outs, x, d = [torch.zeros(200, 512, dtype=torch.bfloat16, device=dev), torch.zeros(50, 4, device=dev)], r(200, 512), r(50, 512)
        call = lambda: ops.ExpertCombineGrad(*outs, d, x, ros, w)
else:
    m = {{"adapters_few": 20, "adapters_sorted": 1100, "adapters_prompts": 3000}}[what]
    x, base, a, b = r(m, 2048), r(m, 8192), r(4, 16, 2048), r(4, 8192, 16)
    ids = torch.randint(-1, 4, (m,), generator=g).to(torch.int32).to(dev)
    if m == 1100:
        x, base, a, b = r(m, 64), r(m, 128), r(4, 16, 64), r(4, 128, 16)
    outs = [torch.zeros_like(base)]
    call = lambda: ops.LowRankAdd(outs[0], base, x, a, b, ids)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):   # the process's first call of the operator
    call()
graph.replay()
torch.cuda.synchronize()
got = [o.clone() for o in outs]
for o in outs:
    o.zero_()
call()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, outs)) and any((o != 0).any() for o in outs)
ops.MatmulStatus()
print("same")
"""


@pytest.mark.parametrize("what", ["norm_rows", "norm_odd", "norm_any", "sort_one", "sort_cluster", "dispatch", "combine", "grad", "adapters_few", "adapters_sorted",
                                  "adapters_prompts"])
def test_first_call_of_a_process_inside_a_captured_graph(what):
    """Kernel attributes and occupancy are looked up at the first call: that one may be a captured one."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALL.format(what=what)], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]
