"""Sizes that the C ABI's 32-bit numbers cannot hold: refused by the Python operators, never passed on without their upper bits.  (On the meta
device: nothing of that size is allocated.)"""
import pytest
import torch

from asc_devkit_b200 import ops

BIG = 2 ** 32 + 8  # 8 in 32 bits


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def refused(call, *args, **kw):
    with pytest.raises(ValueError, match="2\\^31"):
        call(*args, **kw)


@pytest.mark.parametrize("m,n", [(BIG, 1), (1, BIG), (2 ** 31, 8)])
def test_norm(m, n):
    refused(ops.ResidualRmsNormQuant, meta(m, n, dtype=torch.int8), meta(m, dtype=torch.float32), meta(m, n), meta(n), 1e-6)


@pytest.mark.parametrize("m,n,k,lo", [(BIG, 8, 8, 1), (8, BIG, 8, 1), (8, 8, BIG, 1), (8, 8, 8, BIG)])
def test_low_rank_add(m, n, k, lo):
    refused(ops.LowRankAdd, meta(m, n), None, meta(m, k), meta(lo, 8, k), meta(lo, n, 8), meta(m, dtype=torch.int32))


def test_expert_numbers_and_choices():
    ids = meta(4, 2, dtype=torch.int32)
    refused(ops.ExpertSort, meta(BIG, dtype=torch.int64), ids, ids)
    slots = meta(1, BIG, dtype=torch.int32)
    refused(ops.ExpertDispatch, meta(8, 16), meta(1, 16), slots)
    refused(ops.ExpertCombine, meta(1, 16), meta(8, 16), slots)
    refused(ops.ExpertCombineGrad, meta(8, 16), None, meta(1, 16), meta(8, 16), slots)
