"""Routing of the MXFP4 expert layer, on the CPU."""
import pytest
import torch

from mxfp4_b200.ep import build_route
from mxfp4_b200.moe import expert_order


def order_ref(idx, E):
    """Row by row from the definition: expert by expert, token by token."""
    dst, splits, at = [[-1] * idx.shape[1] for _ in range(idx.shape[0])], [0] * E, 0
    for e in range(E):
        for t, ids in enumerate(idx.tolist()):
            for k, i in enumerate(ids):
                if i == e:
                    dst[t][k] = at
                    splits[e] += 1
                    at += 1
    return dst, splits


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E,lo,hi", [(4, 2, 5, 0, 5), (33, 4, 7, -1, 7), (5, 3, 2, -1, 0), (1, 1, 1, -1, 0),
                                         (40, 2, 6, -3, 9), (0, 2, 3, 0, 3)])
def test_ids_without_an_expert_here_have_no_row(T, k, E, lo, hi, dtype):
    g = torch.Generator().manual_seed(T + k)
    idx = torch.randint(lo, hi, (T, k), generator=g).to(dtype)
    dst, splits = expert_order(idx, E)
    want_dst, want_splits = order_ref(idx, E)
    assert dst.dtype == splits.dtype == torch.int32 and splits.is_contiguous()
    assert splits.tolist() == want_splits and dst.shape == (T, k)
    assert dst.tolist() == want_dst


def test_takes_a_dispatchers_ids():
    """What build_route hands a rank: ids local to it and -1 elsewhere."""
    g = torch.Generator().manual_seed(1)
    idx = torch.stack([torch.randperm(8, generator=g)[:3] for _ in range(20)])
    route = build_route(idx, torch.rand(20, 3, generator=g), 2, 8)
    assert (route.local_topk == -1).any()
    dst, splits = expert_order(route.local_topk, 4)
    assert int(splits.sum()) == int((route.local_topk >= 0).sum())
    assert torch.equal(dst >= 0, route.local_topk >= 0)
