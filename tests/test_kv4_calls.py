"""Calls of the 4-bit cache that a serving loop makes at its edges: no requests, no blocks, grad mode."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_kv4 import _cache, _i32, _query


@pytest.mark.gpu
@pytest.mark.parametrize("new", [None, 3])
@pytest.mark.parametrize("selected", [False, True])
def test_a_batch_without_requests(pkg, cuda, new, selected):
    pool = pkg.kv4_pool(4, 2, 128, device=cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    shape = (0, 8, 128) if new is None else (0, new, 8, 128)
    more = {}
    if selected and new is None:
        more = dict(selected=none.new_zeros(0, 2, 5),
                    selected_count=none.new_zeros(0, 2))
    status = none.new_zeros(1)
    out, lse = pkg.attention_kv4(torch.zeros(shape, dtype=torch.float16, device=cuda), pool, none.new_zeros(0, 7), none,
                                 return_lse=True, status=status, **more)
    assert out.shape == shape and out.dtype == torch.float16 and lse.shape == shape[:-1]
    free, top = torch.arange(4, dtype=torch.int32, device=cuda), _i32([4], cuda)
    slots, positions, cu = pkg.plan_blocks(none, none, none.new_zeros(0, 7), free, top, 6, status=status)
    assert slots.tolist() == [-1] * 6 and positions.tolist() == [0] * 6 and cu.tolist() == [0]
    assert free.tolist() == [0, 1, 2, 3] and int(top) == 4 and int(status) == 0
    with pytest.raises(TypeError, match="int32"):
        pkg.plan_blocks(none, none, none.new_zeros(0, 7), free, top, 6, status=status.long())


@pytest.mark.gpu
def test_a_table_without_columns_holds_nothing(pkg, cuda):
    pool = pkg.kv4_pool(4, 2, 128, device=cuda)
    q = torch.randn(3, 4, 128, device=cuda)
    table = torch.zeros(3, 0, dtype=torch.int32, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = pkg.attention_kv4(q, pool, table, _i32([0, 0, 0], cuda), return_lse=True, status=status)
    assert not out.any() and torch.isneginf(lse).all() and int(status) == 0
    out = pkg.attention_kv4(q, pool, table, _i32([0, 5, 50], cuda), status=status)
    assert not out.any() and int(status) == pkg.SA_DEV_BAD_BLOCK


@pytest.mark.gpu
def test_a_query_that_requires_grad_is_refused_in_grad_mode(pkg, cuda):
    rng = np.random.default_rng(1)
    pool, table = _cache(rng, 1, [40], 2, 128, cuda)
    args = [torch.as_tensor(pool, device=cuda), _i32(table, cuda), _i32([40], cuda)]
    q = _query(rng, (1, 4, 128), torch.float32, cuda)
    want = pkg.attention_kv4(q, *args)
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        pkg.attention_kv4(q, *args)
    with torch.no_grad():
        assert torch.equal(pkg.attention_kv4(q, *args), want)
    with torch.inference_mode():
        assert torch.equal(pkg.attention_kv4(q, *args), want)
    assert torch.equal(pkg.attention_kv4(q.detach(), *args), want)


@pytest.mark.gpu
def test_lists_without_room_attend_the_newest_block(pkg, cuda):
    rng = np.random.default_rng(2)
    pool, table = _cache(rng, 2, [70, 20], 2, 64, cuda)
    args = [_query(rng, (2, 4, 64), torch.bfloat16, cuda), torch.as_tensor(pool, device=cuda), _i32(table, cuda),
            _i32([70, 20], cuda)]
    zero, counts = torch.zeros(2, 2, 3, dtype=torch.int32, device=cuda), _i32([[5, 0], [0, -1]], cuda)
    want = pkg.attention_kv4(*args, selected=zero, selected_count=torch.zeros_like(counts))
    assert torch.equal(pkg.attention_kv4(*args, selected=zero[..., :0].contiguous(), selected_count=counts), want)
