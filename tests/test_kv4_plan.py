"""The block plan of the 4-bit cache: requests that shrink behind ones that do not fit, and its largest states."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_oracle as oracle4
from test_kv4 import _i32, _State


def _plan(add, lens, top, max_tokens, width=8):
    """The oracle's plan of a batch whose requests hold blocks 0, 1, ... in order."""
    lens = np.asarray(lens)
    table, at = np.full((len(lens), width), -1, np.int64), 0
    for b, held in enumerate(-(-lens // 32)):
        table[b, :held] = np.arange(at, at + held)
        at += held
    free = np.concatenate([np.arange(at, at + top), np.full(at, -1)])  # room for every block
    return oracle4.plan(np.asarray(add), lens, table, free, top, max_tokens)


def test_oracle_takes_tokens_back_behind_a_prompt_that_does_not_fit():
    """By hand: 100 rows asked of 64; the 40 tokens behind them go, and their two blocks with them."""
    slots, _, cu, lens, _, free, top, refused = _plan([100, -40, 0, 1], [0, 40, 7, 5], 4, 64)
    assert refused == ["slots", None, None, "slots"]
    assert lens.tolist() == [0, 0, 7, 5] and top == 6 and free[4:6].tolist() == [1, 0]
    assert (slots == -1).all() and cu.tolist() == [0, 100, 100, 100, 101]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 40, 300, 2000])
@pytest.mark.parametrize("max_tokens", [0, 64, 5000])
def test_requests_that_do_not_grow_are_served_behind_refused_prompts(pkg, cuda, n, max_tokens):
    rng = np.random.default_rng(n + max_tokens)
    state = _State(rng, n, 200, n * 8, 200, cuda)
    before = state.lens.copy()
    add = np.zeros(n, np.int64)
    add[0] = max_tokens + 100 - before[0] % 7
    add[1::3] = -rng.integers(1, 300, len(add[1::3]))
    add[2::3] = 3
    refused, bits = state.step(pkg, add, max_tokens, cuda)
    assert refused[0] == "slots" and bits == pkg.SA_DEV_SLOTS_FULL
    for b in range(1, n):
        assert (refused[b] == "slots") == (add[b] > 0)
    np.testing.assert_array_equal(state.lens[1:], np.where(add > 0, before, np.maximum(before + add, 0))[1:])


def test_loop_over_given_blocks_ends_in_unsigned_arithmetic():
    """The largest table of the documented limits: a signed index would wrap below zero behind its last block."""
    requests, width, threads = 8192, (1 << 31) // 8192 - 1, 16 * 1024
    given = requests * width  # every request gives every block of its row back
    assert given <= (1 << 31) - 1
    last = given - 1 - (given - 1) % threads  # the last turn's first index
    with np.errstate(over="ignore"):
        signed = np.int32(last) + np.int32(threads)
        unsigned = np.uint32(last) + np.uint32(threads)
    assert signed < 0 and unsigned >= given


@pytest.mark.gpu
def test_a_full_table_of_the_largest_size_given_back(pkg, cuda):
    """8,192 requests of 262,143 blocks each, far more than the pool: flagged, the list full, nothing out of range."""
    n, width, pool = 8192, (1 << 31) // 8192 - 1, 64
    table = torch.zeros(n, width, dtype=torch.int32, device=cuda)
    table[-1] = 7
    lens = torch.full((n,), width * 32, dtype=torch.int32, device=cuda)
    add = torch.full((n,), -(1 << 31), dtype=torch.int32, device=cuda)
    free, top = _i32(np.full(pool, 5), cuda), _i32([10], cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots, positions, cu = pkg.plan_blocks(add, lens, table, free, top, 3, status=status)
    assert int(status) == pkg.SA_DEV_BAD_BLOCK and int(top) == pool
    assert not lens.any() and not cu.any() and (slots == -1).all() and not positions.any()
    # the last blocks given back are the first above the old top: those of the last request
    assert free.tolist() == [5] * 10 + [7] * (pool - 10)
