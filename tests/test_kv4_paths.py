"""attention_kv4 over batches that reach every split and join of its kernels, types and head_dims included."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_kv4 import HALF_STEP, TYPES, _i32


def _filled(pkg, gen, lens, kh, d, device):
    """A pool with the requests' rows packed into scattered blocks, its table, and the table on the GPU."""
    held = -(-np.asarray(lens) // 32)
    total = int(held.sum()) + 1
    pool = pkg.kv4_pool(total, kh, d, device=device)
    x = torch.randn(2, 4096, kh, d, generator=gen, device=device)
    for at in range(0, total * 32, 4096):
        slots = torch.arange(at, min(at + 4096, total * 32), dtype=torch.int32, device=device)
        pkg.pack_kv4(pool, x[0, :len(slots)].roll(at // 32, 2), x[1, :len(slots)].roll(at // 32, 2), slots)
    ids = torch.randperm(total, generator=gen, device=device).cpu().numpy()
    table, ends = np.full((len(lens), max(1, int(held.max()))), -1, np.int64), np.cumsum(held)
    for b in range(len(lens)):
        table[b, :held[b]] = ids[ends[b] - held[b]:ends[b]]
    return pool, _i32(table, device)


def _check_request(pkg, out, lse, q, pool, table, length, b, ids=None):
    """Request b of a call against float64 over the rows that unpack_kv4 gives; ids: logical blocks a KV head.

    Element by element: 2^-20 of the sum of a logit's terms and 2^-19 of the group's largest value, as the kernel's
    FP32 arithmetic allows; 2^-10 of it where BF16 outputs carry FP16 weights; one rounding to the output type.
    """
    kh, d = pool.shape[1], pool.shape[2] // 36
    new, qh = q.shape[1], q.shape[2]
    if length == 0:
        assert not out[b].any() and torch.isneginf(lse[b]).all()
        return
    for h in range(kh):
        where = torch.arange(length, device=q.device)
        if ids is not None:
            blocks = torch.as_tensor(ids[h], device=q.device)
            where = (blocks[:, None] * 32 + torch.arange(32, device=q.device)).reshape(-1)
            where = where[where < length]
        slots = (table[b, where // 32] * 32 + where % 32).int()
        k, v = (t[:, h].double() for t in pkg.unpack_kv4(pool, slots, torch.float32))
        size = v.abs().view(-1, d // 64, 64).amax((0, 2)).repeat_interleave(64)  # |s c + m| of the rows seen
        size = size + (v.view(-1, d // 64, 64).amax(2) - v.view(-1, d // 64, 64).amin(2)).amax(0).repeat_interleave(64)
        for i in range(new):
            rows = slice(h * (qh // kh), (h + 1) * (qh // kh))
            sees = where <= length - new + i
            if not bool(sees.any()):
                assert not out[b, i, rows].any() and torch.isneginf(lse[b, i, rows]).all()
                continue
            x = q[b, i, rows].double() @ k[sees].T / math.sqrt(d)
            terms = (q[b, i, rows].double().abs() @ k[sees].abs().T / math.sqrt(d)).amax(-1, keepdim=True) * 2
            want = torch.softmax(x, -1) @ v[sees]
            weight = 2.0 ** -20 * terms + 2.0 ** -19 + (2.0 ** -10 if out.dtype == torch.bfloat16 else 0.0)
            tol = HALF_STEP[out.dtype] * want.abs() * (1 + 2.0 ** -7) + weight * size + 2.0 ** -25
            off = ((out[b, i, rows].double() - want).abs() / tol).max()
            assert float(off) <= 1, f"request {b}, row {i}, KV head {h}: {float(off):.3g} of the tolerance"
            far = (lse[b, i, rows].double() - torch.logsumexp(x, -1)).abs()
            assert bool((far <= 2.0 ** -20 * terms[:, 0] + 2.0 ** -18 + 2.0 ** -23 * lse[b, i, rows].double().abs()).all())


def _run(pkg, cuda, dtype, d, n, kh, group, new, longest, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    rng = np.random.default_rng(seed)
    lens = [int(x) for x in rng.integers(0, longest + 1, n)]
    lens[0], lens[n // 2], lens[-1] = longest, 0, 1
    pool, table = _filled(pkg, gen, lens, kh, d, cuda)
    q = torch.randn(n, new, kh * group, d, generator=gen, device=cuda).to(dtype)
    out, lse = pkg.attention_kv4(q, pool, table, _i32(lens, cuda), return_lse=True)
    for b in sorted({0, 1, n // 2, n - 1, *rng.integers(0, n, 3).tolist()}):
        _check_request(pkg, out, lse, q, pool, table, lens[b], b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n, kh, group, new, longest", [
    (64, 8, 4, 4, 600),    # 16 rows a tile and a merge of 16 warps for a unit, 64 lists
    (40, 8, 3, 3, 400),    # 9 of 16 rows
    (64, 8, 4, 1, 2000),   # 4 rows, units of some parts
    (100, 4, 8, 1, 900),   # 8 rows
    (33, 1, 2, 1, 9000),   # a CTA a row: few units of many parts, 33 lists
    (70, 2, 1, 7, 50),     # more warps than blocks
    (2, 2, 16, 5, 20000),  # several tiles of rows, hundreds of parts
])
def test_batches_of_every_type_and_head_dim(pkg, cuda, dtype, d, n, kh, group, new, longest):
    _run(pkg, cuda, dtype, d, n, kh, group, new, longest, d * 7 + n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, n, groups, kh, group, budget", [(64, 20, 2, 4, 4, 9), (128, 40, 1, 2, 16, 5), (128, 9, 8, 8, 4, 20),
                                                              (256, 17, 2, 2, 3, 6), (64, 300, 1, 4, 2, 3)])
def test_selections_of_more_than_32_lists(pkg, cuda, dtype, d, n, groups, kh, group, budget):
    gen = torch.Generator(device=cuda).manual_seed(n + d)
    rng = np.random.default_rng(n + d)
    lens = [int(x) for x in rng.integers(0, 1500, n)]
    lens[0], lens[1], lens[2] = 1500, 0, 32
    pool, table = _filled(pkg, gen, lens, kh, d, cuda)
    selected, counts = np.full((n, groups, budget), -1, np.int64), np.zeros((n, groups), np.int64)
    for b, length in enumerate(lens):
        sealed = max(0, -(-length // 32) - 1)
        for g in range(groups):
            counts[b, g] = c = int(rng.integers(0, min(budget, sealed) + 1))
            selected[b, g, :c] = np.sort(rng.choice(sealed, c, replace=False)) if c else []
    q = torch.randn(n, 1, kh * group, d, generator=gen, device=cuda).to(dtype)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = pkg.attention_kv4(q[:, 0], pool, table, _i32(lens, cuda), selected=_i32(selected, cuda),
                                 selected_count=_i32(counts, cuda), return_lse=True, status=status)
    assert int(status) == 0
    for b in sorted({0, 1, 2, n - 1, *rng.integers(0, n, 4).tolist()}):
        newest = max(0, -(-lens[b] // 32) - 1)
        ids = [selected[b, h // (kh // groups), :counts[b, h // (kh // groups)]].tolist() + [newest] for h in range(kh)]
        _check_request(pkg, out[:, None], lse[:, None], q, pool, table, lens[b], b, ids)
