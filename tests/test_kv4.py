"""The 4-bit paged cache: block plan, pack, unpack, attention.

Kernels are checked against the float64 restatement in kv4_oracle.py. Half a
rounding step relative to the value: bf16 2^-8, fp16 2^-11, fp32 2^-24.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

import kv4_oracle as oracle4

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---------------------------------------------------------------- the oracle itself

@pytest.mark.parametrize("d", [64, 128, 256])
def test_oracle_entry_round_trip(d):
    rng = np.random.default_rng(d)
    k, v = rng.standard_normal((2, 32, d))
    entry = oracle4.entry_of(k, v)
    got_k, got_v, _, _ = oracle4.read_entry(entry)
    np.testing.assert_array_equal(got_k, oracle4.values(k))
    np.testing.assert_array_equal(got_v, oracle4.values(v))
    key, value, shift, ks, vs = oracle4.positions(d)  # every nibble and scale has one place
    assert len(set(zip(key.ravel(), shift.ravel()))) == 32 * d == 2 * (16 * d)
    assert len(set(zip(value.ravel(), shift.ravel()))) == 32 * d
    assert value.min() == 16 * d and value.max() == 32 * d - 1
    assert sorted(set(ks.ravel())) == list(range(32 * d, 34 * d, 4))
    assert sorted(set(vs.ravel())) == list(range(34 * d, 35 * d, 2))


def test_oracle_quantisation_error_is_half_a_step():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((50, 128)) * np.exp(3 * rng.standard_normal((50, 1)))
    codes, step, low = oracle4.quantise(x)
    assert codes.min() >= 0 and codes.max() <= 15
    err = np.abs(oracle4.values(x) - x).reshape(50, 2, 64).max(-1)
    assert (err <= step / 2 * (1 + 1e-12)).all()


# ---------------------------------------------------------------- refusals (no GPU)

def test_entry_bytes(pkg):
    lib = pkg.load()
    assert [lib.sa_kv4_entry_bytes(d) for d in (64, 128, 256)] == [2304, 4608, 9216]
    assert [lib.sa_kv4_entry_bytes(d) for d in (0, 32, 96, 512)] == [0, 0, 0, 0]


def _plan_args(**over):
    a = dict(add=16, requests=4, lens=16, table=16, table_blocks=8, free=16, pool_blocks=8, top=16,
             max_tokens=64, slots=16, positions=16, cu=16)
    a.update(over)
    return [a["add"], a["requests"], a["lens"], a["table"], a["table_blocks"], a["free"],
            a["pool_blocks"], a["top"], a["max_tokens"], a["slots"], a["positions"], a["cu"], None, None]


@pytest.mark.parametrize("over, status", [
    (dict(add=None), "INVALID_ARG"), (dict(lens=None), "INVALID_ARG"), (dict(table=None), "INVALID_ARG"),
    (dict(free=None), "INVALID_ARG"), (dict(top=None), "INVALID_ARG"), (dict(slots=None), "INVALID_ARG"),
    (dict(requests=0), "INVALID_ARG"), (dict(table_blocks=0), "INVALID_ARG"),
    (dict(pool_blocks=0), "INVALID_ARG"), (dict(requests=8193), "UNSUPPORTED"),
    (dict(pool_blocks=1 << 26), "UNSUPPORTED"), (dict(table_blocks=1 << 26), "UNSUPPORTED"),
    (dict(max_tokens=0x7FFFFFFF), "UNSUPPORTED"), (dict(requests=8192, table_blocks=1 << 20), "UNSUPPORTED"),
])
def test_plan_refusals(pkg, over, status):
    assert pkg.load().sa_plan_blocks(*_plan_args(**over)) == getattr(pkg, "SA_ERR_" + status)
    assert pkg.load().sa_last_error()


def _pack_args(**over):
    a = dict(pool=16, blocks=4, key=16, value=16, type=1, slots=16, tokens=3, heads=2, d=128)
    a.update(over)
    return [a["pool"], a["blocks"], a["key"], a["value"], a["type"], 256, 128, 256, 128, a["slots"],
            a["tokens"], a["heads"], a["d"], None, None]


def _unpack_args(**over):
    a = dict(pool=16, blocks=4, key=16, value=16, type=1, slots=16, tokens=3, heads=2, d=128)
    a.update(over)
    return [a["pool"], a["blocks"], a["slots"], a["tokens"], a["heads"], a["d"], a["key"], a["value"],
            a["type"], None, None]


@pytest.mark.parametrize("over, status", [
    (dict(pool=None), "INVALID_ARG"), (dict(slots=None), "INVALID_ARG"), (dict(key=None), "INVALID_ARG"),
    (dict(value=None), "INVALID_ARG"), (dict(blocks=0), "INVALID_ARG"), (dict(heads=0), "INVALID_ARG"),
    (dict(type=3), "INVALID_ARG"), (dict(type=-1), "INVALID_ARG"), (dict(pool=8), "INVALID_ARG"),
    (dict(d=96), "UNSUPPORTED"), (dict(d=0), "UNSUPPORTED"), (dict(blocks=1 << 26), "UNSUPPORTED"),
    (dict(tokens=1 << 31), "UNSUPPORTED"), (dict(heads=65537), "UNSUPPORTED"),
])
def test_pack_and_unpack_refusals(pkg, over, status):
    lib = pkg.load()
    assert lib.sa_pack_kv4(*_pack_args(**over)) == getattr(pkg, "SA_ERR_" + status)
    assert lib.sa_unpack_kv4(*_unpack_args(**over)) == getattr(pkg, "SA_ERR_" + status)


def test_no_tokens_is_not_an_error(pkg):
    lib = pkg.load()
    assert lib.sa_pack_kv4(*_pack_args(tokens=0, slots=None, key=None, value=None)) == 0
    assert lib.sa_unpack_kv4(*_unpack_args(tokens=0, slots=None, key=None, value=None)) == 0
    assert lib.sa_unpack_kv4(*_unpack_args(key=8)) == pkg.SA_ERR_INVALID_ARG  # unaligned output


def _attention_args(**over):
    a = dict(q=16, qt=2, pool=16, blocks=4, table=16, width=4, lens=16, selected=None, counts=None, groups=0,
             budget=0, n=2, new=1, qh=8, kh=2, d=128, out=16, ot=2, ws=1 << 12, ws_bytes=1 << 40)
    a.update(over)
    return [a["q"], a["qt"], 0, 0, 0, a["pool"], a["blocks"], a["table"], a["width"], a["lens"], a["selected"],
            a["counts"], a["groups"], a["budget"], a["n"], a["new"], a["qh"], a["kh"], a["d"], C.c_float(0.1),
            a["out"], a["ot"], None, a["ws"], a["ws_bytes"], None, None]


_SEL = dict(selected=16, counts=16, groups=2, budget=3)


@pytest.mark.parametrize("over, status", [
    (dict(q=None), "INVALID_ARG"), (dict(pool=None), "INVALID_ARG"), (dict(table=None), "INVALID_ARG"),
    (dict(lens=None), "INVALID_ARG"), (dict(out=None), "INVALID_ARG"), (dict(n=0), "INVALID_ARG"),
    (dict(new=0), "INVALID_ARG"), (dict(kh=0), "INVALID_ARG"), (dict(qh=0), "INVALID_ARG"),
    (dict(qh=9), "INVALID_ARG"), (dict(blocks=0), "INVALID_ARG"), (dict(width=0), "INVALID_ARG"),
    (dict(qt=5), "INVALID_ARG"), (dict(ot=-1), "INVALID_ARG"), (dict(pool=24), "INVALID_ARG"),
    (dict(qt=2, ot=1), "UNSUPPORTED"), (dict(qt=1, ot=0), "UNSUPPORTED"), (dict(d=32), "UNSUPPORTED"),
    (dict(_SEL, counts=None), "INVALID_ARG"), (dict(_SEL, budget=0), "INVALID_ARG"),
    (dict(_SEL, groups=0), "INVALID_ARG"), (dict(_SEL, groups=3), "INVALID_ARG"),
    (dict(_SEL, new=2), "UNSUPPORTED"), (dict(_SEL, n=5000), "UNSUPPORTED"), (dict(n=8193), "UNSUPPORTED"),
    (dict(ws=None), "CAPACITY"), (dict(ws_bytes=8), "CAPACITY"), (dict(ws=(1 << 12) + 8), "CAPACITY"),
    (dict(blocks=1 << 26), "UNSUPPORTED"), (dict(width=1 << 26), "UNSUPPORTED"),
])
def test_attention_refusals(pkg, over, status):
    lib = pkg.load()
    assert lib.sa_attention_kv4(*_attention_args(**over)) == getattr(pkg, "SA_ERR_" + status)
    assert lib.sa_last_error()


def test_attention_workspace_size(pkg):
    size = pkg.load().sa_attention_kv4_workspace_size
    assert size(1, 1, 8, 2, 128) > 0
    assert size(0, 1, 8, 2, 128) == size(1, 0, 8, 2, 128) == size(1, 1, 7, 2, 128) == 0
    assert size(1, 1, 8, 0, 128) == size(1, 1, 8, 2, 96) == 0


def test_python_refuses_cpu_tensors_and_wrong_types(pkg):
    i32 = torch.zeros(4, dtype=torch.int32)
    pool = torch.zeros(2, 2, 4608, dtype=torch.uint8)
    rows = torch.zeros(4, 2, 128)
    for call in (lambda: pkg.plan_blocks(i32, i32, i32, i32, i32, 4),
                 lambda: pkg.pack_kv4(pool, rows, rows, i32), lambda: pkg.unpack_kv4(pool, i32),
                 lambda: pkg.attention_kv4(rows, pool, i32, i32)):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="head_dim"):
        pkg.kv4_pool(2, 2, 96, device="cpu")


# ---------------------------------------------------------------- plan

def _i32(x, device):
    return torch.as_tensor(np.asarray(x, np.int32), device=device)


class _State:
    """A batch's plan state on the GPU and its numpy copy."""

    def __init__(self, rng, n, width, pool, longest, device):
        lens = rng.integers(0, longest + 1, n)
        held = -(-lens // 32)
        ids = rng.permutation(pool)
        assert held.sum() <= pool
        self.table = np.full((n, width), -7, np.int64)
        at = 0
        for b in range(n):
            self.table[b, :held[b]] = ids[at:at + held[b]]
            at += held[b]
        self.free = np.full(pool, -9, np.int64)
        self.top = pool - at
        self.free[:self.top] = ids[at:]
        self.lens = lens.astype(np.int64)
        self.gpu = [_i32(x, device) for x in (self.lens, self.table, self.free, [self.top])]

    def step(self, pkg, add, max_tokens, device):
        """One step on both sides, compared; returns the oracle's refusals and the status word."""
        status = torch.zeros(1, dtype=torch.int32, device=device)
        got = pkg.plan_blocks(_i32(add, device), *self.gpu, max_tokens, status=status)
        want = oracle4.plan(np.asarray(add), self.lens, self.table, self.free, self.top, max_tokens)
        for name, g, w in zip(("slots", "positions", "cu"), got, want[:3]):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
        _, _, _, self.lens, self.table, self.free, self.top, refused = want
        for name, g, w in zip(("lens", "table", "free", "top"), self.gpu,
                              (self.lens, self.table, self.free, [self.top])):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
        return refused, int(status)


@pytest.mark.gpu
@pytest.mark.parametrize("n, max_tokens", [(1, 1), (1, 40), (3, 0), (33, 200), (257, 1024), (256, 4096),
                                           (300, 5000), (1025, 3000), (8192, 30000)])
def test_plan_matches_the_oracle(pkg, cuda, n, max_tokens):
    rng = np.random.default_rng(n * 31 + max_tokens)
    state = _State(rng, n, 7, n * 5, 150, cuda)
    for _ in range(4):
        add = rng.integers(-60, 1 + 2 * max(1, max_tokens // n), n)
        add[rng.random(n) < 0.1] = -(1 << 31)  # finished
        add[rng.random(n) < 0.05] = 200        # mostly too long for the table
        state.step(pkg, add, max_tokens, cuda)


@pytest.mark.gpu
def test_plan_refusals_name_their_cause(pkg, cuda):
    rng = np.random.default_rng(5)
    state = _State(rng, 4, 4, 9, 0, cuda)
    refused, bits = state.step(pkg, [129, 40, 1, 1], 400, cuda)
    assert refused == ["table", None, None, None] and bits == pkg.SA_DEV_TABLE_FULL
    refused, bits = state.step(pkg, [30, 1, 100, 90], 1000, cuda)  # 5 blocks left
    assert refused == [None, None, None, "pool"] and bits == pkg.SA_DEV_POOL_EMPTY
    refused, bits = state.step(pkg, [1, 1, 1, 1], 2, cuda)
    assert refused == [None, None, "slots", "slots"] and bits == pkg.SA_DEV_SLOTS_FULL
    refused, bits = state.step(pkg, [-5, -100, 0, 0], 8, cuda)
    assert refused == [None] * 4 and bits == 0


@pytest.mark.gpu
def test_plan_sum_of_growth_beyond_32_bits(pkg, cuda):
    state = _State(np.random.default_rng(6), 5, 4, 20, 60, cuda)
    big = (1 << 31) - 1
    add = [3, big, big, big, 2]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots, positions, cu = pkg.plan_blocks(_i32(add, cuda), *state.gpu, 16, status=status)
    assert cu.tolist() == [0, 3, big, big, big, big]
    assert int(status) == pkg.SA_DEV_TABLE_FULL | pkg.SA_DEV_SLOTS_FULL
    assert state.gpu[0].tolist()[1:] == state.lens.tolist()[1:]
    assert (slots[:3] >= 0).all() and (slots[3:] == -1).all()


@pytest.mark.gpu
def test_plan_and_its_inverse_restore_the_state(pkg, cuda):
    rng = np.random.default_rng(11)
    state = _State(rng, 40, 12, 400, 200, cuda)
    lens, free, top = state.lens.copy(), state.free.copy(), state.top
    add = rng.integers(-30, 31, 40)
    add[:5] = -state.lens[:5]
    add = np.maximum(add, -state.lens)
    state.step(pkg, add, 2000, cuda)
    state.step(pkg, -add, 2000, cuda)
    np.testing.assert_array_equal(state.lens, lens)
    np.testing.assert_array_equal(state.free[:top], free[:top])  # the stack; what is above it is not part of it
    assert state.top == top


@pytest.mark.gpu
def test_plan_broken_state_is_flagged(pkg, cuda):
    """A length beyond the table or below zero, a list entry outside the pool, a
    top beyond the list: no access out of range, the request stays as it is."""
    add = _i32([1, 1, 1, 33], cuda)
    lens = _i32([-3, 1000, 5, 0], cuda)
    table = _i32([[0, 1], [2, 3], [4, 5], [6, 7]], cuda)
    free, top = _i32([99, -4, 77, 8, 9], cuda), _i32([3], cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots, _, _ = pkg.plan_blocks(add, lens, table, free, top, 64, status=status)
    assert int(status) & pkg.SA_DEV_BAD_BLOCK
    assert lens.tolist() == [-3, 1000, 6, 33]
    assert slots[:3].tolist() == [-1, -1, 4 * 32 + 5]
    assert (slots[3:] == -1).all()  # both blocks it took are outside the pool
    top = _i32([50], cuda)
    status.zero_()
    pkg.plan_blocks(_i32([0, 0, 0, 0], cuda), _i32([0] * 4, cuda), table, free, top, 4, status=status)
    assert int(status) == pkg.SA_DEV_BAD_BLOCK and top.tolist() == [5]


# ---------------------------------------------------------------- pack and unpack

def _quantised(x):
    """Oracle values of a tensor's rows, float64."""
    return oracle4.values(x.double().cpu().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, heads, d", [(1, 1, 64), (1, 8, 128), (33, 3, 128), (100, 5, 64), (65, 2, 256),
                                              (517, 8, 128)])
def test_pack_then_unpack(pkg, cuda, dtype, tokens, heads, d):
    gen = torch.Generator(device=cuda).manual_seed(tokens + d)
    k = torch.randn(tokens, heads, d, generator=gen, device=cuda).to(dtype)
    v = (torch.randn(tokens, heads, d, generator=gen, device=cuda) * 0.01).to(dtype)
    blocks = tokens // 32 + 3
    slots = torch.randperm(blocks * 32, generator=gen, device=cuda)[:tokens].int()
    pool = pkg.kv4_pool(blocks, heads, d, device=cuda)
    pool.fill_(0xA5)
    before = pool.clone()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    pkg.pack_kv4(pool, k, v, slots, status=status)
    # the bytes: every entry as the oracle lays it out, untouched rows as they were
    entries = {}
    used = np.zeros((blocks, 32), bool)
    for t, s in enumerate(slots.tolist()):
        used[s // 32, s % 32] = True
        for h in range(heads):
            rows = entries.setdefault((s // 32, h), (np.zeros((32, d)), np.zeros((32, d))))
            rows[0][s % 32] = k[t, h].double().cpu().numpy()
            rows[1][s % 32] = v[t, h].double().cpu().numpy()
    host, old = pool.cpu().numpy(), before.cpu().numpy()
    for (block, h), (kr, vr) in entries.items():
        got, want = oracle4.read_entry(host[block, h]), oracle4.read_entry(oracle4.entry_of(kr, vr))
        was = oracle4.read_entry(old[block, h])
        for g, w, o in zip(got[:2], want[:2], was[:2]):
            np.testing.assert_array_equal(g[used[block]], w[used[block]])
            np.testing.assert_array_equal(g[~used[block]], o[~used[block]])
    for out in TYPES:
        ku, vu = pkg.unpack_kv4(pool, slots, out, status=status)
        for got, x in ((ku, k), (vu, v)):
            want = torch.from_numpy(_quantised(x))
            # one rounding to FP32 and one to the output type (16-bit ones keep 2^-25 below FP16's range)
            tol = want.abs() * (HALF_STEP[out] + 2.0 ** -24) * (1 + 2.0 ** -10) + 2.0 ** -25
            assert got.shape == x.shape and got.dtype == out
            assert bool(((got.double().cpu() - want).abs() <= tol).all())
    assert int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_pack_special_rows(pkg, cuda, dtype):
    """Constant groups, ties, denormal and huge ranges, NaN and infinities."""
    d = 128
    x = torch.zeros(12, 1, d, device=cuda)
    x[0] = 0.0
    x[1] = -3.25
    x[2, 0] = torch.arange(d, device=cuda) % 31 * 0.5      # exact halves of a step: ties to even
    x[3, 0] = torch.linspace(-1, 1, d, device=cuda)
    x[4, 0] = torch.linspace(0, 1e-7, d, device=cuda)      # a step below FP16's smallest
    x[5, 0] = torch.linspace(-6e4, 6e4, d, device=cuda)
    x[6, 0, 5] = float("nan")
    x[7, 0, 70] = float("inf")
    x[8, 0, 3] = -float("inf")
    x[9, 0] = torch.linspace(1.0, 1.0 + 2.0 ** -9, d, device=cuda)
    x[10, 0, ::2] = 65504.0
    x[10, 0, 1::2] = -65504.0
    x[11, 0, ::3] = -0.0
    if dtype != torch.float16:
        x[11, 0, 64:] = 1e30   # clamped to the FP16 range
        x[11, 0, 70] = -1e30
    x = x.to(dtype)
    pool = pkg.kv4_pool(1, 1, d, device=cuda)
    slots = torch.arange(12, dtype=torch.int32, device=cuda)
    pkg.pack_kv4(pool, x, x, slots)
    want = _quantised(x)
    for got in pkg.unpack_kv4(pool, slots, torch.float32):
        np.testing.assert_allclose(got.double().cpu().numpy(), want, rtol=2.0 ** -24, atol=0, equal_nan=True)
    assert np.isnan(want[6, 0, :64]).all() and np.isfinite(want[6, 0, 64:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_pack_strided_and_unaligned_rows(pkg, cuda, dtype):
    """Slices of a fused projection, transposed heads, a base off every alignment."""
    gen = torch.Generator(device=cuda).manual_seed(8)
    tokens, heads, d = 37, 3, 64
    base = torch.randn(tokens, 2 * heads * d + 7, generator=gen, device=cuda).to(dtype)
    k = base[:, 1:1 + heads * d].unflatten(1, (heads, d))
    v = torch.randn(heads, tokens, d + 2, generator=gen, device=cuda).to(dtype)[:, :, 2:].transpose(0, 1)
    pool = pkg.kv4_pool(2, heads, d, device=cuda)
    slots = torch.arange(64, dtype=torch.int32, device=cuda)[5:5 + tokens]
    pkg.pack_kv4(pool, k, v, slots.contiguous())
    ku, vu = pkg.unpack_kv4(pool, slots.contiguous(), torch.float32)
    np.testing.assert_allclose(ku.double().cpu().numpy(), _quantised(k), rtol=2.0 ** -24)
    np.testing.assert_allclose(vu.double().cpu().numpy(), _quantised(v), rtol=2.0 ** -24)


@pytest.mark.gpu
def test_pack_and_unpack_skip_padding_and_flag_bad_slots(pkg, cuda):
    pool = pkg.kv4_pool(2, 2, 128, device=cuda)
    before = pool.clone()
    x = torch.randn(4, 2, 128, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    pad = torch.tensor([-1, -2, -(1 << 31), -1], dtype=torch.int32, device=cuda)
    pkg.pack_kv4(pool, x, x, pad, status=status)
    assert torch.equal(pool, before) and int(status) == 0
    bad = torch.tensor([64, 1 << 30, (1 << 31) - 1, 3], dtype=torch.int32, device=cuda)
    pkg.pack_kv4(pool, x, x, bad, status=status)
    assert int(status) == pkg.SA_DEV_BAD_BLOCK
    for got in pkg.unpack_kv4(pool, torch.cat([pad, bad]), torch.float32):
        assert (got[:7] == 0).all()
        np.testing.assert_allclose(got[7:].double().cpu().numpy(), _quantised(x[3:]), rtol=2.0 ** -24)
    status.zero_()
    pkg.unpack_kv4(pool, bad, torch.float16, status=status)
    assert int(status) == pkg.SA_DEV_BAD_BLOCK
    assert pkg.unpack_kv4(pool, pad[:0])[0].shape == (0, 2, 128)
    pkg.pack_kv4(pool, x[:0], x[:0], pad[:0])


# ---------------------------------------------------------------- attention

def _cache(rng, n, lens, kh, d, device, spare=2, scale=1.0):
    """A filled pool with scattered blocks for requests of the given lengths."""
    held = -(-np.asarray(lens) // 32)
    width, total = max(1, int(held.max())), int(held.sum())
    pool = rng.integers(0, 256, (total + spare, kh, 36 * d), dtype=np.uint8)
    halves = pool.view(np.float16)  # scales: steps about 0.3, minima about -2
    steps = np.exp(0.3 * rng.standard_normal((total + spare, kh, 2 * d))) * scale
    halves[..., 16 * d:17 * d:2] = (0.3 * steps[..., :d // 2]).astype(np.float16)
    halves[..., 16 * d + 1:17 * d:2] = (-2 * steps[..., d // 2:d]).astype(np.float16)
    halves[..., 17 * d:17 * d + d // 2] = (0.3 * steps[..., d:d + d // 2]).astype(np.float16)
    halves[..., 17 * d + d // 2:] = (-2 * steps[..., -(d // 2):]).astype(np.float16)
    ids = rng.permutation(total + spare)
    table = np.full((n, width), -1, np.int64)
    at = 0
    for b in range(n):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    return pool, table


def _check(pkg, q, pool, table, lens, device, scale=None, selected=None, counts=None, out_dtype=None, status_bits=0):
    """attention_kv4 against the oracle, with tolerances from the arithmetic.

    A logit in FP32 is off by a few 2^-24 of the sum of its terms' sizes (2^-20 bounds 16 of them), which
    shifts every weight by that much relatively; weights, sums and the merge add 2^-19 of the largest |v|.
    BF16 outputs may carry weights rounded to FP16 twice (2^-11 each); the result rounds once.
    """
    d = q.shape[-1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    status = torch.zeros(1, dtype=torch.int32, device=device)
    dev = lambda x: None if x is None else _i32(x, device)  # noqa: E731
    out, lse = pkg.attention_kv4(q, torch.as_tensor(pool, device=device), dev(table), dev(lens), scale=scale,
                                 selected=dev(selected), selected_count=dev(counts), out_dtype=out_dtype,
                                 return_lse=True, status=status)
    q4 = q if q.dim() == 4 else q[:, None]
    want, want_lse, logit, size = oracle4.attention(q4.double().cpu().numpy(), pool, table, lens, scale,
                                                    selected, counts)
    got = out.double().cpu().numpy().reshape(want.shape)
    weight = 2.0 ** -20 * logit + 2.0 ** -19 + (2.0 ** -10 if out.dtype == torch.bfloat16 else 0.0)
    tol = HALF_STEP[out.dtype] * np.abs(want) * (1 + 2.0 ** -7) + (weight * size)[..., None] + 2.0 ** -25
    np.testing.assert_array_less(np.abs(got - want), tol + 1e-300)
    got_lse = lse.double().cpu().numpy().reshape(want_lse.shape)
    empty = np.isneginf(want_lse)
    np.testing.assert_array_equal(np.isneginf(got_lse), empty)
    off = np.abs(got_lse - want_lse)[~empty]
    assert (off <= (2.0 ** -20 * logit + 2.0 ** -19 + 2.0 ** -23 * np.abs(np.where(empty, 0, want_lse)))[~empty]).all()
    assert (got[empty] == 0).all()
    assert int(status) == status_bits
    return out


def _query(rng, shape, dtype, device):
    return torch.from_numpy(rng.standard_normal(shape)).to(dtype).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [31], [32], [33], [64], [1000], [0, 5, 0, 64, 97, 1, 300]])
def test_attention_lengths(pkg, cuda, dtype, lens):
    rng = np.random.default_rng(len(lens) * 1000 + lens[0])
    pool, table = _cache(rng, len(lens), lens, 2, 128, cuda)
    _check(pkg, _query(rng, (len(lens), 8, 128), dtype, cuda), pool, table, lens, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group, kh", [(1, 3), (2, 1), (3, 2), (4, 8), (5, 1), (7, 2), (8, 1), (12, 1), (16, 2), (40, 1)])
def test_attention_heads(pkg, cuda, dtype, d, group, kh):
    rng = np.random.default_rng(d + group * 7 + kh)
    lens = [95, 200]
    pool, table = _cache(rng, 2, lens, kh, d, cuda)
    _check(pkg, _query(rng, (2, group * kh, d), dtype, cuda), pool, table, lens, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [2, 3, 5, 8, 17, 40])
@pytest.mark.parametrize("group, d", [(1, 64), (4, 128), (5, 256)])
def test_attention_several_new_tokens(pkg, cuda, dtype, new, group, d):
    """Causal among the new tokens; requests shorter than new_tokens have empty rows."""
    rng = np.random.default_rng(new * 10 + group)
    lens = [new, 130, 0, max(1, new - 1), 64 + new, 1]
    pool, table = _cache(rng, 6, lens, 2, d, cuda)
    _check(pkg, _query(rng, (6, new, 2 * group, d), dtype, cuda), pool, table, lens, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [1, 2, 4])
def test_attention_selected(pkg, cuda, dtype, groups):
    rng = np.random.default_rng(groups)
    lens, kh, budget = [1000, 40, 20, 0, 33, 64], 4, 6
    pool, table = _cache(rng, 6, lens, kh, 128, cuda)
    selected = np.full((6, groups, budget), -1, np.int64)
    counts = np.zeros((6, groups), np.int64)
    for b, length in enumerate(lens):
        sealed = max(0, -(-length // 32) - 1)
        for g in range(groups):
            c = min(budget, sealed) if g else min(budget, sealed) // 2
            selected[b, g, :c] = np.sort(rng.choice(sealed, c, replace=False)) if c else []
            counts[b, g] = c
    _check(pkg, _query(rng, (6, 4 * kh, 128), dtype, cuda), pool, table, lens, cuda, selected=selected, counts=counts)


@pytest.mark.gpu
def test_attention_all_blocks_selected_is_the_dense_result(pkg, cuda):
    rng = np.random.default_rng(4)
    lens = [320, 97]
    pool, table = _cache(rng, 2, lens, 2, 128, cuda)
    q = _query(rng, (2, 8, 128), torch.float32, cuda)
    selected = np.tile(np.arange(9), (2, 2, 1))
    counts = np.array([[9, 9], [3, 3]])
    dense = _check(pkg, q, pool, table, lens, cuda)
    chosen = _check(pkg, q, pool, table, lens, cuda, selected=selected, counts=counts)
    assert torch.equal(dense, chosen)


@pytest.mark.gpu
def test_attention_bad_ids_lengths_and_blocks(pkg, cuda):
    """Out-of-range or repeated ids, table entries outside the pool, lengths beyond the
    table: skipped, flagged, never read."""
    rng = np.random.default_rng(9)
    lens = [200, 200]
    pool, table = _cache(rng, 2, lens, 2, 128, cuda)
    q = _query(rng, (2, 4, 128), torch.float32, cuda)
    selected = np.array([[[-1, 2, 2, 4]] * 2, [[0, 3, 1, 6]] * 2])
    counts = np.full((2, 2), 4)
    # what is left of the lists: 2, 4 and 0, 3 (6 is the newest block, 1 is out of order)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = pkg.attention_kv4(q, torch.as_tensor(pool, device=cuda), _i32(table, cuda), _i32(lens, cuda),
                            selected=_i32(selected, cuda), selected_count=_i32(counts, cuda), status=status)
    assert int(status) == pkg.SA_DEV_BAD_BLOCK
    kept = np.array([[[2, 4]] * 2, [[0, 3]] * 2])
    want = _check(pkg, q, pool, table, lens, cuda, selected=kept, counts=np.full((2, 2), 2))
    torch.testing.assert_close(out, want, rtol=1e-5, atol=1e-5)
    table[0, 3], table[1, 0], table[1, 6] = -1, pool.shape[0], 1 << 30
    _check(pkg, q, pool, table, lens, cuda, status_bits=pkg.SA_DEV_BAD_BLOCK)
    _check(pkg, q, pool, table, [-4, 225], cuda, status_bits=pkg.SA_DEV_BAD_BLOCK)
    table[:] = -1
    _check(pkg, q, pool, table, lens, cuda, status_bits=pkg.SA_DEV_BAD_BLOCK)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_ignores_what_is_behind_the_last_token(pkg, cuda, dtype):
    """NaN and infinite scales in rows that are not held change nothing."""
    rng = np.random.default_rng(12)
    lens = [33, 70, 20]
    pool, table = _cache(rng, 3, lens, 2, 128, cuda)
    q = _query(rng, (3, 8, 128), dtype, cuda)
    clean = _check(pkg, q, pool, table, lens, cuda)
    halves = pool.view(np.float16)
    _, _, _, ks, vs = oracle4.positions(128)
    for b, length in enumerate(lens):
        last = table[b, (length - 1) // 32]
        for r in range(length % 32, 32):
            for h in range(2):
                for at in set(ks[r]) | set(vs[r]):
                    halves[last, h, at // 2] = np.float16(np.nan if r % 2 else np.inf)
                halves[last, h, (vs[r] + 128) // 2] = np.float16(-np.inf if r % 3 else np.nan)
                halves[last, h, ks[r] // 2 + 1] = np.float16(-np.inf if r % 3 else np.nan)
    assert torch.equal(_check(pkg, q, pool, table, lens, cuda), clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_nan_in_a_held_row_stays_in_its_request(pkg, cuda, dtype):
    rng = np.random.default_rng(13)
    lens = [70, 70]
    pool, table = _cache(rng, 2, lens, 2, 128, cuda)
    _, _, _, ks, _ = oracle4.positions(128)
    pool.view(np.float16)[table[0, 1], 0, ks[7] // 2] = np.float16(np.nan)
    out = pkg.attention_kv4(_query(rng, (2, 4, 128), dtype, cuda), torch.as_tensor(pool, device=cuda),
                            _i32(table, cuda), _i32(lens, cuda))
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all() and out[1].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-4, 1.0, 2e3])
def test_attention_over_small_and_large_values(pkg, cuda, dtype, size):
    """Steps near FP16's ends, and logits spread over hundreds."""
    rng = np.random.default_rng(14)
    lens = [260, 31]
    pool, table = _cache(rng, 2, lens, 2, 128, cuda, scale=size)
    q = _query(rng, (2, 8, 128), dtype, cuda)
    _check(pkg, q, pool, table, lens, cuda, scale=1 / math.sqrt(128) / size)
    _check(pkg, q, pool, table, lens, cuda, scale=8 / math.sqrt(128) / size)
    _check(pkg, q * 0, pool, table, lens, cuda)
    if dtype != torch.float16:
        _check(pkg, q * 2.0 ** 30, pool, table, lens, cuda, scale=2.0 ** -30 / size)
        _check(pkg, q * 2.0 ** -30, pool, table, lens, cuda, scale=2.0 ** 28 / size)


@pytest.mark.gpu
def test_attention_value_steps_of_very_different_sizes(pkg, cuda):
    rng = np.random.default_rng(15)
    lens = [500]
    pool, table = _cache(rng, 1, lens, 1, 128, cuda)
    halves = pool.view(np.float16)
    spread = 2.0 ** rng.integers(-14, 10, halves[..., 17 * 128:].shape)
    halves[..., 17 * 128:] = (halves[..., 17 * 128:] * spread).astype(np.float16)
    for dtype in TYPES:
        _check(pkg, _query(rng, (1, 8, 128), dtype, cuda), pool, table, lens, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", TYPES)
def test_attention_output_types_and_strided_queries(pkg, cuda, out_dtype):
    rng = np.random.default_rng(16)
    lens = [100, 37, 64]
    pool, table = _cache(rng, 3, lens, 2, 128, cuda)
    fused = _query(rng, (2, 3, 12 * 128 + 3), torch.float32, cuda)
    q = fused[:, :, 1:1 + 8 * 128].unflatten(2, (8, 128)).transpose(0, 1)
    out = _check(pkg, q, pool, table, lens, cuda, out_dtype=out_dtype)
    assert out.dtype == out_dtype and out.is_contiguous()
    assert torch.equal(out, _check(pkg, q.contiguous(), pool, table, lens, cuda, out_dtype=out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("n, longest, kh, group", [(1, 40000, 8, 4), (5, 9000, 2, 8), (64, 700, 4, 2), (300, 100, 8, 1),
                                                   (2000, 40, 1, 4)])
def test_attention_batches(pkg, cuda, n, longest, kh, group):
    """Long and short, few and many: rows split over many CTAs and many rows in one."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    rng = np.random.default_rng(n)
    lens = rng.integers(0, longest + 1, n)
    lens[-1] = longest
    held = -(-lens // 32)
    total, d = int(held.sum()) + 1, 128
    pool = pkg.kv4_pool(total, kh, d, device=cuda)
    x = torch.randn(2, 4096, kh, d, generator=gen, device=cuda)
    for at in range(0, total * 32, 4096):
        slots = torch.arange(at, min(at + 4096, total * 32), dtype=torch.int32, device=cuda)
        pkg.pack_kv4(pool, x[0, :len(slots)].roll(at // 32, 2), x[1, :len(slots)].roll(at // 32, 2), slots)
    ids = rng.permutation(total)
    table = np.full((n, int(held.max())), -1, np.int64)
    ends = np.cumsum(held)
    for b in range(n):
        table[b, :held[b]] = ids[ends[b] - held[b]:ends[b]]
    q = torch.randn(n, group * kh, d, generator=gen, device=cuda)
    out, lse = pkg.attention_kv4(q, pool, _i32(table, cuda), _i32(lens, cuda), return_lse=True)
    # float64 on the GPU over the rows that unpack gives (checked above against the oracle)
    for b in sorted(set(rng.integers(0, n, 6)) | {n - 1, int(np.argmin(lens))}):
        where = torch.arange(int(lens[b]), device=cuda)
        slots = _i32(table[b], cuda)[where // 32] * 32 + where % 32
        k, v = (t.double() for t in pkg.unpack_kv4(pool, slots.int(), torch.float32))
        if lens[b] == 0:
            assert (out[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        s = torch.einsum("hgd,thd->hgt", q[b].double().view(kh, group, d), k) / math.sqrt(d)
        want = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v).reshape(kh * group, d)
        # logits of up to 40 from terms of up to 60 in all, |v| up to 6: 6 * (2^-20 * 60 + 2^-19)
        assert float((out[b].double() - want).abs().max()) <= 6 * (2.0 ** -20 * 60 + 2.0 ** -19)
        want_lse = torch.logsumexp(s, -1).reshape(-1)
        assert float((lse[b].double() - want_lse).abs().max()) <= 2.0 ** -20 * 60 + 2.0 ** -18


@pytest.mark.gpu
def test_offsets_beyond_32_bits(pkg, cuda):
    """Blocks at the end of a pool of more than 4 GiB (and of 2^31 bytes)."""
    heads, d = 8, 128
    blocks = (1 << 32) // (heads * 4608) + 40
    pool = torch.empty(blocks, heads, 4608, dtype=torch.uint8, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(2, 90, heads, d, generator=gen, device=cuda)
    ids = [blocks - 1, blocks - 30, (1 << 31) // (heads * 4608) + 1]
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    where = torch.arange(90, device=cuda)
    slots = (table[0][where // 32] * 32 + where % 32).int()
    pkg.pack_kv4(pool, x[0], x[1], slots)
    k, v = pkg.unpack_kv4(pool, slots, torch.float32)
    np.testing.assert_allclose(k.double().cpu().numpy(), _quantised(x[0]), rtol=2.0 ** -24)
    np.testing.assert_allclose(v.double().cpu().numpy(), _quantised(x[1]), rtol=2.0 ** -24)
    small = torch.empty(3, heads, 4608, dtype=torch.uint8, device=cuda)
    small.copy_(pool[torch.tensor(ids, device=cuda)])
    q = torch.randn(1, 32, d, generator=gen, device=cuda)
    lens = torch.tensor([90], dtype=torch.int32, device=cuda)
    here = torch.arange(3, dtype=torch.int32, device=cuda)[None]
    assert torch.equal(pkg.attention_kv4(q, pool, table, lens), pkg.attention_kv4(q, small, here, lens))


# ---------------------------------------------------------------- together

def _serve(pkg, device, steps, graph=False, stream=None):
    """A batch served for some steps: plan, pack, attention for each of two layers."""
    gen = torch.Generator(device=device).manual_seed(21)
    n, kh, group, d, width, layers = 5, 2, 4, 128, 6, 2
    pools = [pkg.kv4_pool(40, kh, d, device=device) for _ in range(layers)]
    state = [torch.zeros(n, dtype=torch.int32, device=device),
             torch.full((n, width), -1, dtype=torch.int32, device=device),
             torch.arange(40, dtype=torch.int32, device=device),
             torch.tensor([40], dtype=torch.int32, device=device)]
    rows = n * 40
    add = torch.zeros(n, dtype=torch.int32, device=device)
    k, v = (torch.zeros(layers, rows, kh, d, device=device, dtype=torch.float16) for _ in range(2))
    q = torch.zeros(layers, n, group * kh, d, device=device, dtype=torch.float16)

    def step():
        slots, _, _ = pkg.plan_blocks(add, *state, rows)
        outs = []
        for layer in range(layers):
            pkg.pack_kv4(pools[layer], k[layer], v[layer], slots)
            outs.append(pkg.attention_kv4(q[layer], pools[layer], state[1], state[0]))
        return outs

    recorded = None
    history = [[[] for _ in range(n)] for _ in range(layers)]
    results = []
    for s in range(steps):
        new = torch.randint(1, 9, (n,), generator=gen, device=device) if s else torch.full((n,), 37, device=device)
        new[s % n] = -min(len(history[0][s % n]), 11) if s > 2 else new[s % n]
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen, device=device))
        add.copy_(new)
        if graph and recorded is None:
            saved = [t.clone() for t in state] + [p.clone() for p in pools]
            step()  # warm-up before the capture
            for t, o in zip([*state, *pools], saved):
                t.copy_(o)
            torch.cuda.synchronize()
            recorded = torch.cuda.CUDAGraph()
            with torch.cuda.graph(recorded):
                outs = step()
        if graph:
            recorded.replay()
        else:
            outs = step()
        at = 0
        for b, count in enumerate(new.tolist()):
            for layer in range(layers):
                past = history[layer][b]
                if count < 0:
                    del past[count:]
                past += [(k[layer, at + i].clone(), v[layer, at + i].clone()) for i in range(max(count, 0))]
            at += max(count, 0)
        for layer in range(layers):
            for b in range(n):
                kk = torch.from_numpy(_quantised(torch.stack([x[0] for x in history[layer][b]])))
                vv = torch.from_numpy(_quantised(torch.stack([x[1] for x in history[layer][b]])))
                x = torch.einsum("hgd,thd->hgt", q[layer, b].double().cpu().view(kh, group, d), kk) / math.sqrt(d)
                want = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), vv).reshape(kh * group, d)
                got = outs[layer][b].double().cpu()
                # half a step of FP16, and FP32 weights over |v| <= 6 (terms of up to 60 a logit)
                assert float((got - want).abs().max()) <= 2.0 ** -11 * 6 + 6 * (2.0 ** -20 * 60 + 2.0 ** -19)
        results.append([o.clone() for o in outs])
    return results


@pytest.mark.gpu
def test_serving_steps_together(pkg, cuda):
    _serve(pkg, cuda, 12)


@pytest.mark.gpu
def test_serving_steps_from_a_graph_and_on_another_stream(pkg, cuda):
    eager = _serve(pkg, cuda, 6)
    replayed = _serve(pkg, cuda, 6, graph=True)
    stream = torch.cuda.Stream(cuda)
    with torch.cuda.stream(stream):
        other = _serve(pkg, cuda, 6)
    for a, b, c in zip(eager, replayed, other):
        for x, y, z in zip(a, b, c):
            assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.gpu
def test_selection_from_the_cache(pkg, cuda):
    """Prompt rows into the cache, representatives from what it holds, the framework's block
    selection, and the attention over the selected blocks."""
    gen = torch.Generator(device=cuda).manual_seed(31)
    kh, group, d, tokens, budget = 2, 4, 128, 12 * 32 + 5, 5
    qh, sealed = kh * group, 12
    pool = pkg.kv4_pool(16, kh, d, device=cuda)
    state = [torch.zeros(1, dtype=torch.int32, device=cuda), torch.full((1, 16), -1, dtype=torch.int32, device=cuda),
             torch.arange(16, dtype=torch.int32, device=cuda), torch.tensor([16], dtype=torch.int32, device=cuda)]
    slots, positions, cu = pkg.plan_blocks(torch.tensor([tokens], dtype=torch.int32, device=cuda), *state, tokens)
    assert positions.tolist() == list(range(tokens)) and cu.tolist() == [0, tokens]
    k, v = (torch.randn(tokens, kh, d, generator=gen, device=cuda, dtype=torch.float16) for _ in range(2))
    pkg.pack_kv4(pool, k, v, slots)
    held = torch.stack(pkg.unpack_kv4(pool, slots[:sealed * 32], torch.float16), 1).contiguous()
    prompt = torch.randn(qh, sealed * 32, d, generator=gen, device=cuda)
    reps, _ = pkg.build_local_causal_representatives(prompt, held, sealed * 32, qh, kh, d, 32, 32, 4)
    q = torch.randn(1, qh, d, generator=gen, device=cuda)
    ids, _ = pkg.select_shared_blocks(q[0], reps, qh, sealed, d, budget, 1, 1, group=group)
    counts = torch.full((1, kh), budget, dtype=torch.int32, device=cuda)
    out = _check(pkg, q, pool.cpu().numpy(), state[1].cpu().numpy(), [tokens], cuda,
                 selected=ids[None].cpu().numpy(), counts=counts.cpu().numpy())
    # the framework's FP16 attention over the same values (rounded to FP16) is near
    mine = torch.cat([ids[0].long(), torch.tensor([sealed], device=cuda)])
    where = (mine[:, None] * 32 + torch.arange(32, device=cuda)).reshape(-1)
    where = where[where < tokens]
    kk, vv = pkg.unpack_kv4(pool, slots[where].contiguous(), torch.float16)
    packed = torch.stack([kk[:, :1], vv[:, :1]], 1).contiguous()
    near = pkg.attention(packed, q[0, :group].contiguous(), len(where), group, 1, d)
    torch.testing.assert_close(out[0, :group], near, rtol=0, atol=2e-3)


@pytest.mark.gpu
def test_calls_at_once_on_two_streams_and_from_two_graphs(pkg, cuda):
    """Attention over different caches in flight together: each call has a workspace of its own."""
    rng = np.random.default_rng(41)
    cases = []
    for lens in ([5000, 40, 0, 700], [33, 6000, 1200]):
        pool, table = _cache(rng, len(lens), lens, 2, 128, cuda)
        q = _query(rng, (len(lens), 8, 128), torch.float32, cuda)
        cases.append([q, torch.as_tensor(pool, device=cuda), _i32(table, cuda), _i32(lens, cuda)])
    want = [pkg.attention_kv4(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pkg.attention_kv4(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pkg.attention_kv4(*c))
        graphs.append(graph)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@pytest.mark.gpu
def test_a_layer_of_a_larger_tensor_and_a_broadcast_query(pkg, cuda):
    """Pools as slices of one tensor of all layers; a query with stride 0 over the requests."""
    rng = np.random.default_rng(42)
    lens = [90, 33]
    pool, table = _cache(rng, 2, lens, 2, 64, cuda)
    layers = torch.zeros(3, *pool.shape, dtype=torch.uint8, device=cuda)
    layers[1] = torch.as_tensor(pool, device=cuda)
    q = _query(rng, (1, 4, 64), torch.float16, cuda).expand(2, 4, 64)
    out = pkg.attention_kv4(q, layers[1], _i32(table, cuda), _i32(lens, cuda))
    assert torch.equal(out, _check(pkg, q, pool, table, lens, cuda))
    assert (layers[0] == 0).all() and (layers[2] == 0).all()


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run(pkg, cuda):
    """No atomics in any sum: the same call gives the same bytes."""
    rng = np.random.default_rng(43)
    lens = [int(x) for x in rng.integers(0, 4000, 24)]
    pool, table = _cache(rng, 24, lens, 2, 128, cuda)
    dev = [torch.as_tensor(pool, device=cuda), _i32(table, cuda), _i32(lens, cuda)]
    for dtype in TYPES:
        q = _query(rng, (24, 3, 8, 128), dtype, cuda)
        first = pkg.attention_kv4(q, *dev, return_lse=True)
        for _ in range(5):
            again = pkg.attention_kv4(q, *dev, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_one_long_request_among_many_short_ones(pkg, cuda):
    """A unit in hundreds of parts in a batch of many units; the others in one part or none."""
    gen = torch.Generator(device=cuda).manual_seed(44)
    n, kh, d, longest = 400, 2, 128, 30000
    lens = np.full(n, 3)
    lens[::7] = 0
    lens[200] = longest
    held = -(-lens // 32)
    total = int(held.sum())
    pool = pkg.kv4_pool(total, kh, d, device=cuda)
    x = torch.randn(2, total * 32, kh, d, generator=gen, device=cuda)
    pkg.pack_kv4(pool, x[0], x[1], torch.arange(total * 32, dtype=torch.int32, device=cuda))
    table = np.full((n, int(held.max())), -1)
    ends = np.cumsum(held)
    for b in range(n):
        table[b, :held[b]] = np.arange(ends[b] - held[b], ends[b])
    q = torch.randn(n, 4, d, generator=gen, device=cuda)
    out, lse = pkg.attention_kv4(q, pool, _i32(table, cuda), _i32(lens, cuda), return_lse=True)
    assert (out[::7] == 0).all() and torch.isneginf(lse[::7]).all()
    for b in (1, 199, 200, 201, 399):
        slots = torch.arange(int(lens[b]), dtype=torch.int32, device=cuda) + 32 * int(ends[b] - held[b])
        k, v = (t.double() for t in pkg.unpack_kv4(pool, slots, torch.float32))
        s = torch.einsum("hgd,thd->hgt", q[b].double().view(kh, 2, d), k) / math.sqrt(d)
        want = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v).reshape(4, d)
        # as in test_attention_batches: |v| up to 6, a logit summed from up to 60
        assert float((out[b].double() - want).abs().max()) <= 6 * (2.0 ** -20 * 60 + 2.0 ** -19)


@pytest.mark.gpu
def test_selected_counts_outside_the_list_are_cut(pkg, cuda):
    """A count above the budget uses the whole list, one below zero none of it."""
    rng = np.random.default_rng(45)
    lens = [300, 300]
    pool, table = _cache(rng, 2, lens, 1, 128, cuda)
    q = _query(rng, (2, 4, 128), torch.float32, cuda)
    selected = np.array([[[0, 4, 7]], [[1, 2, 3]]])
    want = _check(pkg, q, pool, table, lens, cuda, selected=selected, counts=np.array([[3], [0]]))
    out = pkg.attention_kv4(q, torch.as_tensor(pool, device=cuda), _i32(table, cuda), _i32(lens, cuda),
                            selected=_i32(selected, cuda),
                            selected_count=_i32([[(1 << 31) - 1], [-(1 << 31)]], cuda))
    assert torch.equal(out, want)
