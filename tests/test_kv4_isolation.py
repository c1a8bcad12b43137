"""The 4-bit cache: what one value group, token or request holds stays out of the others.

Bounds are held element by element: an output is measured against the values of its own
group of 64 elements, so that a small group next to a huge one has to be right by itself.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv4_oracle as oracle4
from test_kv4 import HALF_STEP, TYPES, _cache, _i32, _query

BLOCK, GROUP = 32, 64


def _value_places(d):
    """Halfword indices in an entry of the value step and minimum of (row, group): each [32, d / 64]."""
    _, _, _, _, step = oracle4.positions(d)
    step = step[:, ::GROUP] // 2
    return step, step + d // 2


def _set_value(pool, table, d, b, token, head, group, step, minimum):
    s, m = _value_places(d)
    entry = pool.view(np.float16)[table[b, token // BLOCK], head]
    entry[s[token % BLOCK, group]] = np.float16(step)
    entry[m[token % BLOCK, group]] = np.float16(minimum)


def _sizes(pool, table, lens, shape):
    """The largest |step| 15 + |minimum| of an output element's group over the tokens its row sees: [B, T, QH, D]."""
    n, new, qh, d = shape
    kh = pool.shape[1]
    size = np.zeros(shape)
    for b in range(n):
        blocks = -(-int(lens[b]) // BLOCK)
        for h in range(kh if blocks else 0):
            va = np.concatenate([oracle4.read_entry(pool[table[b, i], h])[3] for i in range(blocks)])
            for i in range(new):
                seen = va[:max(0, int(lens[b]) - new + i + 1)]
                if len(seen):
                    size[b, i, h * (qh // kh):(h + 1) * (qh // kh)] = np.nanmax(
                        np.where(np.isfinite(seen), seen, 0.0), 0)
    return size


def _attend(pkg, q, pool, table, lens, device, **more):
    return pkg.attention_kv4(q, torch.as_tensor(pool, device=device), _i32(table, device), _i32(lens, device), **more)


def _check_elements(pkg, q, pool, table, lens, device):
    """attention_kv4 against float64, element by element; not finite exactly where the formula is not.

    A logit in FP32 is off by 2^-20 of the sum of its terms' sizes, which moves every weight by that much; weights,
    sums and joins add 2^-19, and value steps held 2^-14 below their group's largest 2^-24, of the group's largest
    value. BF16 outputs carry weights rounded to FP16 twice (2^-11 each). One rounding to the output type, whose
    subnormals are 2^-25 off in FP16.
    """
    out = _attend(pkg, q, pool, table, lens, device)
    q4 = q if q.dim() == 4 else q[:, None]
    want, _, logit, _ = oracle4.attention(q4.double().cpu().numpy(), pool, table, lens, 1 / math.sqrt(q.shape[-1]))
    got = out.double().cpu().numpy().reshape(want.shape)
    size = _sizes(pool, table, lens, want.shape)
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(want))
    weight = 2.0 ** -20 * logit + 2.0 ** -19 + (2.0 ** -10 if out.dtype == torch.bfloat16 else 0.0)
    tol = HALF_STEP[out.dtype] * np.abs(want) * (1 + 2.0 ** -7) + weight[..., None] * size + 2.0 ** -25
    finite = np.isfinite(want)
    off = np.abs(got[finite] - want[finite]) / tol[finite]
    assert off.max() <= 1, f"{off.max():.3g} of the tolerance"
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("small", [1.0, 0.06])
@pytest.mark.parametrize("step, minimum", [(np.nan, np.nan), (np.inf, 0.0), (8736.0, -65504.0), (300.0, -2000.0),
                                           (0.0, 3.0), (2.0 ** -24, 2.0 ** -24)])
def test_a_group_of_another_size_leaves_the_others_as_they_are(pkg, cuda, dtype, d, small, step, minimum):
    """One token, then every token, with an extreme group 0; the other groups at 0.3 and 0.02 a step."""
    rng = np.random.default_rng(d)
    lens = [700, 45, 33]
    pool, table = _cache(rng, 3, lens, 2, d, cuda, scale=small)
    q = _query(rng, (3, 8, d), dtype, cuda)
    for tokens in ([3], range(700)):
        for token in tokens:
            for head in range(2):
                _set_value(pool, table, d, 0, token, head, 0, step, minimum)
        _check_elements(pkg, q, pool, table, lens, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 65504.0, -1e4])
def test_an_extreme_element_reaches_its_own_group_alone(pkg, cuda, dtype, value):
    """Through pack_kv4: one element of one token's values, and the outputs of all other groups."""
    rng = np.random.default_rng(7)
    kh, d, tokens = 2, 128, 300
    k, v = (torch.from_numpy(rng.standard_normal((tokens, kh, d))).to(dtype).to(cuda) for _ in range(2))
    v = v * 0.03
    v[20, 1, 70] = value
    pool = pkg.kv4_pool(10, kh, d, device=cuda)
    pkg.pack_kv4(pool, k, v, torch.arange(tokens, dtype=torch.int32, device=cuda))
    table = np.arange(10)[None]
    q = _query(rng, (1, 8, d), dtype, cuda)
    out = _check_elements(pkg, q, pool.cpu().numpy(), table, [tokens], cuda)
    clean = pool.clone()
    v[20, 1, 70] = 0
    pkg.pack_kv4(clean, k, v, torch.arange(tokens, dtype=torch.int32, device=cuda))
    was = _check_elements(pkg, q, clean.cpu().numpy(), table, [tokens], cuda)
    assert torch.equal(out[0, :4], was[0, :4]) and torch.equal(out[0, 4:, :64], was[0, 4:, :64])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group, d", [(1, 64), (3, 128), (4, 128), (2, 256)])
@pytest.mark.parametrize("new", [2, 5, 9, 40])
@pytest.mark.parametrize("step, minimum", [(np.nan, np.nan), (np.inf, -np.inf), (8736.0, -65504.0)])
def test_a_later_token_does_not_reach_earlier_rows(pkg, cuda, dtype, group, d, new, step, minimum):
    """Extreme values and NaN keys in the newest tokens: the rows before them keep their bytes."""
    rng = np.random.default_rng(new * 100 + d)
    lens = [64 + new // 2, 32 + new, 700, new]  # new tokens across a block's end, from its first row, far on, alone
    pool, table = _cache(rng, 4, lens, 2, d, cuda)
    q = _query(rng, (4, new, 2 * group, d), dtype, cuda)
    clean = _check_elements(pkg, q, pool, table, lens, cuda)
    _, _, _, key_step, _ = oracle4.positions(d)
    for behind in sorted({1, new // 2, new - 1}):  # the last, a middle and the second token
        dirty = pool.copy()
        for b, length in enumerate(lens):
            token = length - behind
            for head in range(2):
                _set_value(dirty, table, d, b, token, head, 0, step, minimum)
                if d > 64:
                    _set_value(dirty, table, d, b, token, head, 1, -step, minimum)
            dirty.view(np.float16)[table[b, token // BLOCK], 1, key_step[token % BLOCK, 0] // 2] = np.nan
        out = _attend(pkg, q, dirty, table, lens, cuda)
        assert torch.equal(out[:, :new - behind], clean[:, :new - behind])
        assert out[:, new - behind:, group:].isnan().all()  # the second KV head's keys
        if not math.isfinite(step):
            assert not out[:, new - behind:, :, :64].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new, group, longest", [(3, 4, 5000), (8, 1, 900), (6, 8, 300)])
def test_rows_see_their_own_tokens_with_every_element_bounded(pkg, cuda, dtype, new, group, longest):
    """Values that grow along the request: a row that saw one token more or less would be far off."""
    rng = np.random.default_rng(longest)
    lens = [int(x) for x in rng.integers(new, longest, 5)] + [longest, 31 + new, 1]
    pool, table = _cache(rng, len(lens), lens, 2, 128, cuda)
    for b, length in enumerate(lens):
        for k in range(min(new, length)):
            for head in range(2):
                for g in range(2):
                    _set_value(pool, table, 128, b, length - 1 - k, head, g, 2.0 ** (new - k - 3), 3.0 ** (new - k))
    _check_elements(pkg, _query(rng, (len(lens), new, 2 * group, 128), dtype, cuda), pool, table, lens, cuda)


def _at_the_end_of_the_range(cuda, d=128):
    """Rows [6, 1, d] whose held values pass FP16's range: the step is rounded up."""
    x = torch.zeros(6, 1, d, device=cuda)
    x[0, 0, ::2], x[0, 0, 1::2] = 65504.0, -65504.0  # 65,536 at code 15
    x[1, 0, ::2] = 65504.0                            # 65,520: the smallest that FP16 rounds to infinity
    x[2, 0] = torch.linspace(-65504.0, 65504.0, d, device=cuda)
    x[3, 0] = torch.linspace(60000.0, 65504.0, d, device=cuda)
    x[4, 0, ::2], x[4, 0, 1::2] = 1e30, -1e30         # clamped first
    x[5, 0, 3] = float("inf")                         # its group is NaN, whatever the type
    return x


@pytest.mark.gpu
def test_finite_rows_stay_finite_in_every_type(pkg, cuda):
    x = _at_the_end_of_the_range(cuda)
    pool = pkg.kv4_pool(1, 1, 128, device=cuda)
    slots = torch.arange(6, dtype=torch.int32, device=cuda)
    pkg.pack_kv4(pool, x, -x, slots)
    held = pkg.unpack_kv4(pool, slots, torch.float32)
    assert float(held[0][:5].max()) > 65519 and held[0][5, 0, :64].isnan().all()
    for got, want in zip(pkg.unpack_kv4(pool, slots, torch.float16), held):
        assert torch.equal(got.isnan(), want.isnan())
        want = want.clamp(-65504.0, 65504.0)
        off = (got.double() - want.double()).abs().nan_to_num(0.0)
        assert (off <= (want.double().abs() * 2.0 ** -11).nan_to_num(0.0) + 2.0 ** -25).all()
    for got, want in zip(pkg.unpack_kv4(pool, slots, torch.bfloat16), held):
        assert torch.equal(got.isfinite(), want.isfinite())


@pytest.mark.gpu
@pytest.mark.parametrize("query, out", [(torch.float16, None), (torch.float32, torch.float16),
                                        (torch.bfloat16, None), (torch.float32, None)])
@pytest.mark.parametrize("tokens", [1, 40, 4000])
def test_attention_over_finite_rows_is_finite(pkg, cuda, query, out, tokens):
    """All tokens hold the same extreme row: written at once, joined in a CTA, and joined from many parts."""
    x = _at_the_end_of_the_range(cuda)[1:2].expand(tokens, 1, 128)
    pool = pkg.kv4_pool(tokens // 32 + 1, 1, 128, device=cuda)
    pkg.pack_kv4(pool, x * 0, x, torch.arange(tokens, dtype=torch.int32, device=cuda))
    table = np.arange(tokens // 32 + 1)[None]
    got = _attend(pkg, torch.ones(1, 4, 128, dtype=query, device=cuda), pool.cpu().numpy(), table, [tokens], cuda,
                  out_dtype=out)
    want = oracle4.values(x[0, 0].double().cpu().numpy())
    if got.dtype == torch.float16:
        want = want.clip(-65504, 65504)
    assert got.isfinite().all()
    # the sum of equal values: FP32 sums (2^-19) and one rounding; BF16 weights as above
    tol = np.abs(want) * (HALF_STEP[got.dtype] + 2.0 ** -19 + (2.0 ** -10 if got.dtype == torch.bfloat16 else 0)) + 0.1
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new, group, d", [(4, 4, 128), (9, 1, 64), (3, 2, 256)])
def test_ordinary_later_values_and_large_later_keys(pkg, cuda, dtype, new, group, d):
    """Other values in the newest tokens leave the rows before them byte by byte as they are; keys that are far larger
    there may move their running maximum, so those rows are held to float64 again."""
    rng = np.random.default_rng(d + new)
    lens = [60 + new, 1000, new + 1, 31 + new]
    pool, table = _cache(rng, 4, lens, 2, d, cuda)
    q = _query(rng, (4, new, 2 * group, d), dtype, cuda)
    clean = _check_elements(pkg, q, pool, table, lens, cuda)
    _, _, _, key_step, _ = oracle4.positions(d)
    for b, length in enumerate(lens):
        for head in range(2):
            for g in range(d // 64):
                _set_value(pool, table, d, b, length - 1, head, g, 0.21, -1.3)
    out = _check_elements(pkg, q, pool, table, lens, cuda)
    assert torch.equal(out[:, :-1], clean[:, :-1]) and not torch.equal(out[:, -1], clean[:, -1])
    for b, length in enumerate(lens):
        for at in key_step[(length - 1) % BLOCK, ::GROUP] // 2:
            pool.view(np.float16)[table[b, (length - 1) // BLOCK], :, at] = 9.0
    _check_elements(pkg, q, pool, table, lens, cuda)
