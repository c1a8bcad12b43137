"""Workloads of the 4-bit paged KV cache: block planning, packing, reading back, attention.

Four operators of a serving loop that keeps its keys and values in 4 bits:

* ``plan``   -- block tables and slot maps on the GPU from the requests' lengths;
* ``store``  -- quantise new rows into the cache and read the same rows back;
* ``read``   -- dequantise a cached prefix into dense rows;
* ``attend`` -- attention of one or a few new tokens a request over the cache, dense or
  over a selection of its blocks.

``run`` computes them in elementary torch operations, or with ``own`` set through the
package's entry points. A cache entry (block of 32 tokens, KV head) is 36 * head_dim
bytes: key codes, value codes, key steps and minima, value steps and minima; ``_decode``
and ``_encode`` below spell the order out.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
GROUP = 64
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases

def _plan(name, requests, step, prompt, parked):
    return dict(name=name, op="plan", requests=requests, step=step, prompt=prompt, parked=parked)


def _store(name, dtype, requests, tokens, kv_heads, head_dim):
    return dict(name=name, op="store", dtype=dtype, requests=requests, tokens=tokens,
                kv_heads=kv_heads, head_dim=head_dim)


def _read(name, dtype, requests, tokens, kv_heads, head_dim):
    return dict(_store(name, dtype, requests, tokens, kv_heads, head_dim), op="read")


def _attend(name, dtype, requests, tokens, ragged, query_heads, kv_heads, head_dim, new=1, budget=0):
    return dict(name=name, op="attend", dtype=dtype, requests=requests, tokens=tokens,
                ragged=ragged, query_heads=query_heads, kv_heads=kv_heads, head_dim=head_dim,
                new=new, budget=budget)


def listed():
    return [
        # a small batch's decode step, drafted tokens taken back: pure latency
        _plan("plan-decode-8", 8, 1, 0, 0),
        # continuous batching: most requests step, some are parked, others admitted with prompts
        _plan("plan-mixed-256", 256, 1, 700, 40),
        # a large batch of prompts admitted at once
        _plan("plan-prompts-2000", 2000, 1, 257, 600),
        # one decode step of a batch: a row a request
        _store("store-decode-16", "bf16", 16, 16, 8, 128),
        # one prompt chunk of an 8-KV-head model
        _store("store-chunk-8k", "fp16", 1, 8192, 8, 128),
        # prompts of odd lengths, narrow heads
        _store("store-prompts-d64", "bf16", 13, 99991, 5, 64),
        # a short prefix in single precision
        _read("read-prefix-1k", "fp32", 3, 1003, 8, 128),
        # a 32K context read back for the next chunk of its prompt
        _read("read-prefix-32k", "bf16", 1, 32768, 8, 128),
        # one request, short context: latency
        _attend("attend-one-1k", "bf16", 1, 997, False, 16, 8, 128),
        # a 32K context with a budget of 128 blocks, single-precision queries
        _attend("attend-selected-32k", "fp32", 8, 32768, False, 32, 8, 128, budget=128),
        # variable contexts up to 32K, four drafted tokens each
        _attend("attend-ragged-drafts", "fp16", 16, 32768, True, 32, 8, 128, new=4),
        # a full decode batch at 8K
        _attend("attend-batch-8k", "bf16", 64, 8192, False, 32, 8, 128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = _draw(rng, rng.choice(["plan", "store", "read", "attend", "attend", "attend"]))
    del case["name"]
    return case


def _draw(rng, op):
    if op == "plan":
        requests = _log(rng, 1, 3000)
        return _plan("", requests, rng.choice([1, 1, 2, 5]), _log(rng, 1, 600),
                     rng.randrange(0, requests // 3 + 1))
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("store", "read"):
        tokens = _log(rng, 1, 60000 * 8 * 128 // (kv_heads * head_dim) // (2 if dtype == "fp32" else 1))
        tokens = min(tokens, 150000)
        requests = min(tokens, _log(rng, 1, 64))
        return dict(_store("", dtype, requests, tokens, kv_heads, head_dim), op=op)
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    requests = _log(rng, 1, 96)
    tokens = _log(rng, 1, min(131072, 524288 * 8 * 128 // (requests * kv_heads * head_dim) // 2))
    budget = rng.choice([0, 0, _log(rng, 1, 256)])
    new = 1 if budget or rng.random() < 0.6 else rng.randrange(2, 9)
    return _attend("", dtype, requests, tokens, rng.random() < 0.6, group * kv_heads, kv_heads,
                   head_dim, new, budget)


# ------------------------------------------------------------------ the cache's format

def _half_down(x):
    """The largest FP16 value that is not above x (|x| <= 65504)."""
    h = x.half()
    bits = h.view(torch.int16)
    below = torch.where(bits > 0, bits - 1, torch.where(bits == 0, -0x7FFF, bits + 1)).to(torch.int16)
    below = torch.where(bits == -0x8000, -0x7FFF, below).to(torch.int16)
    return torch.where(h.to(x.dtype) > x, below, bits).to(torch.int16).view(torch.float16)


def _quantise(x):
    """(codes uint8, step, minimum) of FP32 rows [..., head_dim] in groups of 64."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    finite = torch.isfinite(g).all(-1)
    g = torch.where(finite[..., None], g, 0.0).clamp(-65504.0, 65504.0)
    low = _half_down(g.amin(-1))
    step = -_half_down(-((g.amax(-1).double() - low.double()) / 15.0))
    away = (g - low.float()[..., None]).double()
    codes = torch.round(away / torch.where(step == 0, 1.0, step).double()[..., None])
    codes = torch.where(step[..., None] == 0, 0.0, codes).clamp(0, 15).to(torch.uint8)
    nan = torch.full_like(step, float("nan"))
    return codes.reshape(x.shape), torch.where(finite, step, nan), torch.where(finite, low, nan)


def _values(codes, step, low):
    """FP32 values of codes [..., head_dim], step and minimum [..., groups]."""
    c = codes.reshape(*step.shape, GROUP).float()
    return (c * step.float()[..., None] + low.float()[..., None]).reshape(codes.shape)


def _nibbles(codes):
    """Pairs of codes along the last axis into bytes, the first in the low half."""
    c = codes.reshape(*codes.shape[:-1], -1, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _encode(k, v):
    """Entries [n, 36 * D] uint8 of FP32 keys and values [n, 32, D]."""
    n, _, d = k.shape
    ng = d // GROUP
    kc, ks, km = _quantise(k)
    vc, vs, vm = _quantise(v)
    # key codes: token, 16-element piece t of every group side by side
    kb = _nibbles(kc.view(n, 32, ng, 4, 16).permute(0, 1, 3, 2, 4)).reshape(n, 16 * d)
    # value codes: token pair, 8-element piece g of every group, 4 elements, token of the pair
    vb = _nibbles(vc.view(n, 16, 2, ng, 8, 2, 4).permute(0, 1, 4, 3, 5, 2, 6)).reshape(n, 16 * d)
    # key scales: group, token % 8, token / 8, (step, minimum)
    kt = torch.stack([ks, km], -1).view(n, 4, 8, ng, 2).permute(0, 3, 2, 1, 4)
    # value scales: steps then minima; group, then the token order (t, j, h, b) of token 16j + 8h + 2t + b
    vt = torch.stack([vs, vm], 1).view(n, 2, 2, 2, 4, 2, ng).permute(0, 1, 6, 4, 2, 3, 5)
    flat = lambda x: x.contiguous().view(torch.uint8).reshape(n, 2 * d)  # noqa: E731
    return torch.cat([kb, vb, flat(kt), flat(vt)], 1)


def _decode(entries):
    """FP32 keys and values [..., 32, D] of entries [..., 36 * D]."""
    lead, d = entries.shape[:-1], entries.shape[-1] // 36
    ng = d // GROUP
    e = entries.reshape(-1, 36 * d)
    n = e.shape[0]
    both = lambda b: torch.stack([b & 15, b >> 4], -1)  # noqa: E731
    kc = both(e[:, :16 * d].reshape(n, 32, 4, ng, 8)).permute(0, 1, 3, 2, 4, 5).reshape(n, 32, d)
    vc = both(e[:, 16 * d:32 * d].reshape(n, 16, 8, ng, 2, 2, 2))
    vc = vc.permute(0, 1, 5, 3, 2, 4, 6, 7).reshape(n, 32, d)
    kt = e[:, 32 * d:34 * d].contiguous().view(torch.float16).view(n, ng, 8, 4, 2).permute(4, 0, 3, 2, 1)
    vt = e[:, 34 * d:].contiguous().view(torch.float16).view(n, 2, ng, 4, 2, 2, 2)
    vt = vt.permute(1, 0, 4, 5, 3, 6, 2)
    ks, km = kt.reshape(2, n, 32, ng)
    vs, vm = vt.reshape(2, n, 32, ng)
    return (_values(kc, ks, km).reshape(*lead, 32, d), _values(vc, vs, vm).reshape(*lead, 32, d))


# ------------------------------------------------------------------ inputs

def _rows(gen, shape):
    """Keys as they come out of a rotary embedding (a few strong channels), and values."""
    d = shape[-1]
    channel = torch.exp(0.6 * torch.randn(d, generator=gen, device=DEVICE))
    k = torch.randn(*shape, generator=gen, device=DEVICE) * channel
    return k, torch.randn(*shape, generator=gen, device=DEVICE)


def _pool(gen, blocks, kv_heads, head_dim):
    """A cache of `blocks` blocks, every entry filled."""
    entries = blocks * kv_heads
    pool = torch.empty(entries, 36 * head_dim, dtype=torch.uint8, device=DEVICE)
    chunk = 1 << 15
    for at in range(0, entries, chunk):
        n = min(chunk, entries - at)
        pool[at:at + n] = _encode(*_rows(gen, (n, BLOCK, head_dim)))
    return pool.view(blocks, kv_heads, 36 * head_dim)


def _slots(gen, requests, tokens):
    """(slots int32 [tokens], blocks): runs of tokens in scattered blocks, each run starting
    anywhere inside its first block."""
    each, more = divmod(tokens, requests)
    counts = torch.tensor([each + (b < more) for b in range(requests)], device=DEVICE)
    first = torch.randint(0, BLOCK, (requests,), generator=gen, device=DEVICE)
    blocks = (first + counts + BLOCK - 1) // BLOCK
    total = int(blocks.sum())
    ids = torch.randperm(total + 3, generator=gen, device=DEVICE)
    start = torch.cumsum(blocks, 0) - blocks
    b = torch.repeat_interleave(torch.arange(requests, device=DEVICE), counts)
    position = first[b] + torch.arange(tokens, device=DEVICE) - (torch.cumsum(counts, 0) - counts)[b]
    slots = ids[start[b] + position // BLOCK] * BLOCK + position % BLOCK
    return slots.to(torch.int32), total + 3


def _prepare_plan(case, gen):
    n, parked = case["requests"], case["parked"]
    lens = torch.randint(1, 2000, (n,), generator=gen, device=DEVICE)
    add = torch.full((n,), case["step"], device=DEVICE)
    order = torch.randperm(n, generator=gen, device=DEVICE)
    if parked:  # some requests are parked, as many come back with their prompts
        out, back = order[:parked], order[parked:2 * parked]
        lengths = torch.randint(1, case["prompt"] + 1, (2, parked), generator=gen, device=DEVICE)
        lens[out], add[out] = lengths[0], -lengths[0]
        lens[back], add[back] = 0, lengths[1]
    width = (max(2000, case["prompt"]) + case["step"]) // BLOCK + 2
    held = (lens + BLOCK - 1) // BLOCK
    total, blocks = int(held.sum()), n * width
    spare = blocks - total
    ids = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    at = torch.arange(width, device=DEVICE)[None, :] < held[:, None]
    table[at] = ids[:total]
    free = torch.full((blocks,), -1, dtype=torch.int32, device=DEVICE)
    free[:spare] = ids[total:]
    tokens = n * case["step"] + parked * case["prompt"]  # room for the step's tokens
    i32 = lambda x: x.to(torch.int32).contiguous()  # noqa: E731
    return dict(add=i32(add), back=i32(-add), lens=i32(lens), table=table, free=free,
                top=torch.tensor([spare], dtype=torch.int32, device=DEVICE), tokens=tokens)


def _prepare_attend(case, gen):
    n, new = case["requests"], case["new"]
    longest = max(case["tokens"], new)
    lens = torch.full((n,), longest, device=DEVICE)
    if case["ragged"]:
        lens = torch.randint(new, longest + 1, (n,), generator=gen, device=DEVICE)
        if n >= 4:
            lens[n // 2] = 0  # a slot of the batch without a request
    held = (lens + BLOCK - 1) // BLOCK
    width, total = max(1, int(held.max())), int(held.sum())
    pool = _pool(gen, total + 2, case["kv_heads"], case["head_dim"])
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    at = torch.arange(width, device=DEVICE)[None, :] < held[:, None]
    table[at] = torch.randperm(total + 2, generator=gen, device=DEVICE)[:total].to(torch.int32)
    q = torch.randn(n, new, case["query_heads"], case["head_dim"], generator=gen, device=DEVICE)
    state = dict(q=q.to(TYPES[case["dtype"]]), pool=pool, table=table, lens=lens.to(torch.int32),
                 selected=None, counts=None)
    if case["budget"]:  # the first block, the last ones and scattered others, for each KV head
        sealed = (held - 1).clamp_min(0)
        score = torch.rand(n, case["kv_heads"], width, generator=gen, device=DEVICE)
        at = torch.arange(width, device=DEVICE)
        score[..., 0] = 2.0
        score = torch.where(at >= sealed[:, None, None] - 4, 3.0, score)
        score = torch.where(at >= sealed[:, None, None], -1.0, score)
        ids = torch.topk(score, min(case["budget"], width), -1).indices
        counts = sealed.clamp_max(ids.shape[-1])
        used = torch.arange(ids.shape[-1], device=DEVICE) < counts[:, None, None]
        ids = torch.where(used, ids, 1 << 30).sort(-1).values
        state["selected"] = torch.where(used, ids, -1).to(torch.int32)
        state["counts"] = counts[:, None].expand(n, case["kv_heads"]).contiguous().to(torch.int32)
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    op = case["op"]
    if op == "plan":
        state = _prepare_plan(case, gen)
    elif op == "attend":
        state = _prepare_attend(case, gen)
    else:
        heads, d, tokens = case["kv_heads"], case["head_dim"], case["tokens"]
        slots, blocks = _slots(gen, case["requests"], tokens)
        state = dict(slots=slots, head_dim=d)
        if op == "read":
            state["pool"] = _pool(gen, blocks, heads, d)
        else:
            # keys and values are the last two thirds of a projection's output rows
            k, v = _rows(gen, (tokens, heads * d))
            qkv = torch.cat([torch.zeros_like(k), k, v], 1).to(TYPES[case["dtype"]])
            state["pool"] = torch.zeros(blocks, heads, 36 * d, dtype=torch.uint8, device=DEVICE)
            state["k"] = qkv[:, heads * d:2 * heads * d].view(tokens, heads, d)
            state["v"] = qkv[:, 2 * heads * d:].view(tokens, heads, d)
    state["op"], state["dtype"] = op, TYPES.get(case.get("dtype"))
    return state


# ------------------------------------------------------------------ one pass

def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _plan_plain(add, lens, table, free, top, tokens):
    """The plan's outputs and the state after it, as new tensors."""
    n, width = table.shape
    add, lens, start = add.long(), lens.long(), top.long()
    grow = add.clamp_min(0)
    ends = torch.cumsum(grow, 0)
    begins = ends - grow
    after = (lens + add).clamp_min(0)
    held, want = (lens + BLOCK - 1) // BLOCK, (after + BLOCK - 1) // BLOCK
    refused = (want > width) | (ends > tokens)
    need = torch.where(refused, 0, (want - held).clamp_min(0))
    refused = refused | ((need > 0) & (torch.cumsum(need, 0) > start))
    need = torch.where(refused, 0, need)
    after, want = torch.where(refused, lens, after), torch.where(refused, held, want)
    j = torch.arange(width, device=add.device)[None, :]
    taken = (j >= held[:, None]) & (j < want[:, None])
    at = start - 1 - ((torch.cumsum(need, 0) - need)[:, None] + j - held[:, None])
    new_table = torch.where(taken, free[at.clamp(0, free.numel() - 1)], table)
    gone = (held - want).clamp_min(0)
    given = (j >= want[:, None]) & (j < held[:, None])
    place = start - need.sum() + gone.sum() - 1 - ((torch.cumsum(gone, 0) - gone)[:, None] + j - want[:, None])
    new_free = free.clone()
    new_free[place[given]] = table[given]
    i = torch.arange(tokens, device=add.device)
    b = torch.searchsorted(ends, i, right=True)
    inside = b < n
    b = b.clamp_max(n - 1)
    position = torch.where(inside, lens[b] + i - begins[b], 0)
    good = inside & ~refused[b]
    slot = new_table[b, (position // BLOCK).clamp_max(width - 1)].long() * BLOCK + position % BLOCK
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return ([i32(torch.where(good, slot, -1)), i32(position), i32(cu)],
            [i32(after), new_table, new_free, i32(start - need.sum() + gone.sum())])


def _attend_plain(s):
    q, pool, table, lens = s["q"].float(), s["pool"], s["table"].long(), s["lens"].long()
    n, new, heads, d = q.shape
    kv_heads = pool.shape[1]
    held = (lens + BLOCK - 1) // BLOCK
    if s["selected"] is None:
        logical = torch.arange(table.shape[1], device=q.device).expand(n, kv_heads, -1)
        used = logical < held[:, None, None]
    else:  # the selected blocks, then the block of the newest token
        last = (held - 1)[:, None, None].expand(n, kv_heads, 1)
        logical = torch.cat([s["selected"].long(), last], -1)
        used = torch.arange(logical.shape[-1], device=q.device) < s["counts"].long()[..., None]
        used = used | (torch.arange(logical.shape[-1], device=q.device) == logical.shape[-1] - 1)
        used = used & (held > 0)[:, None, None]
    logical = torch.where(used, logical, 0)
    block = torch.gather(table[:, None, :].expand(-1, kv_heads, -1), 2, logical).clamp_min(0)
    k, v = _decode(pool[block, torch.arange(kv_heads, device=q.device)[None, :, None]])
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    position = (logical[..., None] * BLOCK + torch.arange(BLOCK, device=q.device)).flatten(2)
    limit = lens[:, None] - new + torch.arange(new, device=q.device)  # newest position a row sees
    seen = used.repeat_interleave(BLOCK, -1)[:, :, None] & (position[:, :, None] <= limit[:, None, :, None])
    rows = q.view(n, new, kv_heads, heads // kv_heads, d).permute(0, 2, 1, 3, 4)
    x = torch.matmul(rows.flatten(2, 3), k.transpose(-1, -2)).view(*rows.shape[:-1], -1) / math.sqrt(d)
    seen = seen[:, :, :, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)).masked_fill(~seen, 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).view(rows.shape) / torch.where(total == 0, 1.0, total)
    lse = torch.where(total == 0, -math.inf, top + torch.log(total))[..., 0]
    return [o.permute(0, 2, 1, 3, 4).reshape(n, new, heads, d).to(s["q"].dtype),
            lse.permute(0, 2, 1, 3).reshape(n, new, heads)]


def run(state):
    s, op = state, state["op"]
    if own:
        sa = _package()
        if op == "plan":
            ahead = sa.plan_blocks(s["add"], s["lens"], s["table"], s["free"], s["top"], s["tokens"])
            back = sa.plan_blocks(s["back"], s["lens"], s["table"], s["free"], s["top"], s["tokens"])
            return [*ahead, *back, s["lens"], s["table"], s["free"], s["top"]]
        if op == "store":
            sa.pack_kv4(s["pool"], s["k"], s["v"], s["slots"])
        if op in ("store", "read"):
            return sa.unpack_kv4(s["pool"], s["slots"], s["dtype"])
        return sa.attention_kv4(s["q"], s["pool"], s["table"], s["lens"], selected=s["selected"],
                                selected_count=s["counts"], return_lse=True)
    if op == "plan":
        ahead, (lens, table, free, top) = _plan_plain(s["add"], s["lens"], s["table"], s["free"],
                                                      s["top"], s["tokens"])
        back, after = _plan_plain(s["back"], lens, table, free, top, s["tokens"])
        return [*ahead, *back, *after]
    if op == "store":
        return [_values(*_quantise(x.float())).to(s["dtype"]) for x in (s["k"], s["v"])]
    if op == "read":
        slots = s["slots"].long()
        block, token = slots // BLOCK, slots % BLOCK
        name, at = torch.unique(block, return_inverse=True)
        k, v = _decode(s["pool"][name])
        return [x.to(s["dtype"]).transpose(1, 2)[at, token] for x in (k, v)]
    return _attend_plain(s)


# ------------------------------------------------------------------ work and exact values

def work(case):
    op = case["op"]
    if op == "plan":
        n, parked = case["requests"], case["parked"]
        room = n * case["step"] + parked * case["prompt"]
        # twice: lengths, changes and offsets; slots and positions; the blocks taken and given back
        return {"bytes": 2 * (n * 16 + room * 8 + parked * case["prompt"] // 64 * 16), "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    elements = case["tokens"] * 2 * case["kv_heads"] * case["head_dim"]
    if op == "read":
        return {"bytes": elements * (0.5625 + size) + case["tokens"] * 4, "flops": 2 * elements}
    if op == "store":  # rows in, entries out; entries in, rows out
        return {"bytes": elements * (2 * size + 2 * 0.5625) + case["tokens"] * 8, "flops": 8 * elements}
    tokens = (case["tokens"] + case["new"]) / 2 if case["ragged"] else max(case["tokens"], case["new"])
    if case["budget"]:
        tokens = min(tokens, (case["budget"] + 1) * BLOCK)
    n, qh, d = case["requests"], case["query_heads"], case["head_dim"]
    return {"bytes": n * (tokens * 2 * case["kv_heads"] * d * 0.5625 + case["new"] * qh * (2 * d * size + 4)),
            "flops": 4.0 * n * tokens * case["new"] * qh * d}


def _exact_half(x, up):
    """The FP16 neighbour of float64 values that is not below (up) or not above them."""
    with np.errstate(over="ignore"):
        h = x.astype(np.float16)
    off = h.astype(np.float64) < x if up else h.astype(np.float64) > x
    return np.where(off, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h).astype(np.float64)


def _exact_store(x):
    """The definition in float64: what the cache holds for rows x."""
    rows, heads, d = x.shape
    out = torch.empty(rows, heads, d, dtype=torch.float64)
    step_rows = max(1, (1 << 22) // (heads * d))
    for at in range(0, rows, step_rows):
        g = x[at:at + step_rows].double().cpu().numpy().reshape(-1, 64)
        low = _exact_half(g.min(1), up=False)[:, None]
        step = _exact_half((g.max(1) - low[:, 0]) / 15, up=True)[:, None]
        code = np.where(step > 0, np.rint((g - low) / np.where(step > 0, step, 1)), 0)
        out[at:at + step_rows] = torch.from_numpy((low + step * code).reshape(-1, heads, d))
    return out


def _exact_entry(bytes_, d):
    """Float64 keys and values [32, m, d] of entries [m, 36 d], element by element position."""
    r, c = torch.meshgrid(torch.arange(32), torch.arange(d), indexing="ij")
    group, e, ng = c // 64, c % 64, d // 64
    key_at = r * (d // 2) + 8 * ng * (e // 16) + 8 * group + e % 16 // 2
    value_at = 16 * d + r // 2 * d + 8 * ng * (e // 8) + 8 * group + 4 * (e % 8 // 4) + 2 * (r % 2) + e % 4 // 2
    key_scale = 16 * d + (group * 8 + r % 8) * 8 + r // 8 * 2
    value_scale = 17 * d + group * 32 + r % 8 // 2 * 8 + r // 16 * 4 + r % 16 // 8 * 2 + r % 2
    halves = bytes_.contiguous().view(torch.float16)
    odd = (c % 2 * 4).to(bytes_.device).reshape(-1).to(torch.uint8)
    take = lambda t, at: t[:, at.reshape(-1).to(t.device)]  # noqa: E731
    code = lambda at: ((take(bytes_, at) >> odd) & 15).double()  # noqa: E731
    k = code(key_at) * take(halves, key_scale).double() + take(halves, key_scale + 1).double()
    v = code(value_at) * take(halves, value_scale).double() + take(halves, value_scale + ng * 32).double()
    return k.view(-1, 32, d), v.view(-1, 32, d)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        return [_exact_store(s["k"]), _exact_store(s["v"])]
    d = case["head_dim"]
    if case["op"] == "read":
        slots = s["slots"].long().cpu()
        keys, values = [], []
        for at in range(0, len(slots), 4096):  # a token's whole block is decoded, and its row taken
            part = slots[at:at + 4096]
            name, inverse = torch.unique(part // 32, return_inverse=True)
            heads = s["pool"].shape[1]
            k, v = _exact_entry(s["pool"][name.to(s["pool"].device)].reshape(-1, 36 * d), d)
            keys.append(k.view(-1, heads, 32, d)[inverse, :, part % 32])
            values.append(v.view(-1, heads, 32, d)[inverse, :, part % 32])
        return [torch.cat(keys), torch.cat(values)]
    n, new, qh, kh = case["requests"], case["new"], case["query_heads"], case["kv_heads"]
    if n * kh > 1000 or sum(s["lens"].tolist()) * kh * d > 1 << 30:
        return None  # more than some seconds
    out = torch.zeros(n, new, qh, d, dtype=torch.float64, device=DEVICE)
    lse = torch.full((n, new, qh), -math.inf, dtype=torch.float64, device=DEVICE)
    for b in range(n):
        length = int(s["lens"][b])
        blocks = -(-length // 32)
        for h in range(kh if blocks else 0):
            mine = list(range(blocks))
            if s["selected"] is not None:
                mine = s["selected"][b, h, :int(s["counts"][b, h])].tolist() + [blocks - 1]
            mine = torch.tensor(mine, device=DEVICE)
            k, v = _exact_entry(s["pool"][s["table"][b, mine].long(), h], d)
            where = (mine[:, None] * 32 + torch.arange(32, device=DEVICE)).reshape(-1)
            k, v = k.reshape(-1, d), v.reshape(-1, d)
            for i in range(new):
                sees = where <= length - new + i
                if not bool(sees.any()):
                    continue
                mine_q = slice(h * (qh // kh), (h + 1) * (qh // kh))
                x = s["q"][b, i, mine_q].double() @ k[sees].T / math.sqrt(d)
                lse[b, i, mine_q] = torch.logsumexp(x, -1)
                out[b, i, mine_q] = torch.softmax(x, -1) @ v[sees]
    return [out, lse]
