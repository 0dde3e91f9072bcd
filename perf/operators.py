"""The operators between a batch's hidden rows and its paged cache, as cases that can be timed and compared.

  tables    block tables, slot map and positions of a batch, from the requests' lengths, with the pages taken from a stack of free
            ones (``ops.batch_tables``)
  rope      rotary positions of query and key rows: half and interleaved pairs, part of the head, scaled frequencies, strided rows, and
            the transposed rotation that takes gradients back (``ops.rope_rows``)
  append    the rows of several requests into the paged cache through a slot map, with the rotary positions of q and k on the way
            (``ops.kv_append_slots``)
  linear    product of 8-bit rows and 8-bit weights with a scale for each token and each channel, from 16-bit rows (quantised in the
            pass) or from rows that are 8 bits already (``ops.quantize_rows``, ``ops.int8_linear``)

With ``own`` false a pass computes the same in elementary torch operations in 32 bits (angles in 64); with ``own`` true it makes the
framework's calls.  Both take the same inputs; the weight that the framework keeps laid out is made by ``prepare``, as a program
does when it loads a checkpoint.
"""
import math
import types

import numpy as np
import torch

own = False

PAGE, HEAD_DIM = 256, 128
LARGEST_PRODUCT = 8192 * 4096 * 16384  # rows * columns * channels, and
LARGEST_ROWS = 8192 * 40               # rows * heads, and
LARGEST_TABLE = 1 << 20                # rows of a batch: what no drawn case exceeds


def _tables(name, requests, mean_rows, mean_cached, max_blocks, ended=0.0, idle=0.0):
    return dict(name=name, kind="tables", requests=requests, mean_rows=mean_rows, mean_cached=mean_cached, max_blocks=max_blocks,
                ended=ended, idle=idle)


def _rope(name, rows, q_heads, kv_heads, rotary, interleaved, bf16, first, base=10000.0, stretch=1.0, magnitude=1.0, transposed=False, fused=True):
    return dict(name=name, kind="rope", rows=rows, q_heads=q_heads, kv_heads=kv_heads, rotary=rotary, interleaved=interleaved, bf16=bf16,
                first=first, base=base, stretch=stretch, magnitude=magnitude, transposed=transposed, fused=fused)


def _append(name, requests, rows, q_heads, kv_heads, rotary, interleaved, bf16, first, padding=0, base=10000.0, magnitude=1.0):
    return dict(name=name, kind="append", requests=requests, rows=rows, q_heads=q_heads, kv_heads=kv_heads, rotary=rotary,
                interleaved=interleaved, bf16=bf16, first=first, padding=padding, base=base, magnitude=magnitude)


def _linear(name, rows, columns, channels, bf16, quantize):
    return dict(name=name, kind="linear", rows=rows, columns=columns, channels=channels, bf16=bf16, quantize=quantize)


def listed():
    return [
        # one decode step of a small batch: a token each, a page now and then
        _tables("tables_decode_16", 16, 1, 8192, 512),
        # a busy server's step: a thousand requests with prompts in chunks of very different lengths, some idle, some just ended
        _tables("tables_ragged_1000", 1000, 900, 3000, 64, ended=0.05, idle=0.1),
        # the rows of one verify tree far into a long context, with stretched frequencies as long-context models have them
        _rope("rope_60_128k", 60, 32, 2, 128, False, True, 131000, base=1000000.0, stretch=4.0, magnitude=1.1386),
        # a prompt of odd length in a model that rotates half of each head, pairs side by side, in the fused projection's output
        _rope("rope_8191_half_head", 8191, 32, 8, 64, True, False, 0),
        # gradients of a training chunk's queries and keys back through the rotation
        _rope("rope_back_2048", 2048, 32, 2, 128, False, True, 4096, transposed=True, fused=False),
        # a decode step of 64 requests: one row each, every row in a page of its own
        _append("append_decode_64", 64, 64, 32, 8, 128, False, False, 5000),
        # prompt chunks of seven requests in one launch, padded to a graph's size
        _append("append_ragged_8192", 7, 8000, 32, 2, 128, False, True, 1000, padding=192, magnitude=1.1386, base=1000000.0),
        # rows that come rotated: keys and values alone, odd count
        _append("append_plain_4001", 3, 4001, 0, 4, 0, False, False, 77),
        # one token's fused q/k/v projection
        _linear("linear_1_4608", 1, 4096, 4608, False, True),
        # the target head on a 60-node tree with an 8-bit weight
        _linear("linear_60_73448", 60, 4096, 73448, False, True),
        # odd everything, rows that are 8 bits already
        _linear("linear_333_odd", 333, 4099, 12289, True, False),
        # a prompt chunk through a wide projection
        _linear("linear_8192_16384", 8192, 4096, 16384, True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "append", "linear", "linear"])
    bf16 = rng.random() < 0.5
    if kind == "tables":
        requests = _log(rng, 1, 4096)
        mean = _log(rng, 1, max(1, min(8192, LARGEST_TABLE // requests // 2)))
        case = _tables("", requests, mean, _log(rng, 1, 20000), rng.choice([64, 128, 500]), rng.choice([0.0, 0.05, 0.3]), rng.choice([0.0, 0.1, 0.5]))
    elif kind == "rope":
        q_heads, kv_heads = rng.choice([(32, 2), (32, 4), (32, 8), (16, 16), (7, 1), (32, 0)])
        case = _rope("", _log(rng, 1, LARGEST_ROWS // (q_heads + kv_heads)), q_heads, kv_heads, rng.choice([128, 128, 64, 32, 96, 42]), rng.random() < 0.5, bf16,
                     _log(rng, 1, 1000000), base=rng.choice([10000.0, 500000.0, 1000000.0]), stretch=rng.choice([1.0, 4.0, 32.0]),
                     magnitude=rng.choice([1.0, 1.1386]), transposed=rng.random() < 0.3, fused=rng.random() < 0.5)
    elif kind == "append":
        q_heads, kv_heads = rng.choice([(32, 2), (32, 4), (32, 8), (16, 16), (0, 2), (0, 8)])
        rows = _log(rng, 1, LARGEST_ROWS // (q_heads + 2 * kv_heads))
        rotary = rng.choice([128, 128, 64, 96]) if q_heads else 0
        if rng.random() < 0.4:  # a decode step
            rows = requests = _log(rng, 1, 256)
        else:
            requests = rng.choice([1, min(rows, _log(rng, 1, 64))])
        case = _append("", requests, rows, q_heads, kv_heads, rotary, rng.random() < 0.5, bf16, _log(rng, 1, 1000000),
                       padding=rng.choice([0, 0, 5, 100]), base=rng.choice([10000.0, 1000000.0]), magnitude=rng.choice([1.0, 1.1386]))
    else:
        rows, columns = _log(rng, 1, 8192), _log(rng, 64, 16384)
        channels = min(_log(rng, 64, 73448), max(64, LARGEST_PRODUCT // (rows * columns)))
        case = _linear("", rows, columns, channels, bf16, rng.random() < 0.5)
    del case["name"]
    return case


class _Maker:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))
        self.host = np.random.Generator(np.random.Philox(key=[int(seed), 7]))

    def normal(self, *shape, bf16):
        return torch.empty(shape, dtype=torch.bfloat16 if bf16 else torch.float16, device="cuda").normal_(generator=self.gen)

    def int8(self, *shape):
        """Rounded normal values that use the range as a quantiser leaves them."""
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, 32.0, generator=self.gen).round_().clamp_(-127, 127).to(torch.int8)

    def uniform(self, lo, hi, *shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(lo, hi, generator=self.gen)


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _container(t):
    """A 16-bit tensor as the framework's calls take it: bfloat16 travels as its bit pattern."""
    return None if t is None else t.view(torch.float16)


def _frequencies(c):
    half = max(c["rotary"] // 2, 1)
    return (c["base"] ** (-np.arange(half) / half) / c.get("stretch", 1.0)).astype(np.float32)


# ---- tables: a batch's pages and slots ----

def _prepare_tables(c, seed):
    g = _Maker(seed).host
    B, M = c["requests"], c["max_blocks"]
    # the pool and the padded number of rows are the server's, whatever comes: a batch may use them up
    pages = 32 + 2 * (B * (c["mean_cached"] + c["mean_rows"]) // PAGE) + 3 * B + 2 * M
    max_rows = 64 * (1 + B * c["mean_rows"] * 5 // 4 // 64)
    cached = np.minimum(g.geometric(1.0 / c["mean_cached"], B), (M - 1) * PAGE)
    if (-(-cached // PAGE)).sum() > pages:
        cached = np.minimum(cached, pages // B * PAGE)
    new = g.geometric(1.0 / c["mean_rows"], B)
    new[g.random(B) < c["idle"]] = 0
    new = np.diff(np.minimum(np.concatenate([[0], np.minimum(new, M * PAGE - cached).cumsum()]), max_rows))
    new[g.random(B) < c["ended"]] = -1
    held = -(-cached // PAGE)
    order = g.permutation(pages).astype(np.int32)
    tables = np.zeros((B, M), np.int32)
    tables[np.arange(M)[None, :] < held[:, None]] = order[:held.sum()]
    stack = np.zeros(pages, np.int32)
    free = pages - int(held.sum())
    stack[:free] = order[held.sum():]
    put = lambda a: _device(a.astype(np.int32))  # noqa: E731
    return types.SimpleNamespace(kv_lens=put(cached), new_lens=put(new), held=put(held), tables=put(tables), stack=put(stack),
                                 counts=put(np.array([free, 0])), max_rows=max_rows, M=M, pages=pages,
                                 spare=torch.zeros(pages + 1, dtype=torch.int32, device="cuda"))


def _tables_plain(s):
    kv, new, M = s.kv_lens.long(), s.new_lens.long(), s.M
    ended, rows, held = new < 0, new.clamp(min=0), s.held.long().clamp(0, M)
    row_end = rows.cumsum(0)
    released = torch.where(ended, held, 0)
    released_end = released.cumsum(0)
    count = s.counts[0].long().clamp(0, s.pages)
    top = (count + released_end[-1]).clamp(max=s.pages)
    blocks = (kv + rows + PAGE - 1) // PAGE
    bad = ~ended & ((kv < 0) | (blocks > M) | ((rows > 0) & (row_end > s.max_rows)))
    need = torch.where(ended | bad, 0, (blocks - held).clamp(min=0))
    need_end = need.cumsum(0)
    refused = bad | ((need > 0) & (need_end > top))
    granted = ~ended & ~refused
    # pages given back go on the stack in request order, behind those that are free already (an entry of its own takes the rest)
    b = torch.arange(M, device=kv.device)[None, :]
    spot = torch.where(ended[:, None] & (b < held[:, None]), count + (released_end - released)[:, None] + b, s.pages).clamp(max=s.pages)
    spare = s.spare
    spare[:s.pages] = s.stack
    spare[spot.flatten()] = s.tables.flatten()
    s.stack.copy_(spare[:s.pages])
    # pages taken come off its top in request order
    fresh = granted[:, None] & (b >= held[:, None]) & (b < blocks[:, None])
    place = (top - 1 - (need_end - need)[:, None] - (b - held[:, None])).clamp(0, s.pages - 1)
    s.tables.copy_(torch.where(fresh, s.stack[place], s.tables))
    row = torch.arange(s.max_rows, device=kv.device)
    r = torch.searchsorted(row_end, row, right=True).clamp(max=kv.numel() - 1)
    inside = (row < row_end[-1]) & granted[r]
    at = kv[r] + row - (row_end - rows)[r]
    page = s.tables[r, (at // PAGE).clamp(0, M - 1)].long()
    taken = torch.where(granted, need, 0).sum()
    offsets = torch.cat([row_end.new_zeros(1), row_end]).clamp(max=s.max_rows)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return dict(kv_lens=i32(torch.where(granted, kv + rows, torch.where(ended, 0, kv))), held=i32(torch.where(granted, torch.maximum(held, blocks), torch.where(ended, 0, held))),
                counts=i32(torch.stack([top - taken, refused.sum()])), row_offsets=i32(offsets), positions=i32(torch.where(inside, at, -1)),
                slots=i32(torch.where(inside, page * PAGE + at % PAGE, -1)), block_tables=s.tables, free_pages=s.stack)


def _run_tables(s):
    if not own:
        return _tables_plain(s)
    from cpm.cu_amd import ops
    out = ops.batch_tables(s.kv_lens, s.new_lens, s.tables, s.held, s.stack, s.counts, s.max_rows)
    return dict(out, block_tables=s.tables, free_pages=s.stack)


def _exact_tables(c, seed):
    """The same by walking through the requests one by one."""
    s = _prepare_tables(c, seed)
    kv, new, held, tables, stack = (t.cpu().numpy().astype(np.int64) for t in (s.kv_lens, s.new_lens, s.held, s.tables, s.stack))
    count, B = int(s.counts[0]), len(kv)
    lens, held_out, offsets, refused = kv.copy(), held.copy(), [0], 0
    for r in range(B):
        if new[r] < 0:
            stack[count:count + held[r]] = tables[r, :held[r]]
            count, lens[r], held_out[r] = count + held[r], 0, 0
    positions, slots, dry, free = np.full(s.max_rows, -1), np.full(s.max_rows, -1), False, count
    for r in range(B):
        n = max(int(new[r]), 0)
        first = offsets[-1]
        offsets.append(min(first + n, s.max_rows))
        if new[r] < 0:
            continue
        blocks = -(-int(kv[r] + n) // PAGE)
        if blocks > s.M or (n and first + n > s.max_rows):
            refused += 1
            continue
        need = max(0, blocks - held[r])
        if need and (dry or need > free):
            dry, refused = True, refused + 1
            continue
        for b in range(held[r], blocks):
            free -= 1
            tables[r, b] = stack[free]
        lens[r], held_out[r] = kv[r] + n, max(held[r], blocks)
        at = kv[r] + np.arange(n)
        positions[first:first + n] = at
        slots[first:first + n] = tables[r, at // PAGE] * PAGE + at % PAGE
    put = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32))  # noqa: E731
    return dict(kv_lens=put(lens), held=put(held_out), counts=put([free, refused]), row_offsets=put(offsets), positions=put(positions),
                slots=put(slots), block_tables=put(tables), free_pages=put(stack))


# ---- rope: rotary positions ----

def _rows_in_hand(c, make, heads, n):
    """q and k rows (and v's) as views of the fused projection's output, or as tensors of their own."""
    if c.get("fused", True):
        x = make.normal(n, sum(heads) * HEAD_DIM, bf16=c["bf16"])
        at = np.cumsum([0] + list(heads)) * HEAD_DIM
        return [x[:, lo:hi].view(n, h, HEAD_DIM) if h else None for lo, hi, h in zip(at, at[1:], heads)]
    return [make.normal(n, h, HEAD_DIM, bf16=c["bf16"]) if h else None for h in heads]


def _prepare_rope(c, seed):
    make = _Maker(seed)
    n = c["rows"]
    q, k, _ = _rows_in_hand(c, make, (c["q_heads"], c["kv_heads"], c["kv_heads"]), n)
    first = c["first"] + int(make.host.integers(0, 64))
    # a tree's rows sit a few levels behind the prefix, a prompt's follow each other
    positions = first + (make.host.integers(0, 6, n) if n <= 128 else np.arange(n))
    out = [None if t is None else torch.zeros(t.shape, dtype=t.dtype, device="cuda") for t in (q, k)]
    return _with_containers(c, types.SimpleNamespace(c=c, q=q, k=k, q_out=out[0], k_out=out[1], positions=_device(positions.astype(np.int32)),
                                                     inv_freq=_device(_frequencies(c)), magnitude=c["magnitude"], interleaved=c["interleaved"]))


def _with_containers(c, s):
    s.own16 = types.SimpleNamespace(**{name: _container(getattr(s, name, None)) for name in ("q", "k", "v", "q_out", "k_out", "x", "out")})
    if own:  # the element type of the 16-bit tensors is set once by a program that uses the framework
        from cpm.cu_amd import lib
        lib.get().set_option(b"dtype", 1 if c["bf16"] else 0)
    return s


def _turned(x, cos, sin, interleaved):
    """x [n, heads, D] with its first 2 * cos.shape[-1] values of each head turned, in the type of cos."""
    r = 2 * cos.shape[-1]
    t = x[..., :r].to(cos.dtype)
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :r // 2], t[..., r // 2:])
    c, s = cos[:, None, :], sin[:, None, :]
    pair = (a * c - b * s, a * s + b * c)
    t = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([t, x[..., r:].to(cos.dtype)], -1)


def _cos_sin(s, transposed, dtype):
    angle = s.positions.double()[:, None] * s.inv_freq.double()[None, :]
    m = s.magnitude
    return (torch.cos(angle) * m).to(dtype), (torch.sin(angle) * (-m if transposed else m)).to(dtype)


def _run_rope(s):
    if own:
        from cpm.cu_amd import ops
        o = s.own16
        ops.rope_rows(o.q, o.k, s.positions, s.inv_freq, interleaved=s.interleaved, magnitude=s.magnitude, transposed=s.c["transposed"], q_out=o.q_out, k_out=o.k_out)
    else:
        cos, sin = _cos_sin(s, s.c["transposed"], torch.float32)
        s.q_out.copy_(_turned(s.q, cos, sin, s.interleaved))
        if s.k is not None:
            s.k_out.copy_(_turned(s.k, cos, sin, s.interleaved))
    return dict(q=s.q_out, k=s.k_out)


def _by_complex(x, s, transposed):
    """The rotation as a product of complex numbers in 64 bits."""
    r = 2 * s.inv_freq.numel()
    t = x[..., :r].double()
    z = torch.complex(t[..., 0::2].contiguous(), t[..., 1::2].contiguous()) if s.interleaved else torch.complex(t[..., :r // 2].contiguous(), t[..., r // 2:].contiguous())
    angle = s.positions.double()[:, None] * s.inv_freq.double()[None, :]
    turn = torch.polar(torch.full_like(angle, s.magnitude), -angle if transposed else angle)
    z = z * turn[:, None, :]
    t = torch.view_as_real(z).flatten(-2) if s.interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([t, x[..., r:].double()], -1)


def _exact_rope(c, seed):
    s = _prepare_rope(c, seed)
    return dict(q=_by_complex(s.q, s, c["transposed"]), k=None if s.k is None else _by_complex(s.k, s, c["transposed"]))


# ---- append: rows of several requests into the paged cache ----

def _prepare_append(c, seed):
    make = _Maker(seed)
    g, R, n = make.host, min(c["requests"], c["rows"]), c["rows"]
    cuts = np.sort(g.choice(n - 1, R - 1, replace=False) + 1) if R > 1 else np.zeros(0, np.int64)
    lengths = np.diff(np.concatenate([[0], cuts, [n]]))
    firsts = c["first"] + g.integers(0, 4 * PAGE, R)
    positions, blocks, base = [], [], 0
    for length, first in zip(lengths, firsts):
        at = first + np.arange(length)
        positions.append(at)
        blocks.append(base + at // PAGE - first // PAGE)
        base += int((first + length - 1) // PAGE - first // PAGE + 1)
    positions, blocks = np.concatenate(positions), np.concatenate(blocks)
    pages = n // PAGE + 2 * R + 2
    slots = g.permutation(pages)[blocks] * PAGE + positions % PAGE
    behind = np.full(c["padding"], -1)
    total = n + c["padding"]
    Hq, Hkv = c["q_heads"], c["kv_heads"]
    q, k, v = _rows_in_hand(c, make, (Hq, Hkv, Hkv), total)
    dtype = torch.bfloat16 if c["bf16"] else torch.float16
    # (the last page takes what the plain form writes for rows without a slot)
    pools = [make.normal(pages + 1, Hkv, *s, bf16=c["bf16"]) for s in ((PAGE, HEAD_DIM), (HEAD_DIM, PAGE))]
    s = types.SimpleNamespace(c=c, q=q, k=k, v=v, k_pool=pools[0], v_pool=pools[1], pages=pages, slots=_device(np.concatenate([slots, behind]).astype(np.int32)),
                              positions=_device(np.concatenate([positions, behind]).astype(np.int32)), q_out=torch.zeros((total, Hq, HEAD_DIM), dtype=dtype, device="cuda") if Hq else None,
                              inv_freq=_device(_frequencies(c)) if c["rotary"] else None, magnitude=c["magnitude"], interleaved=c["interleaved"])
    if own:
        from cpm.cu_amd.kvcache import PagedKVCache
        s.cache = PagedKVCache.from_pools([_container(s.k_pool[:pages])], [_container(s.v_pool[:pages])], torch.zeros(pages, dtype=torch.int32, device="cuda"))
    return _with_containers(c, s)


def _v_slot(t):
    """Where a page's dim rows keep token t: bits 2 and 3 of its number change places."""
    return (t & ~12) | ((t & 4) << 1) | ((t & 8) >> 1)


def _into_pools(s, k, v):
    at = torch.where(s.slots < 0, s.pages * PAGE, s.slots).long()
    page, slot = at // PAGE, at % PAGE
    s.k_pool[page, :, slot] = k
    s.v_pool[page, :, :, _v_slot(slot)] = v


def _run_append(s):
    if own:
        from cpm.cu_amd import ops
        o = s.own16
        ops.kv_append_slots(s.cache, 0, o.k, o.v, s.slots, q=o.q, q_out=o.q_out, positions=s.positions if s.inv_freq is not None else None,
                            inv_freq=s.inv_freq, interleaved=s.interleaved, magnitude=s.magnitude)
    else:
        k = s.k
        if s.inv_freq is not None:
            cos, sin = _cos_sin(s, False, torch.float32)
            k = _turned(s.k, cos, sin, s.interleaved).to(s.k.dtype)
            turned = _turned(s.q, cos, sin, s.interleaved).to(s.q.dtype)
            s.q_out.copy_(torch.where((s.positions < 0)[:, None, None], s.q_out, turned))
        _into_pools(s, k, s.v)
    return dict(q=s.q_out, k=s.k_pool[:s.pages], v=s.v_pool[:s.pages])


def _exact_append(c, seed):
    s = _prepare_append(c, seed)
    n = c["rows"]
    put = slice(0, n)
    slots = s.slots[put].long()
    k_pool, v_pool = s.k_pool[:s.pages].double(), s.v_pool[:s.pages].double()
    k, q = s.k.double(), None
    if s.inv_freq is not None:
        q = s.q_out.double()
        q[put] = _by_complex(s.q, s, False)[put]
        k = _by_complex(s.k, s, False)
    token_major = v_pool[..., _v_slot(torch.arange(PAGE, device="cuda"))].permute(0, 3, 1, 2).reshape(s.pages * PAGE, -1, HEAD_DIM).contiguous()
    token_major[slots] = s.v[put].double()
    rows = k_pool.permute(0, 2, 1, 3).reshape(s.pages * PAGE, -1, HEAD_DIM).contiguous()
    rows[slots] = k[put]
    k_pool = rows.view(s.pages, PAGE, -1, HEAD_DIM).permute(0, 2, 1, 3).contiguous()
    v_pool = token_major.view(s.pages, PAGE, -1, HEAD_DIM).permute(0, 2, 3, 1)[..., _v_slot(torch.arange(PAGE, device="cuda"))].contiguous()
    return dict(q=q, k=k_pool, v=v_pool)


# ---- linear: products in 8 bits ----

def _prepare_linear(c, seed):
    make = _Maker(seed)
    n, K, V = c["rows"], c["columns"], c["channels"]
    s = types.SimpleNamespace(c=c, K=K, w=make.int8(V, K), w_scales=make.uniform(0.2, 1.0, V) * 0.0003, x=None, xq=None, x_scales=None)
    if c["quantize"]:
        # hidden rows: a few channels much larger than the others
        loud = 1.0 + 9.0 * (make.uniform(0.0, 1.0, K) < 0.01).float()
        s.x = (make.normal(n, K, bf16=c["bf16"]).float() * loud).to(torch.bfloat16 if c["bf16"] else torch.float16)
    else:
        # rows that an earlier operator left in 8 bits: whole pieces of 64, zeros behind the last column
        s.xq = torch.zeros((n, -(-K // 64) * 64), dtype=torch.int8, device="cuda")
        s.xq[:, :K] = make.int8(n, K)
        s.x_scales = make.uniform(0.2, 1.0, n) * 0.05
    s.out = torch.zeros((n, V), dtype=torch.bfloat16 if c["bf16"] else torch.float16, device="cuda")
    if own:
        from cpm.cu_amd import ops
        s.weight = ops.Int8Weight(s.w, s.w_scales)
    return _with_containers(c, s)


def _run_linear(s):
    if own:
        from cpm.cu_amd import ops
        xq, scales = (s.xq, s.x_scales) if s.x is None else ops.quantize_rows(s.own16.x)
        ops.int8_linear(xq, scales, s.weight, out=s.own16.out)
        return s.out
    if s.x is None:
        x, scales = s.xq[:, :s.K].float(), s.x_scales
    else:
        x = s.x.float()
        largest = x.abs().amax(1)
        scales = largest / 127.0
        x = torch.where(largest[:, None] > 0, torch.round(x * 127.0 / largest[:, None]), 0.0)
    s.out.copy_(x @ s.w.float().t() * (scales[:, None] * s.w_scales[None, :]))
    return s.out


def _exact_linear(c, seed):
    s = _prepare_linear(c, seed)
    if s.x is None:
        x, scales = s.xq[:, :s.K].double(), s.x_scales.double()
    else:
        largest = s.x.double().abs().amax(1)
        scales, x = largest / 127.0, torch.round(s.x.double() * 127.0 / largest[:, None])
    y = torch.matmul(x, s.w.double().t().contiguous())
    return y * scales[:, None] * s.w_scales.double()[None, :]


_PREPARE = dict(tables=_prepare_tables, rope=_prepare_rope, append=_prepare_append, linear=_prepare_linear)
_RUN = dict(tables=_run_tables, rope=_run_rope, append=_run_append, linear=_run_linear)
_EXACT = dict(tables=_exact_tables, rope=_exact_rope, append=_exact_append, linear=_exact_linear)


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, seed)
    s.run = _RUN[case["kind"]]
    return s


def run(state):
    return state.run(state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


def work(case):
    c, kind = case, case["kind"]
    if kind == "tables":
        B, rows = c["requests"], c["requests"] * c["mean_rows"]
        # lengths and page counts in and out, offsets; a position and a slot for each row; an entry read and written for each page
        return dict(bytes=4 * 6 * B + 8 * rows + 8 * (rows // PAGE + c["ended"] * B * c["mean_cached"] / PAGE), flops=0)
    if kind == "rope":
        values = c["rows"] * (c["q_heads"] + c["kv_heads"]) * HEAD_DIM
        return dict(bytes=4 * values + 4 * c["rows"], flops=3 * values * c["rotary"] / HEAD_DIM)
    if kind == "append":
        values = c["rows"] * (c["q_heads"] + 2 * c["kv_heads"]) * HEAD_DIM
        return dict(bytes=4 * values + 8 * c["rows"], flops=3 * c["rows"] * (c["q_heads"] + c["kv_heads"]) * c["rotary"])
    n, K, V = c["rows"], c["columns"], c["channels"]
    return dict(bytes=n * K * (2 if c["quantize"] else 1) + V * K + 2 * n * V + 4 * (n + V), flops=2 * n * K * V)
