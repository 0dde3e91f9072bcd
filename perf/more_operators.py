"""The operators of a batch's step behind its paged cache, as cases that can be timed and compared.

  prompt    attention of the new rows of several requests, causal, grouped heads, over everything that their pages hold: whole
            prompts, chunks far into a context, single rows between them (``ops.prompt_attention``)
  decode    attention of one new row of each request over its pages (``ops.decode_attention``)
  logits    penalties for repeated tokens, biases and masks of a grammar on rows of logits, and their arg-max, for requests' rows or for
            the nodes of a draft tree (``ops.adjust_logits``)

With ``own`` false a pass computes the same in elementary torch operations in 32 bits; with ``own`` true it makes the framework's
calls.  Both take the same inputs: pools of pages, the requests' tables, and the positions that a plan of the batch gives.
"""
import math
import types

import numpy as np
import torch

own = False

PAGE, HEAD_DIM = 256, 128
LARGEST_PROMPT = 32 * 8192 * 4097   # query heads * rows * mean keys, and
LARGEST_DECODE = 1 << 21            # requests * longest * KV heads, and
LARGEST_LOGITS = 512 * 73448        # rows * vocabulary: what no drawn case exceeds


def _prompt(name, requests, rows, cached, q_heads, kv_heads, bf16, singles=0.0):
    return dict(name=name, kind="prompt", requests=requests, rows=rows, cached=cached, q_heads=q_heads, kv_heads=kv_heads, bf16=bf16, singles=singles)


def _decode(name, requests, longest, q_heads, kv_heads, bf16, ragged=True, idle=0.0):
    return dict(name=name, kind="decode", requests=requests, longest=longest, q_heads=q_heads, kv_heads=kv_heads, bf16=bf16, ragged=ragged, idle=idle)


def _logits(name, rows, vocabulary, history, bf16, biases=0, grammar=False, tree=False):
    return dict(name=name, kind="logits", rows=rows, vocabulary=vocabulary, history=history, bf16=bf16, biases=biases, grammar=grammar, tree=tree)


def listed():
    return [
        # a short question to an idle server
        _prompt("prompt_37", 1, 37, 0, 32, 2, False),
        # a long document in one piece
        _prompt("prompt_8192", 1, 8192, 0, 32, 2, False),
        # nine prompts of very different lengths in one launch, eight KV heads
        _prompt("prompt_ragged_9", 9, 6007, 0, 32, 8, True),
        # a step of chunked prefill: three chunks at tens of thousands of cached tokens, and thirteen requests' single rows between them
        _prompt("prompt_chunks_long", 16, 589, 24000, 32, 2, True, singles=0.8),
        # as many KV heads as query heads, odd length
        _prompt("prompt_mha_1777", 1, 1777, 300, 16, 16, False),
        # one user's next token at a short context: a chain of round trips
        _decode("decode_1_500", 1, 500, 32, 2, False, ragged=False),
        # one user's next token far into a book
        _decode("decode_1_131000", 1, 131000, 32, 2, True, ragged=False),
        # a server's step: requests of very different lengths, some of them idle
        _decode("decode_64_ragged", 64, 16000, 32, 8, True, idle=0.1),
        # many short conversations
        _decode("decode_200_short", 200, 900, 32, 2, False),
        # one request's next token with penalties
        _logits("logits_1", 1, 73448, 700, False),
        # a draft tree's nodes, each with the tokens on its way and a mask of its own
        _logits("logits_tree_60", 60, 73448, 20000, False, biases=8, grammar=True, tree=True),
        # a server's step, odd vocabulary
        _logits("logits_512_odd", 512, 73447, 1500, True, biases=40, grammar=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "logits"])
    bf16 = rng.random() < 0.5
    heads = rng.choice([(32, 2), (32, 4), (32, 8), (16, 16), (14, 2), (7, 1), (32, 1)])
    if kind == "prompt":
        rows = _log(rng, 1, 8192)
        requests = min(rows, _log(rng, 1, 40))
        room = LARGEST_PROMPT // (heads[0] * rows) - rows
        cached = min(_log(rng, 1, 100000), max(room, 0), (1 << 21) // (requests * heads[1])) if rng.random() < 0.6 else 0
        case = _prompt("", requests, rows, cached, *heads, bf16, singles=rng.choice([0.0, 0.0, 0.5]))
    elif kind == "decode":
        requests = _log(rng, 1, 256)
        longest = _log(rng, 1, max(1, min(131000, LARGEST_DECODE // (requests * heads[1]))))
        case = _decode("", requests, longest, *heads, bf16, ragged=rng.random() < 0.7, idle=rng.choice([0.0, 0.0, 0.2]))
    else:
        vocabulary = rng.choice([73448, 73448, 32768, _log(rng, 1000, 160000)])
        tree = rng.random() < 0.3
        rows = _log(rng, 1, min(128 if tree else 512, LARGEST_LOGITS // vocabulary))
        case = _logits("", rows, vocabulary, _log(rng, 1, 60000 if tree else max(1, 2000000 // rows)) if rng.random() < 0.9 else 0, bf16, biases=rng.choice([0, 1, 30, 300]),
                       grammar=rng.random() < 0.5, tree=tree)
    del case["name"]
    return case


class _Maker:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))
        self.host = np.random.Generator(np.random.Philox(key=[int(seed), 11]))

    def normal(self, *shape, bf16, std=1.0):
        return torch.empty(shape, dtype=torch.bfloat16 if bf16 else torch.float16, device="cuda").normal_(0.0, std, generator=self.gen)


def _device(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(dtype))).cuda()


def _container(t):
    """A 16-bit tensor as the framework's calls take it: bfloat16 travels as its bit pattern."""
    return None if t is None else t.view(torch.float16)


def _ready(c, s):
    if own:  # the element type of the 16-bit tensors is set once by a program that uses the framework
        from cpm.cu_amd import lib
        lib.get().set_option(b"dtype", 1 if c["bf16"] else 0)
    return s


# ---- attention: requests' pages and rows ----

def _paged(c, make, lengths, first_of, rows):
    """Pools that hold `lengths` tokens of each request, tables, and rows of queries that sharpen some of the scores."""
    held = -(-lengths // PAGE)
    pages = int(held.sum()) + 1
    order = make.host.permutation(pages)
    tables = np.zeros((len(lengths), max(1, int(held.max()))), np.int64)
    tables[np.arange(tables.shape[1])[None, :] < held[:, None]] = order[:held.sum()]
    Hq, Hkv, bf16 = c["q_heads"], c["kv_heads"], c["bf16"]
    s = types.SimpleNamespace(c=c, lengths=[int(x) for x in lengths], first_of=[int(x) for x in first_of], scale=1.0 / math.sqrt(HEAD_DIM),
                              k_pool=make.normal(pages, Hkv, PAGE, HEAD_DIM, bf16=bf16), v_pool=make.normal(pages, Hkv, HEAD_DIM, PAGE, bf16=bf16),
                              q=make.normal(rows, Hq, HEAD_DIM, bf16=bf16, std=1.5), tables=_device(tables))
    s.out = torch.zeros_like(s.q)
    s.row_offsets = _device(np.concatenate([first_of, [rows]]))
    if own:
        from cpm.cu_amd.kvcache import PagedKVCache
        s.cache = PagedKVCache.from_pools([_container(s.k_pool)], [_container(s.v_pool)], s.tables[0])
        s.own16 = types.SimpleNamespace(q=_container(s.q), out=_container(s.out))
    return s


def _v_slot(t):
    """Where a page's dim rows keep token t: bits 2 and 3 of its number change places."""
    return (t & ~12) | ((t & 4) << 1) | ((t & 8) >> 1)


def _prepare_prompt(c, seed):
    make = _Maker(seed)
    g, R, n = make.host, min(c["requests"], c["rows"]), c["rows"]
    new = np.ones(R, np.int64)
    many = np.flatnonzero(g.random(R) >= c["singles"])
    if len(many) == 0:
        many = np.array([R // 2])
    share = g.exponential(1.0, len(many)) + 0.05
    more = np.floor((n - R) * share / share.sum()).astype(np.int64)
    more[0] += n - R - more.sum()
    new[many] += more
    cached = np.zeros(R, np.int64) if not c["cached"] else np.maximum(1, (c["cached"] * g.uniform(0.5, 1.0, R)).astype(np.int64))
    s = _paged(c, make, cached + new, np.cumsum(new) - new, n)
    s.new = [int(x) for x in new]
    s.positions = _device(np.concatenate([p + np.arange(x) for p, x in zip(cached, new)]))
    return _ready(c, s)


def _run_prompt(s):
    if own:
        from cpm.cu_amd import ops
        ops.prompt_attention(s.own16.q, s.cache, 0, s.tables, s.row_offsets, s.positions, out=s.own16.out)
        return s.out
    Hkv = s.k_pool.shape[1]
    slot = _v_slot(torch.arange(PAGE, device="cuda"))
    for r, (first, n, L) in enumerate(zip(s.first_of, s.new, s.lengths)):
        pages = s.tables[r, :-(-L // PAGE)].long()
        k = s.k_pool[pages].permute(1, 0, 2, 3).reshape(Hkv, -1, HEAD_DIM)[:, :L].float()
        v = s.v_pool[pages][..., slot].permute(1, 0, 3, 2).reshape(Hkv, -1, HEAD_DIM)[:, :L].float()
        q = s.q[first:first + n].float().view(n, Hkv, -1, HEAD_DIM).transpose(0, 1).reshape(Hkv, -1, HEAD_DIM)
        x = torch.matmul(q, k.transpose(1, 2)).mul_(s.scale).view(Hkv, n, -1, L)
        hidden = torch.arange(L, device="cuda")[None, :] > s.positions[first:first + n, None]
        x.masked_fill_(hidden[None, :, None, :], -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True)).exp_()
        y = torch.matmul(x.view(Hkv, -1, L), v) / x.sum(-1).view(Hkv, -1, 1)
        s.out[first:first + n] = y.view(Hkv, n, -1, HEAD_DIM).transpose(0, 1).reshape(n, -1, HEAD_DIM)
    return s.out


def _prepare_decode(c, seed):
    make = _Maker(seed)
    g, R = make.host, c["requests"]
    lengths = np.full(R, c["longest"], np.int64)
    if c["ragged"]:
        lengths = np.maximum(1, np.exp(g.uniform(math.log(max(1.0, c["longest"] / 100)), math.log(c["longest"]), R)).astype(np.int64))
        lengths[g.integers(0, R)] = c["longest"]
    idle = g.random(R) < c["idle"]
    idle[0] = False
    first_of = np.cumsum(~idle) - ~idle
    rows = R  # a step of one size, whoever is idle: the rows behind the last one are left out
    s = _paged(c, make, lengths, first_of, rows)
    s.row_offsets = _device(np.concatenate([first_of, [R - idle.sum()]]))
    s.busy = _device(np.flatnonzero(~idle), np.int64)
    s.positions = _device(np.concatenate([lengths[~idle] - 1, np.full(int(idle.sum()), -1)]))
    return _ready(c, s)


def _run_decode(s):
    if own:
        from cpm.cu_amd import ops
        ops.decode_attention(s.own16.q, s.cache, 0, s.tables, s.positions, row_offsets=s.row_offsets, out=s.own16.out)
        return s.out
    Hkv, R = s.k_pool.shape[1], s.busy.numel()
    pages = s.tables[s.busy].long()
    k = s.k_pool[pages].float().transpose(1, 2).reshape(R, Hkv, -1, HEAD_DIM)
    v = s.v_pool[pages].float().permute(0, 2, 1, 4, 3)[:, :, :, _v_slot(torch.arange(PAGE, device="cuda"))].reshape(R, Hkv, -1, HEAD_DIM)
    q = s.q[:R].float().view(R, Hkv, -1, HEAD_DIM)
    x = torch.matmul(q, k.transpose(2, 3)) * s.scale
    hidden = torch.arange(k.shape[2], device="cuda")[None, :] > s.positions[:R, None]
    x.masked_fill_(hidden[:, None, None, :], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    y = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    s.out[:R] = y.view(R, -1, HEAD_DIM)
    return s.out


def _exact_attention(s, rows):
    """Row sets (request, first row, rows) with all keys in the order of their positions, head by head, in 64 bits."""
    out = s.out.double()
    group = s.q.shape[1] // s.k_pool.shape[1]
    slot = _v_slot(torch.arange(PAGE, device="cuda"))
    for r, first, n in rows:
        at = torch.arange(s.lengths[r], device="cuda")
        page = s.tables[r].long()[at // PAGE]
        seen = at[:, None] <= s.positions[first:first + n].long()[None, :]
        for g in range(s.k_pool.shape[1]):
            k = s.k_pool[page, g, at % PAGE].double()
            v = s.v_pool[page, g, :, slot[at % PAGE]].double()
            for h in range(g * group, (g + 1) * group):
                x = torch.mm(k, s.q[first:first + n, h].double().t().contiguous()) * s.scale  # [keys, rows]
                x = torch.where(seen, x, -math.inf)
                x = torch.exp(x - torch.logsumexp(x, 0, keepdim=True))
                out[first:first + n, h] = torch.mm(x.t().contiguous(), v)
    return out


# ---- logits: penalties, biases, masks ----

def _prepare_logits(c, seed):
    make = _Maker(seed)
    g, n, V, bf16 = make.host, c["rows"], c["vocabulary"], c["bf16"]
    R = 1 if c["tree"] else n
    L = max(1, 2 * c["history"])
    lens = np.minimum(L, g.integers(c["history"] // 2, c["history"] * 3 // 2 + 1, R)) if c["history"] else np.zeros(R, np.int64)
    # words come back: most of a text's tokens are among a few thousand
    often = g.permutation(V)[:max(1, min(V // 4, 3000))]
    tokens = np.where(g.random((R, L)) < 0.8, often[(g.random((R, L)) ** 3 * len(often)).astype(np.int64)], g.integers(0, V, (R, L)))
    s = types.SimpleNamespace(c=c, logits=make.normal(n, V, bf16=bf16, std=3.0), out=torch.zeros((n, V), dtype=torch.bfloat16 if bf16 else torch.float16, device="cuda"),
                              tokens=_device(tokens), lens=_device(lens), bias_ids=None, bias_values=None, allowed=None, draft_ids=None, tree_mask=None,
                              penalties=_device(np.stack([g.uniform(1.0, 1.3, R), g.uniform(0.0, 0.5, R), g.uniform(0.0, 0.3, R)], 1), np.float32))
    if c["biases"]:
        nb = min(c["biases"], V)
        s.bias_ids = _device(np.stack([g.choice(V, nb, replace=False) for _ in range(R)]))
        s.bias_values = _device(g.uniform(-5.0, 5.0, (R, nb)), np.float32)
    if c["grammar"]:
        # some places of a grammar allow nearly everything, others a handful of tokens
        share = np.where(g.random(n) < 0.5, 0.9, 0.001)[:, None]
        bits = torch.rand((n, -(-V // 32) * 32), device="cuda", generator=make.gen) < _device(share, np.float32)
        bits[torch.arange(n), torch.from_numpy(g.integers(0, V, n)).cuda()] = True
        word = (bits.view(n, -1, 32).long() << torch.arange(32, device="cuda")).sum(-1)
        s.allowed = torch.where(word >= 1 << 31, word - (1 << 32), word).int()
    if c["tree"]:
        parent = np.array([0] + [int(g.integers(max(0, t - 12), t)) for t in range(1, n)])
        way = np.zeros((n, n), bool)
        for t in range(n):
            way[t] = way[parent[t]]
            way[t, t] = True
        words = np.zeros((n, -(-n // 64)), np.uint64)
        for j in range(n):
            words[:, j // 64] |= way[:, j].astype(np.uint64) << np.uint64(j % 64)
        s.tree_mask = torch.from_numpy(words.view(np.int64)).cuda()
        s.way = torch.from_numpy(way).cuda()
        s.draft_ids = _device(np.where(g.random(n) < 0.5, often[g.integers(0, len(often), n)], g.integers(0, V, n)))
    s.own16 = types.SimpleNamespace(logits=_container(s.logits), out=_container(s.out))
    return _ready(c, s)


def _run_logits(s):
    if own:
        from cpm.cu_amd import ops
        _, ids = ops.adjust_logits(s.own16.logits, penalties=s.penalties, tokens=s.tokens, lens=s.lens, bias_ids=s.bias_ids, bias_values=s.bias_values,
                                   allowed=s.allowed, draft_ids=s.draft_ids, tree_mask=s.tree_mask, out=s.own16.out)
        return dict(logits=s.out, ids=ids)
    n, V = s.logits.shape
    R, L = s.tokens.shape
    inside = (torch.arange(L, device="cuda")[None, :] < s.lens[:, None]).float()
    count = torch.zeros((R, V), dtype=torch.float32, device="cuda").scatter_add_(1, s.tokens.long(), inside)
    if s.draft_ids is not None:
        count = count.expand(n, V).contiguous().scatter_add_(1, s.draft_ids.long()[None, :].expand(n, n).contiguous(), s.way.float())
    repetition, presence, frequency = s.penalties[:, 0:1], s.penalties[:, 1:2], s.penalties[:, 2:3]
    z = s.logits.float()
    again = torch.where(z > 0, z / repetition, z * repetition) - frequency * count - presence
    z = torch.where(count > 0, again, z)
    if s.bias_ids is not None:
        z = z + torch.zeros((R, V), dtype=torch.float32, device="cuda").scatter_add_(1, s.bias_ids.long(), s.bias_values)
    if s.allowed is not None:
        bit = (s.allowed[:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        z = z.masked_fill(bit.view(n, -1)[:, :V] == 0, -math.inf)
    s.out.copy_(z)
    best = s.out.float().amax(1, keepdim=True)
    at = torch.arange(V, dtype=torch.int32, device="cuda")
    return dict(logits=s.out, ids=torch.where(s.out == best, at, V).amin(1).to(torch.int32))


def _exact_logits(s):
    """Row by row, with the counts of its tokens."""
    n, V = s.logits.shape
    out = s.logits.cpu().double().numpy()
    tokens, lens, penalties = s.tokens.cpu().numpy(), s.lens.cpu().numpy(), s.penalties.cpu().double().numpy()
    bias_ids, bias_values, allowed = (None if t is None else t.cpu().numpy() for t in (s.bias_ids, s.bias_values, s.allowed))
    for t in range(n):
        r = 0 if s.c["tree"] else t
        used = tokens[r, :lens[r]]
        if s.c["tree"]:
            used = np.concatenate([used, s.draft_ids.cpu().numpy()[s.way[t].cpu().numpy()]])
        v, times = np.unique(used, return_counts=True)
        repetition, presence, frequency = penalties[r]
        z = out[t, v]
        out[t, v] = np.where(z > 0, z / repetition, z * repetition) - presence - frequency * times
        if bias_ids is not None:
            out[t, bias_ids[r]] += bias_values[r].astype(np.float64)
        if allowed is not None:
            out[t, np.unpackbits(allowed[t].view(np.uint8), bitorder="little")[:V] == 0] = -math.inf
    return dict(logits=torch.from_numpy(out), ids=None)


_PREPARE = dict(prompt=_prepare_prompt, decode=_prepare_decode, logits=_prepare_logits)
_RUN = dict(prompt=_run_prompt, decode=_run_decode, logits=_run_logits)


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, seed)
    s.run = _RUN[case["kind"]]
    return s


def run(state):
    return state.run(state)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "prompt":
        return _exact_attention(s, list(zip(range(len(s.new)), s.first_of, s.new)))
    if case["kind"] == "decode":
        return _exact_attention(s, [(int(r), row, 1) for row, r in enumerate(s.busy.cpu())])
    return _exact_logits(s)


def work(case):
    c, kind = case, case["kind"]
    if kind == "logits":
        n, V, R = c["rows"], c["vocabulary"], 1 if c["tree"] else c["rows"]
        return dict(bytes=4 * n * V + (n * V / 8 if c["grammar"] else 0) + 4 * R * c["history"] + 8 * R * c["biases"] + 4 * n, flops=0)
    row, token = 2 * 2 * c["q_heads"] * HEAD_DIM, 2 * 2 * c["kv_heads"] * HEAD_DIM
    if kind == "decode":
        # (the mean of lengths spread evenly over the logarithm of a factor of 100)
        keys = (c["requests"] * (0.99 / math.log(100.0) if c["ragged"] and c["requests"] > 1 else 1.0)) * c["longest"] * (1.0 - c["idle"])
        return dict(bytes=row * c["requests"] + token * keys, flops=4 * c["q_heads"] * HEAD_DIM * keys)
    requests, n, cached = min(c["requests"], c["rows"]), c["rows"], 0.75 * c["cached"]
    # (rows spread unevenly over the requests that have more than one: about twice the square of their mean)
    many = max(1.0, requests * (1.0 - c["singles"]))
    length = n if many <= 1 else 2 * n / many
    return dict(bytes=row * n + token * (requests * cached + n), flops=4 * c["q_heads"] * HEAD_DIM * n * (cached + length / 2))
