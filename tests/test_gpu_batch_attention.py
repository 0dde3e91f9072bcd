"""Attention of a batch's rows over its pages (prompts, chunks, single rows) on the GPU, against softmax sums in 64 bits.

Tolerance of a result o = sum p v / sum p, with A = sum p |v| / sum p of the same row and dim, h half a step of the type (2^-11 in fp16, 2^-8 in bf16) and N keys:
  h |o|                      the result's rounding,
  2 h A                      each probability is rounded by at most h of itself, in the numerator and in the sum it is divided by,
  2 (2^-21 + 2 ln 2 2^-24 |s| + 130 2^-24 S) A
                             its exponent: the power's own error, the rounding of the scaled score |s| and of its reference, and the score's sum of 128 products
                             of absolute sum S / scale in 32 bits; numerator and sum,
  2 (N / 8 + 64) 2^-24 A     two sums in 32 bits, eight products or more an addition,
  N 2^-25 max |v|            fp16 only: probabilities below 2^-14 are rounded by 2^-25 at most, and the largest is at least 1,
twice the last four, for second orders.
"""
import math

import numpy as np
import pytest

from cpm.cu_amd import synth

pytestmark = pytest.mark.gpu

PAGE, D = 256, 128
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}
SCALE = 1.0 / math.sqrt(D)


def _type(torch, dtype):
    return torch.bfloat16 if dtype else torch.float16


class Batch:
    """Requests of (cached, new) tokens: pools, tables, rows.  What nobody owns is `filler` (a number, or None for random values)."""

    def __init__(self, torch, seed, requests, Hq, Hkv, dtype=0, spread=1.0, filler=None, spare_pages=1, table_blocks=None):
        from cpm.cu_amd.kvcache import PagedKVCache, v_slot
        self.torch, self.dtype, self.requests, self.Hq, self.Hkv = torch, dtype, requests, Hq, Hkv
        g = synth.rng(seed, 400)
        self.g = g
        lengths = np.array([c + n for c, n in requests])
        held = -(-lengths // PAGE)
        pages = int(held.sum()) + spare_pages
        order = g.permutation(pages)
        M = max(int(held.max()), 1) if table_blocks is None else table_blocks
        tables = g.integers(0, pages, (len(requests), M))
        tables[np.arange(M)[None, :] < held[:, None]] = order[:held.sum()]
        gen = torch.Generator(device="cuda").manual_seed(seed)
        T = _type(torch, dtype)
        rand = lambda *s, std=1.0: torch.empty(s, dtype=T, device="cuda").normal_(0.0, std, generator=gen)  # noqa: E731
        self.rand = rand
        self.k, self.v = rand(pages, Hkv, PAGE, D), rand(pages, Hkv, D, PAGE)
        self.tables = torch.from_numpy(tables.astype(np.int32)).cuda()
        self.lengths = lengths
        if filler is not None:
            owned = torch.zeros((pages, PAGE), dtype=torch.bool, device="cuda")
            for r, L in enumerate(lengths):
                at = torch.arange(int(L), device="cuda")
                owned[self.tables[r].long()[at // PAGE], at % PAGE] = True
            self.k.masked_fill_(~owned[:, None, :, None], filler)
            slot = v_slot(torch.arange(PAGE, device="cuda"))
            owned_v = torch.zeros_like(owned)
            owned_v[:, slot] = owned
            self.v.masked_fill_(~owned_v[:, None, None, :], filler)
        new = np.array([n for _, n in requests])
        self.offsets = np.concatenate([[0], new.cumsum()])
        self.n = int(new.sum())
        self.q = rand(self.n, Hq, D, std=spread)
        self.positions = np.concatenate([c + np.arange(n) for c, n in requests]) if self.n else np.zeros(0, int)
        self.cache = PagedKVCache.from_pools([self.k.view(torch.float16)], [self.v.view(torch.float16)], self.tables[0])
        self.slot = v_slot(torch.arange(PAGE, device="cuda"))

    def dev(self, a):
        return self.torch.from_numpy(np.asarray(a).astype(np.int32)).cuda()

    def keys(self, r, g, upto=None):
        """K and V of request r's tokens on a KV head, [L, 128] in 64 bits."""
        at = self.torch.arange(int(self.lengths[r]) if upto is None else upto, device="cuda")
        page = self.tables[r].long()[at // PAGE]
        return self.k[page, g, at % PAGE].double(), self.v[page, g, :, self.slot[at % PAGE]].double()

    def expect(self, q=None, scale=SCALE, skip=()):
        """(results, limits) [n, Hq, 128] in 64 bits."""
        torch = self.torch
        q = self.q if q is None else q
        ref = torch.zeros((self.n, self.Hq, D), dtype=torch.float64, device="cuda")
        lim = torch.zeros_like(ref)
        h = HALF_STEP[self.dtype]
        for r, (cached, n) in enumerate(self.requests):
            if n == 0 or r in skip:
                continue
            lo = int(self.offsets[r])
            for g in range(self.Hkv):
                k, v = self.keys(r, g)
                N = k.shape[0]
                seen = torch.arange(N, device="cuda")[None, :] <= (cached + torch.arange(n, device="cuda"))[:, None]
                for head in range(g * self.Hq // self.Hkv, (g + 1) * self.Hq // self.Hkv):
                    x = q[lo:lo + n, head].double()
                    s = torch.where(seen, (x @ k.t().contiguous()) * scale, -math.inf)
                    S = torch.where(seen, (x.abs() @ k.abs().t().contiguous()) * scale, 0.0).amax(1, keepdim=True)
                    big = torch.where(seen, s.abs(), 0.0).amax(1, keepdim=True)
                    p = torch.exp(s - s.amax(1, keepdim=True))
                    total = p.sum(1, keepdim=True)
                    o, A = (p @ v) / total, (p @ v.abs()) / total
                    ref[lo:lo + n, head] = o
                    inner = 2 * h + 2 * (2.0 ** -21 + 2 * 0.7 * 2.0 ** -24 * big + 130 * 2.0 ** -24 * S) + 2 * (N / 8 + 64) * 2.0 ** -24
                    tiny = N * 2.0 ** -25 * v.abs().max() if self.dtype == 0 else 0.0
                    lim[lo:lo + n, head] = h * o.abs() + 2.0 ** -25 + 2 * (inner * A + tiny)
        return ref, lim

    def run(self, kind="prompt", q=None, out=None, positions=None, offsets=None, scale=None):
        from cpm.cu_amd import ops
        torch = self.torch
        f16 = lambda t: t.view(torch.float16)  # noqa: E731
        q = self.q if q is None else q
        out = torch.full((q.shape[0], self.Hq, D), 7.0, dtype=q.dtype, device="cuda") if out is None else out
        positions = self.dev(self.positions if positions is None else positions)
        offsets = self.dev(self.offsets if offsets is None else offsets)
        if kind == "prompt":
            ops.prompt_attention(f16(q), self.cache, 0, self.tables, offsets, positions, scale=scale, out=f16(out))
        else:
            ops.decode_attention(f16(q), self.cache, 0, self.tables, positions, row_offsets=offsets, scale=scale, out=f16(out))
        torch.cuda.synchronize()
        return out

    def check(self, out, expect=None):
        ref, lim = self.expect() if expect is None else expect
        over = ((out.double() - ref).abs() - lim)
        worst = float(over.max()) if over.numel() else -1.0
        assert worst <= 0 and bool(self.torch.isfinite(out.float()).all()), "off by %.3g more than the roundings allow, at %s" % (worst, np.unravel_index(int(over.argmax()), tuple(over.shape)))


HEADS = [(32, 2), (7, 1), (16, 16), (14, 2), (32, 8)]
PROMPTS = [
    [(0, 1)], [(0, 2)], [(0, 63)], [(0, 64)], [(0, 65)], [(0, 255)], [(0, 257)], [(63, 1)], [(64, 1)], [(255, 2)], [(256, 1)],
    [(0, 65), (3, 1), (255, 1), (256, 2), (0, 1)], [(0, 300), (0, 0), (700, 37), (12, 0), (1, 130)], [(1000, 1)] * 9,
]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("requests", PROMPTS, ids=lambda r: "_".join("%d+%d" % x for x in r[:4]))
def test_prompt_attention(gpu, set_option, dtype, heads, requests):
    set_option("dtype", dtype)
    b = Batch(gpu, 1, requests, *heads, dtype=dtype, spread=1.5, filler=float("nan"))
    b.check(b.run())


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads, requests", [
    ((32, 2), [(0, 2100)]), ((8, 8), [(0, 1500), (100, 3)]), ((32, 2), [(20000, 5)]), ((32, 2), [(9001, 40), (50000, 1), (3, 1), (17000, 129)]), ((4, 1), [(30011, 64)]),
    ((16, 16), [(4097, 300)]), ((64, 1), [(12000, 9)])], ids=str)
def test_prompt_attention_of_long_ones(gpu, set_option, dtype, heads, requests):
    """Several tiles of rows, and keys that are cut into pieces."""
    set_option("dtype", dtype)
    b = Batch(gpu, 2, requests, *heads, dtype=dtype, spread=1.2, filler=float("inf"))
    b.check(b.run())


DECODES = [[0], [1], [62], [63], [64], [65], [255], [256], [0, 1, 2, 3], [700, 5, 64, 127, 128, 2000, 0], [3000], [12345], [300] * 70]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads", HEADS + [(32, 1), (17, 1)], ids=str)
@pytest.mark.parametrize("cached", DECODES, ids=lambda c: "_".join(map(str, c[:4])) + "x%d" % len(c))
def test_decode_attention(gpu, set_option, dtype, heads, cached):
    set_option("dtype", dtype)
    b = Batch(gpu, 3, [(c, 1) for c in cached], *heads, dtype=dtype, spread=1.5, filler=float("nan"), table_blocks=max(8, max(cached) // PAGE + 1))
    expect = b.expect()
    b.check(b.run("decode"), expect)
    if max(cached) < 4 * PAGE:
        b.tables = b.tables[:, :max(cached) // PAGE + 1].contiguous()
        b.check(b.run("decode"), expect)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads, cached", [((32, 2), [100000]), ((32, 8), [40000, 3, 17, 26000, 900]), ((16, 16), [9000] * 3), ((32, 4), list(range(0, 6000, 37)))], ids=["one", "ragged", "mha", "many"])
def test_decode_attention_of_long_ones(gpu, set_option, dtype, heads, cached):
    set_option("dtype", dtype)
    b = Batch(gpu, 4, [(c, 1) for c in cached], *heads, dtype=dtype, spread=1.2, filler=float("-inf"))
    b.check(b.run("decode"))


def test_decode_attention_without_offsets(gpu):
    from cpm.cu_amd import ops
    b = Batch(gpu, 5, [(c, 1) for c in (5, 1000, 64)], 32, 2)
    b.check(ops.decode_attention(b.q, b.cache, 0, b.tables, b.dev(b.positions)))


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_rows_left_out_stay_as_they_were(gpu, kind):
    torch = gpu
    requests = [(40, 1), (0, 0), (300, 1), (7, 1), (500, 1)] if kind == "decode" else [(40, 3), (0, 0), (300, 70), (7, 1), (500, 20)]
    b = Batch(torch, 6, requests, 32, 2)
    positions = b.positions.copy()
    lo, hi = b.offsets[2], b.offsets[3]
    positions[lo:hi] = -1  # refused
    extra = 5
    q = torch.cat([b.q, b.rand(extra, 32, D)])
    out = torch.full((b.n + extra, 32, D), 7.0, dtype=torch.float16, device="cuda")
    b.run(kind, q=q, out=out, positions=np.concatenate([positions, [-1] * extra]))
    assert bool((out[lo:hi] == 7.0).all()) and bool((out[b.n:] == 7.0).all())
    ref, lim = b.expect(skip=(2,))
    keep = torch.ones(b.n, dtype=torch.bool, device="cuda")
    keep[lo:hi] = False
    assert bool(((out[:b.n].double() - ref).abs() <= lim)[keep].all())


def test_decode_attention_leaves_out_requests_of_several_rows(gpu):
    torch = gpu
    b = Batch(torch, 7, [(40, 1), (10, 3), (300, 1)], 14, 2)
    out = b.run("decode")
    assert bool((out[1:4] == 7.0).all())
    ref, lim = b.expect(skip=(1,))
    assert bool(((out.double() - ref).abs() <= lim)[[0, 4]].all())


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_rows_behind_the_tables_are_left_out(gpu, kind):
    """Positions from max_blocks * 256 on have no pages."""
    torch = gpu
    new = 1 if kind == "decode" else 40
    b = Batch(torch, 8, [(200, new), (PAGE * 2 - 20 if kind == "prompt" else PAGE * 2, new), (5, new)], 32, 2, table_blocks=3)
    b.tables = b.tables[:, :2].contiguous()
    out = b.run(kind)
    lo, hi = int(b.offsets[1]) + (20 if kind == "prompt" else 0), int(b.offsets[2])
    assert bool((out[lo:hi] == 7.0).all())
    b2 = Batch(torch, 8, [(200, new), (PAGE * 2 - 20 if kind == "prompt" else PAGE * 2, new), (5, new)], 32, 2, table_blocks=3)
    ref, lim = b2.expect()
    ok = (out.double() - ref).abs() <= lim
    assert bool(ok[:lo].all()) and bool(ok[hi:].all())


@pytest.mark.parametrize("kind", ["prompt", "decode"])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_of_a_fused_projection(gpu, kind, in_place):
    """q and out as parts of wider rows; out in q's place, or beside it in the same rows."""
    torch = gpu
    Hq, Hkv = 32, 8
    b = Batch(torch, 9, [(77, 1), (1000, 1), (5000, 1)] if kind == "decode" else [(0, 100), (5000, 3), (64, 64)], Hq, Hkv)
    wide = b.rand(b.n, 2 * Hq + Hkv, D)
    wide[:, Hkv:Hkv + Hq] = b.q
    before = wide.clone()
    q = wide[:, Hkv:Hkv + Hq]
    out = q if in_place else wide[:, Hkv + Hq:]
    expect = b.expect()
    b.run(kind, q=q, out=out)
    b.check(out.contiguous(), expect)
    assert torch.equal(wide[:, :Hkv], before[:, :Hkv])
    other = wide[:, Hkv + Hq:] if in_place else wide[:, Hkv:Hkv + Hq]
    assert torch.equal(other, before[:, Hkv + Hq:] if in_place else before[:, Hkv:Hkv + Hq])


def test_what_a_row_does_not_see_does_not_reach_it(gpu):
    """Infinities and NaN in the keys and values of later rows, in a tile that earlier rows are in: theirs are unchanged, to the bit; the later rows have what the formula gives."""
    torch = gpu
    for dtype_heads in ((32, 2), (4, 4)):
        b = Batch(torch, 10, [(100, 90), (0, 33)], *dtype_heads)
        clean = b.run().clone()
        Hkv = dtype_heads[1]
        for r, at, value, dim in ((0, 150, float("inf"), 5), (0, 170, float("nan"), 127), (0, 171, float("-inf"), 5), (1, 9, float("inf"), 64)):
            page = int(b.tables[r, at // PAGE])
            b.v[page, :, dim, int(b.slot[at % PAGE])] = value
        page = int(b.tables[1, 0])
        b.k[page, :, 20, 3] = float("nan")
        out = b.run()
        first = {0: 150 - 100, 1: 9}
        for r, (cached, n) in enumerate(b.requests):
            lo = int(b.offsets[r])
            assert torch.equal(out[lo:lo + first[r]], clean[lo:lo + first[r]])
        a, c = out[:90].float(), out[90:].float()
        seen = clean[:90].float()
        assert bool((a[50:71, :, 5] == float("inf")).all()) and bool(a[71:, :, 5].isnan().all()) and bool(a[70:, :, 127].isnan().all())
        rest = [d for d in range(D) if d not in (5, 127)]
        assert torch.equal(a[:, :, rest], seen[:, :, rest])
        assert bool((c[9:20, :, 64] == float("inf")).all()) and bool(c[20:].isnan().all()) and Hkv
        assert torch.equal(c[:20, :, :64], clean[90:110].float()[:, :, :64])


@pytest.mark.parametrize("dtype", [0, 1])
def test_scores_that_grow_along_the_keys(gpu, set_option, dtype):
    """The reference of the softmax has to follow, and to leave what came before behind: scores from -60 to 60 over the keys, up and down."""
    torch = gpu
    set_option("dtype", dtype)
    for sign in (1.0, -1.0):
        for kind, requests in (("prompt", [(0, 400), (3000, 2)]), ("decode", [(399, 1), (3000, 1)])):
            b = Batch(torch, 11, requests, 32, 2, dtype=dtype)
            b.q[:, :, 0] = sign * 16.0
            for r, L in enumerate(b.lengths):
                at = torch.arange(int(L), device="cuda")
                ramp = (at / (int(L) - 1) * 2 - 1) * 42.0
                b.k[b.tables[r].long()[at // PAGE], :, at % PAGE, 0] = ramp[:, None].to(b.k.dtype)
            b.check(b.run(kind))


@pytest.mark.parametrize("kind", ["prompt", "decode"])
@pytest.mark.parametrize("blocks", [2, 4, 5])
def test_columns_of_wider_tables(gpu, kind, blocks):
    """The first columns of tables that have more, as a server's have (up to 4 of them a decoding step has another kernel)."""
    b = Batch(gpu, 19, [(200, 1), (PAGE * (blocks - 1) + 70, 1), (5, 1)], 32, 2, table_blocks=40, filler=float("nan"))
    b.tables = b.tables[:, :blocks]
    b.check(b.run(kind))


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_a_given_scale(gpu, kind):
    b = Batch(gpu, 12, [(300, 1), (64, 1)], 32, 2)
    b.check(b.run(kind, scale=0.31), b.expect(scale=0.31))


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_far_into_a_large_pool(gpu, kind):
    """Pages that begin beyond 4 GiB of each pool."""
    torch = gpu
    Hkv, pages = 16, 4500
    b = Batch(torch, 13, [(600, 1), (20, 1)] if kind == "decode" else [(600, 20), (0, 40)], 16, Hkv)
    big_k = torch.zeros((pages, Hkv, PAGE, D), dtype=torch.float16, device="cuda")
    big_v = torch.zeros((pages, Hkv, D, PAGE), dtype=torch.float16, device="cuda")
    own = b.k.shape[0]
    big_k[pages - own:], big_v[pages - own:] = b.k, b.v
    b.k, b.v, b.tables = big_k, big_v, b.tables + (pages - own)
    b.cache.k, b.cache.v, b.cache.num_pages = [big_k], [big_v], pages
    b.check(b.run(kind))


def test_many_requests(gpu):
    torch = gpu
    g = synth.rng(14, 1)
    cached = [int(x) for x in g.integers(0, 500, 4096)]
    b = Batch(torch, 14, [(c, 1) for c in cached], 2, 1)
    expect = b.expect()
    b.check(b.run("decode"), expect)
    b.check(b.run("prompt"), expect)
    b = Batch(torch, 15, [(int(c), int(n)) for c, n in zip(g.integers(0, 300, 1500), g.integers(0, 9, 1500))], 8, 2)
    b.check(b.run("prompt"))


@pytest.mark.parametrize("requests", [[(0, 37)], [(3000, 40), (0, 0), (7, 1), (9000, 3)]], ids=["one", "cut"])
def test_wide_tables_give_the_same_bits(gpu, requests):
    """Tables of many columns allow for lengths at which the tiles are listed by a launch of their own."""
    torch = gpu
    b = Batch(torch, 17, requests, 32, 2)
    narrow = b.run()
    b.check(narrow)
    tables = torch.full((len(requests), 4096), -1, dtype=torch.int32, device="cuda")
    tables[:, :b.tables.shape[1]] = b.tables
    b.tables = tables
    assert torch.equal(b.run().view(torch.int16), narrow.view(torch.int16))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads, count", [((32, 2), 300), ((32, 8), 70), ((4, 1), 1500), ((34, 2), 200)], ids=str)
def test_short_requests_in_wide_tables(gpu, set_option, dtype, heads, count):
    """Many of them are taken whole, as in narrow tables; some have no row, one has two."""
    torch = gpu
    set_option("dtype", dtype)
    g = synth.rng(18, count)
    requests = [(int(c), 0 if i % 17 == 5 else 2 if i == 9 else 1) for i, c in enumerate(g.integers(0, 1023, count))]
    b = Batch(torch, 18, requests, *heads, dtype=dtype, filler=float("nan"), table_blocks=50)
    out = b.run("decode")
    two = int(b.offsets[9])
    assert bool((out[two:two + 2] == 7.0).all())
    ref, lim = b.expect()
    ref[two:two + 2], lim[two:two + 2] = 7.0, 0.0
    b.check(out, (ref, lim))
    assert torch.equal(b.run("decode").view(torch.int16), out.view(torch.int16))


def test_prompt_decode_and_tree_attention_agree(gpu):
    from cpm.cu_amd import ops
    torch = gpu
    b = Batch(torch, 16, [(900, 1)], 32, 2)
    ref, lim = b.expect()
    for out in (b.run("prompt"), b.run("decode"), ops.tree_attention(b.q, b.cache, 0, b.dev([901]), 1024)):
        assert bool(((out.double() - ref).abs() <= lim).all())


def test_pages_outside_the_pool_are_read_inside_it(gpu):
    """A table's number that is no page's: the nearest one, for both operators; nothing outside the pool is touched."""
    torch = gpu
    for kind, requests in (("prompt", [(300, 5)]), ("decode", [(300, 1)])):
        b = Batch(torch, 17, requests, 32, 2)
        last = b.k.shape[0] - 1
        b.tables = b.dev([[-5, 1 << 30]])
        out = b.run(kind)
        b.tables = b.dev([[0, last]])
        assert torch.equal(out, b.run(kind))


def test_no_rows(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    b = Batch(torch, 18, [(30, 1)], 32, 2)
    empty = torch.empty((0, 32, D), dtype=torch.float16, device="cuda")
    assert ops.prompt_attention(empty, b.cache, 0, b.tables, b.dev([0, 0]), b.dev([])).shape == (0, 32, D)
    assert ops.decode_attention(empty, b.cache, 0, b.tables, b.dev([]), row_offsets=b.dev([0, 0])).shape == (0, 32, D)
    for kind in ("prompt", "decode"):  # a step in which nobody has a row
        assert bool((b.run(kind, offsets=[0, 0], positions=[-1]) == 7.0).all())


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_in_a_graph_with_other_lengths(gpu, kind):
    """One captured call, replayed with other offsets, positions and tables."""
    torch = gpu
    from cpm.cu_amd import ops
    if kind == "decode":
        steps = [[(500, 1), (3, 1), (4000, 1)], [(501, 1), (0, 0), (30, 1)], [(1, 1), (2, 1), (9000, 1)], [(0, 0), (0, 0), (64, 1)]]
    else:
        steps = [[(0, 300), (20, 1), (9000, 7)], [(300, 10), (0, 500), (0, 0)], [(0, 1), (0, 1), (0, 1)], [(8000, 200), (8000, 200), (8000, 101)]]
    rows, M = 512 if kind == "prompt" else 3, 40
    batches = [Batch(torch, 20 + i, s, 32, 2, table_blocks=M) for i, s in enumerate(steps)]
    pages = max(b.k.shape[0] for b in batches)
    k = torch.zeros((pages, 2, PAGE, D), dtype=torch.float16, device="cuda")
    v = torch.zeros((pages, 2, D, PAGE), dtype=torch.float16, device="cuda")
    from cpm.cu_amd.kvcache import PagedKVCache
    tables = torch.zeros((3, M), dtype=torch.int32, device="cuda")
    cache = PagedKVCache.from_pools([k], [v], tables[0])
    q, out = torch.zeros((rows, 32, D), dtype=torch.float16, device="cuda"), torch.zeros((rows, 32, D), dtype=torch.float16, device="cuda")
    offsets, positions = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.full((rows,), -1, dtype=torch.int32, device="cuda")

    def call():
        if kind == "prompt":
            ops.prompt_attention(q, cache, 0, tables, offsets, positions, out=out)
        else:
            ops.decode_attention(q, cache, 0, tables, positions, row_offsets=offsets, out=out)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for turn in range(2):
        for b in batches:
            k[:b.k.shape[0]].copy_(b.k)
            v[:b.v.shape[0]].copy_(b.v)
            tables.copy_(b.tables)
            offsets.copy_(b.dev(b.offsets))
            positions.fill_(-1)
            positions[:b.n] = b.dev(b.positions)
            q[:b.n] = b.q
            out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert bool((out[b.n:] == 7.0).all())
            if turn == 0:
                b.check(out[:b.n])
                b.first = out[:b.n].clone()
            else:
                assert torch.equal(out[:b.n], b.first)  # (and the same bits again)


def test_two_graphs_and_eager_calls_side_by_side(gpu):
    """Calls share no memory but their arguments: two captured calls on two streams, and eager ones of other sizes between them."""
    torch = gpu
    from cpm.cu_amd import ops
    jobs = [Batch(torch, 30, [(0, 700), (5000, 40)], 32, 2), Batch(torch, 31, [(12000, 1), (40, 1), (7000, 1)], 32, 8), Batch(torch, 32, [(20000, 3)], 16, 2)]
    kinds = ["prompt", "decode", "prompt"]
    alone = [b.run(kind).clone() for b, kind in zip(jobs, kinds)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    args = [(b.dev(b.offsets), b.dev(b.positions)) for b in jobs]

    def call(i, out):
        b, (offsets, positions) = jobs[i], args[i]
        if kinds[i] == "prompt":
            ops.prompt_attention(b.q, b.cache, 0, b.tables, offsets, positions, out=out)
        else:
            ops.decode_attention(b.q, b.cache, 0, b.tables, positions, row_offsets=offsets, out=out)
    for i in range(2):
        outs.append(torch.zeros_like(jobs[i].q))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            call(i, outs[i])
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        eager = torch.zeros_like(jobs[2].q)
        call(2, eager)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], alone[0]) and torch.equal(outs[1], alone[1]) and torch.equal(eager, alone[2])


def test_wrong_tensors_are_refused(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    b = Batch(torch, 33, [(30, 1), (5, 1)], 32, 2)
    off, pos = b.dev(b.offsets), b.dev(b.positions)
    bad = [
        dict(q=b.q.float()), dict(q=b.q[:, :, :64]), dict(q=b.q.transpose(1, 2)), dict(q=b.q[:1]), dict(tables=b.tables.long()), dict(tables=b.tables[:1]), dict(tables=b.tables[0]),
        dict(off=b.dev([0, 1])), dict(off=off.cpu()), dict(pos=pos.float()), dict(pos=pos[:1]), dict(out=torch.empty((2, 32, 64), dtype=torch.float16, device="cuda")),
        dict(out=torch.empty((2, 32, D), dtype=torch.float32, device="cuda")), dict(tables=b.tables.cpu()), dict(tables=b.tables.repeat(1, 4)[:, ::2])]
    for kw in bad:
        a = dict(q=b.q, tables=b.tables, off=off, pos=pos, out=None)
        a.update(kw)
        with pytest.raises(AssertionError):
            ops.prompt_attention(a["q"], b.cache, 0, a["tables"], a["off"], a["pos"], out=a["out"])
        with pytest.raises(AssertionError):
            ops.decode_attention(a["q"], b.cache, 0, a["tables"], a["pos"], row_offsets=a["off"], out=a["out"])
    with pytest.raises(ValueError, match="query heads"):
        ops.prompt_attention(b.q[:, :31].contiguous(), b.cache, 0, b.tables, off, pos)
    with pytest.raises(ValueError, match="16 bytes"):
        wide = torch.zeros((2, 32 * D + 4), dtype=torch.float16, device="cuda")
        ops.prompt_attention(wide[:, 4:].view(2, 32, D), b.cache, 0, b.tables, off, pos)
    with pytest.raises(ValueError, match="scale"):
        ops.decode_attention(b.q, b.cache, 0, b.tables, pos, scale=0.0)
    with pytest.raises(ValueError, match="need row_offsets"):
        ops.decode_attention(torch.cat([b.q, b.q]), b.cache, 0, b.tables, torch.cat([pos, pos]))


def test_a_batch_step_from_plan_to_tokens(gpu):
    """A plan, its appends, attention of everything at once, a head, penalties and a mask: two steps of three requests, prompts and then single rows."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    Hq, Hkv, V = 16, 2, 500
    gen = torch.Generator(device="cuda").manual_seed(40)
    rand = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda").normal_(generator=gen)  # noqa: E731
    cache = PagedKVCache(1, Hkv, 12, fill=float("nan"))
    batch = ops.PageBatch(cache, max_requests=3, max_blocks=6)
    head = rand(V, Hq * D) * 0.05
    texts = [[], [], []]
    kept = [(torch.zeros((0, Hkv, D), device="cuda"),) * 2 for _ in range(3)]
    for step, lens in enumerate(([300, 5, 129], [1, 1, 0], [1, 1, 1])):
        rows = 512 if step == 0 else 3
        single = step > 0
        where = batch.plan(torch.tensor(lens, dtype=torch.int32, device="cuda"), rows)
        q, k, v = rand(rows, Hq, D), rand(rows, Hkv, D), rand(rows, Hkv, D)
        ops.kv_append_slots(cache, 0, k, v, where["slots"])
        out = torch.zeros((rows, Hq, D), dtype=torch.float16, device="cuda")
        assert batch.attention(q, 0, where, single=single, out=out) is out
        n, first, last_rows, requests = sum(lens), 0, [], []
        for r, m in enumerate(lens):
            kept[r] = tuple(torch.cat([a, b[first:first + m].float()]) for a, b in zip(kept[r], (k, v)))
            if m:
                K, Vv = (x.double().repeat_interleave(Hq // Hkv, 1) for x in kept[r])
                x = q[first + m - 1].double()
                p = torch.softmax((K * x[None]).sum(-1) * SCALE, 0)
                ref = (p[:, :, None] * Vv).sum(0)
                A = (p[:, :, None] * Vv.abs()).sum(0)
                assert bool(((out[first + m - 1].double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2 * (2 * 2.0 ** -11 + 2.0 ** -15) * A + 2.0 ** -14).all())
                last_rows.append(first + m - 1)
                requests.append(r)
            first += m
        assert bool((out[n:] == 0).all())
        hidden = out[last_rows].reshape(len(last_rows), -1).contiguous()
        _, logits = ops.lm_head_argmax(hidden, head.contiguous(), want_logits=True)
        L = max(map(len, texts)) + 1
        tokens = torch.tensor([t + [-1] * (L - len(t)) for t in texts], dtype=torch.int32, device="cuda")
        lens_t = torch.tensor([len(t) for t in texts], dtype=torch.int32, device="cuda")
        allowed = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
        allowed[0, 0] = -2  # never token 0
        adjusted, ids = ops.adjust_logits(logits, torch.tensor([[1.5, 0.5, 0.25]] * 3, device="cuda"), tokens, lens_t, torch.tensor(requests, dtype=torch.int32, device="cuda"),
                                          allowed=allowed.expand(len(requests), -1))
        z = logits.float().cpu().numpy()
        for i, r in enumerate(requests):
            for t in set(texts[r]):
                z[i, t] = (z[i, t] / np.float32(1.5) if z[i, t] > 0 else z[i, t] * np.float32(1.5)) - np.float32(0.25) * np.float32(texts[r].count(t)) - np.float32(0.5)
            z[i, 0] = -np.inf
            want = int(np.argmax(z[i].astype(np.float16)))
            assert int(ids[i]) == want and np.array_equal(adjusted[i].cpu().numpy(), z[i].astype(np.float16))
            texts[r].append(want)
