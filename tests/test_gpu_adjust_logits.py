"""Penalties, biases, masks and the arg-max of adjusted logits on the GPU against numpy, operation by operation in 32 bits (the description names every rounding: results are
equal to the bit), and against the formula in 64 bits.

Tolerance against 64 bits: at most six roundings in 32 bits (2^-24 each, of at most the largest value on the way, M) and one to the type, h of the result.  A token
with b biases has b further roundings, of sums of at most the sum of their magnitudes each, which M contains: 6 + b of them in all."""
import numpy as np
import pytest

from cpm.cu_amd import synth

pytestmark = pytest.mark.gpu

F = np.float32


def _bits(torch, dtype, z):
    """float32 -> the type, as float32 again (rounded once)."""
    return torch.from_numpy(z).to(torch.bfloat16 if dtype else torch.float16).float().numpy()


def _adjust(z, real, penalties, texts, biases, allowed):
    """One row z [V] in the precision of `real`."""
    z = z.astype(real)
    if penalties is not None:
        rep, pres, freq = (real(x) for x in penalties)
        texts = texts[(texts >= 0) & (texts < len(z))]
        at, c = np.unique(texts, return_counts=True)
        with np.errstate(over="ignore", invalid="ignore"):
            again = np.where(z[at] > 0, z[at] / rep, z[at] * rep)
            z[at] = again - freq * c.astype(real) - pres
    if biases is not None:
        sums = {}
        for v, x in zip(*biases):
            if 0 <= v < len(z):
                sums[int(v)] = real(sums.get(int(v), real(0)) + real(x))
        add = np.zeros(len(z), real)
        for v, x in sums.items():
            add[v] = x
        z = z + add
    if allowed is not None:
        z[~allowed] = -np.inf
    return z


class Case:
    def __init__(self, torch, seed, n, V, R=None, L=0, nb=0, mask=False, tree=False, requests=False, dtype=0, lens=None):
        g = synth.rng(seed, 500)
        self.torch, self.dtype, self.n, self.V = torch, dtype, n, V
        self.R = 1 if tree else n if R is None else R
        z = _bits(torch, dtype, (g.standard_normal((n, V)) * 3).astype(F))
        self.z = z
        self.penalties = np.stack([g.uniform(1.0, 2.0, self.R), g.uniform(-0.5, 0.5, self.R), g.uniform(0.0, 0.3, self.R)], 1).astype(F)
        self.tokens = g.integers(-2, min(V + 2, 300), (self.R, L)).astype(np.int32)
        if L > 4:
            self.tokens[:, ::3] = g.integers(0, V, self.tokens[:, ::3].shape)
        self.lens = (g.integers(0, L + 1, self.R) if lens is None else np.full(self.R, lens)).astype(np.int32)
        self.requests = g.integers(-1, self.R + 1, n).astype(np.int32) if requests else None
        self.bias_ids = g.integers(-1, V + 1, (self.R, nb)).astype(np.int32) if nb else None
        self.bias_values = (g.standard_normal((self.R, nb)) * 4).astype(F) if nb else None
        self.allowed = g.random((n, V)) < g.choice([0.5, 0.01], n)[:, None] if mask else None
        self.way = self.draft_ids = None
        if tree:
            self.way = np.zeros((n, n), bool)
            for t in range(n):
                if t:
                    self.way[t] = self.way[g.integers(0, t)]
                self.way[t, t] = True
            self.draft_ids = g.integers(0, min(V, 40), n).astype(np.int32)

    def rows(self, real):
        out = []
        for t in range(self.n):
            r = (0 if self.R == 1 else t) if self.requests is None else int(self.requests[t])
            if not 0 <= r < self.R:
                r = -1
            text = self.tokens[r, :self.lens[r]] if r >= 0 else np.zeros(0, int)
            if self.way is not None:
                text = np.concatenate([text, self.draft_ids[self.way[t]]])
            out.append(_adjust(self.z[t], real, self.penalties[r] if r >= 0 else None, text, (self.bias_ids[r], self.bias_values[r]) if self.bias_ids is not None and r >= 0 else None,
                               None if self.allowed is None else self.allowed[t]))
        return np.stack(out)

    def args(self):
        torch = self.torch
        cu = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        allowed = mask = None
        if self.allowed is not None:
            W = -(-self.V // 32)
            padded = np.zeros((self.n, W * 32), bool)
            padded[:, :self.V] = self.allowed
            allowed = np.packbits(padded, axis=1, bitorder="little").view(np.int32)
        if self.way is not None:
            W = -(-self.n // 64)
            padded = np.zeros((self.n, W * 64), bool)
            padded[:, :self.n] = self.way
            mask = np.packbits(padded, axis=1, bitorder="little").view(np.int64)
        return dict(penalties=cu(self.penalties), tokens=cu(self.tokens), lens=cu(self.lens), requests=cu(self.requests), bias_ids=cu(self.bias_ids), bias_values=cu(self.bias_values),
                    allowed=cu(allowed), draft_ids=cu(self.draft_ids), tree_mask=cu(mask))

    def logits(self):
        return self.torch.from_numpy(self.z).to(self.torch.bfloat16 if self.dtype else self.torch.float16).cuda()

    def check(self, out, ids):
        got = out.float().cpu().numpy()
        want = _bits(self.torch, self.dtype, self.rows(F).astype(F))
        assert np.array_equal(got, want), "%d of %d differ, first at %s" % ((got != want).sum(), got.size, np.argwhere(got != want)[0])
        exact, h = self.rows(np.float64), 2.0 ** (-8 if self.dtype else -11)
        fine = np.isfinite(exact)
        M = np.abs(self.z).astype(np.float64) * 2 + 8 + np.abs(np.where(fine, exact, 0))
        steps = np.full(M.shape, 6)
        if self.bias_ids is not None:
            for t in range(self.n):
                r = (0 if self.R == 1 else t) if self.requests is None else int(self.requests[t])
                if 0 <= r < self.R:
                    used = (self.bias_ids[r] >= 0) & (self.bias_ids[r] < self.V)
                    np.add.at(M[t], self.bias_ids[r][used], np.abs(self.bias_values[r][used].astype(np.float64)))
                    np.add.at(steps[t], self.bias_ids[r][used], 1)
        assert (np.abs(got[fine] - exact[fine]) <= (h * np.abs(exact) + 2.0 ** -25 + steps * 2.0 ** -24 * M)[fine]).all() and np.array_equal(got[~fine], exact[~fine])
        if ids is not None:
            best = np.where(np.isneginf(want).all(1), -1, want.argmax(1))
            assert np.array_equal(ids.cpu().numpy(), best)


def _run(case, **kw):
    from cpm.cu_amd import ops
    torch = case.torch
    out, ids = ops.adjust_logits(case.logits().view(torch.float16), **dict(case.args(), **kw))
    torch.cuda.synchronize()
    return out.view(torch.bfloat16 if case.dtype else torch.float16), ids


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("V", [1, 7, 8, 31, 33, 4089, 4096, 4097, 8200, 73448])
@pytest.mark.parametrize("kw", [dict(n=1, L=9), dict(n=3, L=700, nb=5, mask=True), dict(n=9, R=4, L=40, nb=300, requests=True), dict(n=5, R=1, L=100, mask=True), dict(n=17, tree=True, L=60, nb=3, mask=True),
                                dict(n=2, mask=True), dict(n=2, nb=1024)], ids=["one", "each", "mapped", "shared", "tree", "mask", "biases"])
def test_adjust_logits(gpu, set_option, dtype, V, kw):
    set_option("dtype", dtype)
    case = Case(gpu, V, V=V, dtype=dtype, **kw)
    case.check(*_run(case))


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128])
def test_trees_of_every_size(gpu, n):
    case = Case(gpu, n, n=n, V=9001, tree=True, L=5000, nb=2)
    case.check(*_run(case))


@pytest.mark.parametrize("L", [4096, 4097, 8192, 8193])
@pytest.mark.parametrize("V", [40, 8191, 16385, 50001])
def test_slices_of_every_size(gpu, set_option, L, V):
    """What the text has room for decides how much of the vocabulary a workgroup takes."""
    set_option("dtype", L & 1)
    case = Case(gpu, L, n=4, V=V, R=3, L=L, nb=200, mask=True, requests=True, dtype=L & 1)
    case.check(*_run(case))


@pytest.mark.parametrize("kw", [dict(n=640, V=40003, R=1, L=3000, nb=40, mask=True), dict(n=127, V=131073, tree=True, L=9000, nb=5), dict(n=640, V=40003, R=1, nb=3)], ids=["text", "tree", "biases"])
@pytest.mark.parametrize("want_ids", [True, False])
def test_many_rows_of_one_text(gpu, set_option, kw, want_ids):
    """A workgroup has several rows, one behind the other, each beginning elsewhere on 16 bytes."""
    set_option("dtype", int(want_ids))
    case = Case(gpu, 8, dtype=int(want_ids), **kw)
    skip = {} if "L" in kw else dict(penalties=None, tokens=None, lens=None)
    if skip:
        case.penalties[:] = [1.0, 0.0, 0.0]
    out, ids = _run(case, want_ids=want_ids, **skip)
    case.check(out, ids)


def test_long_texts(gpu):
    case = Case(gpu, 1, n=3, V=5000, L=200000, lens=199999)
    case.check(*_run(case))


@pytest.mark.parametrize("lens", [0, -3, 50, 99])
def test_lengths_of_texts(gpu, lens):
    """Nothing counts of an empty text; lens beyond the places is all of them."""
    case = Case(gpu, 2, n=4, V=900, L=50, lens=lens)
    got = _run(case)
    case.lens = np.clip(case.lens, 0, 50)
    case.check(*got)


def test_a_bias_that_stands_several_times(gpu):
    """The values are added up in their order: 1e8 + 1 - 1e8 - 0.25 is -0.25 in 32 bits, and 1 only in another order."""
    case = Case(gpu, 3, n=1, V=100, nb=7)
    case.bias_ids[0] = [5, 5, 9, 5, 5, 9, 5]
    case.bias_values[0] = [1e8, 1.0, 3.0, -1e8, 1e-3, -1.0, -0.25]
    case.check(*_run(case))


def test_rows_with_nothing_left(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    V = 5000
    z = torch.zeros((4, V), dtype=torch.float16, device="cuda")
    allowed = torch.zeros((4, -(-V // 32)), dtype=torch.int32, device="cuda")
    allowed[1, 100] = 1 << 7
    z[1, 3] = float("nan")
    z[2] = float("nan")
    allowed[2] = -1
    z[3] = float("-inf")
    allowed[3] = -1
    z[3, 4000] = -65504.0
    out, ids = ops.adjust_logits(z, allowed=allowed)
    assert ids.tolist() == [-1, 3207, -1, 4000]
    assert bool((out[0] == float("-inf")).all()) and int((out[1] > float("-inf")).sum()) == 1 and bool(out[2].isnan().all())


def test_infinities_and_nan(gpu):
    """In masked places they do not matter; elsewhere a NaN is no candidate, and an infinity is the largest."""
    torch = gpu
    from cpm.cu_amd import ops
    z = torch.randn((3, 300), generator=torch.Generator().manual_seed(1)).half().cuda()
    z[0, 10], z[0, 20], z[0, 30] = float("nan"), float("inf"), 60000.0
    z[1, 10], z[1, 299] = float("inf"), float("inf")
    z[2, 0] = -0.0
    z[2, 1:] = torch.cat([torch.zeros(1), -torch.ones(298)]).half()
    allowed = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    allowed[0, 0] = ~((1 << 10) | (1 << 20))
    out, ids = ops.adjust_logits(z, penalties=torch.tensor([[0.5, 0.0, 0.0]] * 3, device="cuda"), tokens=torch.tensor([[30], [5], [7]], dtype=torch.int32, device="cuda"),
                                 lens=torch.ones(3, dtype=torch.int32, device="cuda"), allowed=allowed)
    assert ids.tolist() == [30, 10, 0]  # (60000 / 0.5 is beyond the type: an infinity; equal ones: the lowest; the zeros are equal)
    assert out[0, 10] == float("-inf") and out[0, 20] == float("-inf") and out[0, 30] == float("inf")


@pytest.mark.parametrize("offset, stride", [(0, 1000), (1, 1000), (3, 1003), (0, 1003)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_anywhere(gpu, offset, stride, in_place):
    """Rows on any 2 bytes, at any distance, the results in their place or somewhere else; what lies between the rows stays."""
    torch = gpu
    from cpm.cu_amd import ops
    n, V = 5, 997
    for tree in (False, True):
        case = Case(torch, 4, n=n, V=V, L=30, nb=4, mask=True, tree=tree)
        wide = torch.full((n * stride + 16,), 3.0, dtype=torch.float16, device="cuda")
        rows = wide[offset:offset + n * stride].view(n, stride)[:, :V]
        rows.copy_(case.logits())
        before = wide.clone()
        target = rows
        if not in_place:
            there = torch.full((n * 1001 + 16,), 4.0, dtype=torch.float16, device="cuda")
            target = there[2:2 + n * 1001].view(n, 1001)[:, :V]
        out, ids = ops.adjust_logits(rows, out=target, **case.args())
        assert out is target
        case.check(out, ids)
        if in_place:
            rows.copy_(before[offset:offset + n * stride].view(n, stride)[:, :V])
            assert torch.equal(wide, before)
        else:
            assert torch.equal(wide, before)
            target.fill_(4.0)
            assert bool((there == 4.0).all())


def test_one_mask_for_all_rows(gpu):
    torch = gpu
    case = Case(gpu, 5, n=6, V=700, L=5, mask=True)
    case.allowed[:] = case.allowed[0]
    mask = case.args()["allowed"][:1]
    case.check(*_run(case, allowed=mask.expand(6, -1)))
    wide = torch.full((6, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:25] = mask
    case.check(*_run(case, allowed=wide[:, 3:25]))


def test_without_ids_and_without_anything(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    case = Case(gpu, 6, n=3, V=5003, L=10)
    out, ids = _run(case, want_ids=False)
    assert ids is None
    case.check(out, None)
    z = case.logits()
    out, ids = ops.adjust_logits(z)
    assert torch.equal(out, z) and torch.equal(ids.long(), z.float().argmax(1))
    out, ids = ops.adjust_logits(z[:0])
    assert out.shape == (0, 5003) and ids.shape == (0,)


def test_in_a_graph(gpu):
    """Replayed with other logits, texts and masks, beside the same call on another stream."""
    torch = gpu
    from cpm.cu_amd import ops
    cases = [Case(gpu, 60 + i, n=60, V=20000, L=300, nb=3, mask=True, tree=True) for i in range(3)]
    z, a = cases[0].logits(), cases[0].args()
    out = torch.empty_like(z)
    ops.adjust_logits(z, out=out, **a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, ids = ops.adjust_logits(z, out=out, **a)
    side, other = torch.cuda.Stream(), Case(gpu, 70, n=200, V=7001, L=30)
    oz, oa = other.logits(), other.args()
    torch.cuda.synchronize()
    for case in cases * 2:
        z.copy_(case.logits())
        for name, t in case.args().items():
            if t is not None:
                a[name].copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = ops.adjust_logits(oz, **oa)
        torch.cuda.synchronize()
        case.check(out, ids)
        other.check(*beside)


def test_wrong_tensors_are_refused(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    case = Case(gpu, 7, n=4, V=100, L=10, nb=2, mask=True)
    z, good = case.logits(), case.args()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for kw in (dict(penalties=good["penalties"].double()), dict(penalties=good["penalties"][:, :2].contiguous()), dict(tokens=None), dict(lens=None), dict(lens=i32(3)), dict(tokens=good["tokens"].long()),
               dict(tokens=i32(3, 10)), dict(bias_ids=None), dict(bias_values=None), dict(bias_ids=i32(4, 3)), dict(allowed=i32(4, 3)), dict(allowed=i32(3, 4)), dict(allowed=good["allowed"].t()),
               dict(requests=i32(3)), dict(draft_ids=i32(4)), dict(tree_mask=torch.zeros((4, 1), dtype=torch.int64, device="cuda")), dict(penalties=good["penalties"].cpu()),
               dict(out=torch.empty((4, 99), dtype=torch.float16, device="cuda")), dict(out=z.float()), dict(penalties=None)):
        with pytest.raises(AssertionError):
            ops.adjust_logits(z, **dict(good, **kw))
    with pytest.raises(AssertionError):
        ops.adjust_logits(z.float(), **good)
    with pytest.raises(ValueError, match="need requests"):
        ops.adjust_logits(z[:3], **dict(good, allowed=None))
    with pytest.raises(ValueError, match="biases"):
        ops.adjust_logits(z, bias_ids=i32(4, 1025), bias_values=torch.zeros((4, 1025), device="cuda"))
    with pytest.raises(ValueError, match="one request"):
        ops.adjust_logits(z, **dict(good, draft_ids=i32(4), tree_mask=torch.zeros((4, 1), dtype=torch.int64, device="cuda")))
    with pytest.raises(ValueError, match="other logits"):
        wide = torch.zeros((5, 100), dtype=torch.float16, device="cuda")
        ops.adjust_logits(wide[:4], out=wide[1:])
