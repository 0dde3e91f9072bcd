"""Attention of a batch's rows where its running sums are delicate: keys whose scores are minus infinity, one key far above all others, and long requests of which
every tile has to count.

Tolerance: that of test_gpu_batch_attention.py, with its last term by what is rounded.  In fp16 a probability, relative to the row's largest and times 2^shift, is
rounded by 2^-25 at most where it is below 2^-14; the sum of the products is divided by the sum of all, `total` (1 at least):
  (number of probabilities below 2^(-14 - shift)) 2^(-25 - shift) max |v| / total
in the numerator, and no more than that through the sum it is divided by.  shift 0 holds for any reference that is not above the row's largest score.
"""
import math

import pytest

from test_gpu_batch_attention import D, HALF_STEP, PAGE, SCALE, Batch

pytestmark = pytest.mark.gpu


def _expect(b, hidden=lambda at: at < 0, shift=0):
    """Results, limits [n, Hq, 128], each tile's share of the probabilities [n, Hq, tiles] and the limit of a share of 1 [n, Hq], in 64 bits; hidden(positions): keys
    whose scores are minus infinity."""
    torch = b.torch
    ref = torch.zeros((b.n, b.Hq, D), dtype=torch.float64, device="cuda")
    lim, of_one = torch.zeros_like(ref), torch.zeros_like(ref[:, :, 0])
    share = torch.zeros((b.n, b.Hq, -(-int(b.lengths.max()) // 64)), dtype=torch.float64, device="cuda")
    h = HALF_STEP[b.dtype]
    for r, (cached, n) in enumerate(b.requests):
        lo = int(b.offsets[r])
        if n == 0:
            continue
        for g in range(b.Hkv):
            k, v = b.keys(r, g)
            k = torch.where(k.isfinite(), k, 0.0)
            N = k.shape[0]
            at = torch.arange(N, device="cuda")
            seen = (at[None, :] <= (cached + torch.arange(n, device="cuda"))[:, None]) & ~hidden(at)[None, :]
            for head in range(g * b.Hq // b.Hkv, (g + 1) * b.Hq // b.Hkv):
                x = b.q[lo:lo + n, head].double()
                s = torch.where(seen, (x @ k.t().contiguous()) * SCALE, -math.inf)
                S = torch.where(seen, (x.abs() @ k.abs().t().contiguous()) * SCALE, 0.0).amax(1, keepdim=True)
                big = torch.where(seen, s.abs(), 0.0).amax(1, keepdim=True)
                p = torch.exp(s - s.amax(1, keepdim=True))
                total = p.sum(1, keepdim=True)
                o, A = (p @ v) / total, (p @ v.abs()) / total
                ref[lo:lo + n, head] = o
                inner = 2 * h + 2 * (2.0 ** -21 + 2 * 0.7 * 2.0 ** -24 * big + 130 * 2.0 ** -24 * S) + 2 * (N / 8 + 64) * 2.0 ** -24
                few = (seen & (p < 2.0 ** (-14 - shift))).sum(1, keepdim=True)
                tiny = few * 2.0 ** (-25 - shift) / total if b.dtype == 0 else torch.zeros_like(total)
                lim[lo:lo + n, head] = h * o.abs() + 2.0 ** -25 + 2 * (inner * A + tiny * v.abs().max())
                of_one[lo:lo + n, head] = (h + 2 * (inner + tiny))[:, 0]
                padded = torch.nn.functional.pad(p / total, (0, -N % 64))
                share[lo:lo + n, head, :padded.shape[1] // 64] = padded.view(n, -1, 64).sum(2)
    return ref, lim, share, of_one


def _places(b, r):
    at = b.torch.arange(int(b.lengths[r]), device="cuda")
    return at, b.tables[r].long()[at // PAGE]


ROWS = {"prompt": [(128, 70), (1100, 40), (1, 200)], "prompt_cut": [(20000, 5), (9001, 40), (50000, 1)], "decode": [(1200, 1), (100, 1), (300, 1), (700, 1)], "decode_cut": [(20000, 1), (50000, 1), (150, 1)]}


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads", [(32, 2), (7, 1)], ids=str)
@pytest.mark.parametrize("level", ["far_below", "rising", "level"])
@pytest.mark.parametrize("which", ["first", "half"])
@pytest.mark.parametrize("rows", list(ROWS))
def test_tiles_whose_scores_are_minus_infinity(gpu, set_option, dtype, heads, level, which, rows):
    """Infinities in the keys of whole tiles, ahead of finite ones: the tiles weigh nothing, the others all that they have."""
    torch = gpu
    set_option("dtype", dtype)
    b = Batch(torch, 50, [(max(c, 128), n) for c, n in ROWS[rows]] if which == "half" else [(max(c, 64), n) for c, n in ROWS[rows]], *heads, dtype=dtype, spread=0.3)
    hidden = (lambda at: at < 64) if which == "first" else (lambda at: at // 128 % 2 == 0)  # noqa: E731
    b.q[:, :, 0], b.q[:, :, 1] = 1.0, 16.0
    for r in range(len(b.requests)):
        at, page = _places(b, r)
        # scores in powers of two: -30; 6 and then, of every 512 keys, 8 in a few; 0
        octaves = {"far_below": 0.0 * at - 30, "rising": torch.where(at % 512 >= 460, 8.0, 6.0), "level": 0.0 * at}[level]
        b.k[page, :, at % PAGE, 1] = (octaves * math.log(2) / (16.0 * SCALE))[:, None].to(b.k.dtype)
        b.k[page, :, at % PAGE, 0] = torch.where(hidden(at), -math.inf, 0.0)[:, None].to(b.k.dtype)
    b.check(b.run(rows.split("_")[0]), _expect(b, hidden)[:2])


@pytest.mark.parametrize("kind, heads, requests", [
    ("decode", (7, 1), [(1000, 1)] * 5), ("decode", (32, 2), [(2500, 1)] * 200), ("decode", (16, 16), [(60, 1), (3000, 1)]), ("prompt", (32, 2), [(0, 900), (700, 130)]), ("prompt", (7, 1), [(3000, 200)])],
    ids=["decode_1000", "decode_2500", "decode_mha", "prompt_two", "prompt_far"])
@pytest.mark.parametrize("gap", [12.0, 14.0, 16.5, 18.0])
@pytest.mark.parametrize("place", ["first", "middle"])
def test_one_key_far_above_the_others(gpu, kind, heads, requests, gap, place):
    """e^gap times as much weight on one key, whose value is 0: the result is what the many small probabilities of the others add up to (fp16)."""
    torch = gpu
    b = Batch(torch, 51, requests, *heads, spread=0.3)
    b.q[:, :, 0] = 16.0
    for r in range(len(b.requests)):
        at, page = _places(b, r)
        above = at == (0 if place == "first" else int(b.requests[r][0]) // 2)
        b.k[page, :, at % PAGE, 0] = torch.where(above, gap / (16.0 * SCALE), 0.0)[:, None].half()
        v = torch.where(above[:, None, None], 0.0, 32.0 + 16.0 * b.v[page, :, :, b.slot[at % PAGE]].float())
        b.v[page, :, :, b.slot[at % PAGE]] = v.half()
    shift = {"prompt": 10, "decode": 12}[kind]
    b.check(b.run(kind), _expect(b, shift=shift)[:2])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("kind, heads, requests", [
    ("decode", (32, 2), [(100000, 1)]), ("decode", (7, 1), [(131000, 1)]), ("decode", (32, 8), [(40000, 1), (3, 1), (17, 1), (26000, 1), (900, 1)]), ("decode", (16, 16), [(9000, 1)] * 3),
    ("prompt", (32, 2), [(9001, 40), (50000, 1), (3, 1), (17000, 129)]), ("prompt", (4, 1), [(30011, 64)])],
    ids=["decode_2_heads", "decode_1_head", "decode_ragged", "decode_mha", "prompt_ragged", "prompt_chunk"])
def test_every_tile_of_long_requests_counts(gpu, set_option, dtype, kind, heads, requests):
    """The values of a tile of 64 keys are 1 in a dim of its own and 0 elsewhere, 128 tiles at a time: each dim is its tile's share of the probabilities.  A tile that is lost or counted
    twice moves its dim by far more than the limit, as is checked first."""
    torch = gpu
    set_option("dtype", dtype)
    b = Batch(torch, 52, requests, *heads, dtype=dtype, spread=1.0)
    _, _, share, of_one = _expect(b)
    tiles = share.shape[2]
    mark = torch.cat([torch.eye(D, device="cuda"), torch.zeros((1, D), device="cuda")]).to(b.v.dtype)
    for first in range(0, tiles, D):
        for r in range(len(requests)):
            at, page = _places(b, r)
            tile = at // 64 - first
            b.v[page, :, :, b.slot[at % PAGE]] = mark[torch.where((tile >= 0) & (tile < D), tile, D)][:, None, :].expand(-1, heads[1], -1)
        ref = torch.nn.functional.pad(share[:, :, first:first + D], (0, max(0, first + D - tiles)))
        lim = of_one[:, :, None] * ref + 2.0 ** -25
        several = (ref > 2.0 ** -20) & (ref < 0.9)  # (all of a row that sees one tile is that tile's; a row's last tile may be next to nothing)
        assert bool((ref * (1 - ref) / (1 + ref) > 2 * lim)[several].all()) and bool(several.any())
        b.check(b.run(kind), (ref, lim))
