"""Batches on the GPU: block tables and slot maps, rotary positions, appends through slots and 8-bit products against plain
implementations in 64 bits (whole numbers: equal), at the sizes, masks and layouts where they can go wrong.

Tolerances: a 16-bit result is a 32-bit value rounded once (half a step of the type: 2^-11 of the value in fp16, 2^-8 in bf16, 2^-25 where
fp16 runs out of exponents), and the 32-bit value carries the errors that are counted beside each test.
"""
import numpy as np
import pytest

from cpm.cu_amd import synth

pytestmark = pytest.mark.gpu

PAGE, D = 256, 128
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}


def _types(torch, dtype):
    return torch.bfloat16 if dtype else torch.float16


def _close(got, ref, dtype, inner):
    """got within half a step of its type of a value that is within `inner` (an array of absolute errors) of ref."""
    got, ref = got.double().cpu().numpy(), ref.double().cpu().numpy()
    inner = inner.double().cpu().numpy() if hasattr(inner, "cpu") else inner
    limit = (np.abs(ref) + inner) * HALF_STEP[dtype] + 2.0 ** -25 + inner
    worst = np.max(np.abs(got - ref) - limit) if got.size else -1.0
    assert worst <= 0, "off by %.3g more than the roundings allow" % worst


# ---- block tables and slot maps ----

def _walk(kv, new, tables, held, stack, count, max_rows):
    """Request by request, as the operator's description has it."""
    B, M = tables.shape
    tables, stack = tables.copy(), stack.copy()
    F = len(stack)
    h = np.clip(held, 0, M)
    count = min(max(int(count), 0), F)
    for r in range(B):
        if new[r] < 0:
            for b in range(h[r]):
                if count < F:
                    stack[count] = tables[r, b]
                    count += 1
    lens, held_out, offsets, refused, dry = kv.copy(), h.copy(), [0], 0, False
    positions, slots = np.full(max_rows, -1), np.full(max_rows, -1)
    total = 0
    for r in range(B):
        n = max(int(new[r]), 0)
        first = total
        total += n
        offsets.append(min(total, max_rows))
        if new[r] < 0:
            lens[r] = held_out[r] = 0
            continue
        blocks = -(-(int(kv[r]) + n) // PAGE)
        if kv[r] < 0 or blocks > M or (n and total > max_rows):
            refused += 1
            continue
        need = max(0, blocks - int(h[r]))
        if need and (dry or need > count):
            dry, refused = True, refused + 1
            continue
        for b in range(h[r], blocks):
            count -= 1
            tables[r, b] = stack[count]
        lens[r], held_out[r] = kv[r] + n, max(int(h[r]), blocks)
        for i in range(n):
            at = int(kv[r]) + i
            page = int(tables[r, at // PAGE])
            positions[first + i] = at
            slots[first + i] = page * PAGE + at % PAGE if 0 <= page < F else -1
    return dict(kv_lens=lens, held=held_out, counts=[count, refused], row_offsets=offsets, positions=positions, slots=slots), tables, stack


def _batch(seed, B, M, mean_cached, mean_new, ended=0.0, idle=0.0, spare=1.0, over=0.0):
    g = synth.rng(seed, 300)
    kv = np.minimum(g.geometric(1.0 / mean_cached, B) - 1, M * PAGE)
    new = g.geometric(1.0 / mean_new, B)
    new = np.where(g.random(B) < over, new, np.minimum(new, M * PAGE - kv))
    new[g.random(B) < idle] = 0
    new[g.random(B) < ended] = -1
    held = -(-kv // PAGE)
    more = g.random(B) < 0.2  # pages kept from rows that were not accepted
    held = np.minimum(held + more, M)
    need = np.maximum(-(-(kv + np.maximum(new, 0)) // PAGE) - held, 0).sum()
    pages = int(held.sum() + max(1, round(need * spare)))
    order = g.permutation(pages)
    tables = g.integers(0, pages, (B, M))  # (what lies behind a request's pages is of no matter)
    tables[np.arange(M)[None, :] < held[:, None]] = order[:held.sum()]
    stack = g.integers(0, pages, pages)
    free = pages - int(held.sum())
    stack[:free] = order[held.sum():]
    return kv, new, tables, held, stack, free


def _run_tables(torch, kv, new, tables, held, stack, count, max_rows):
    from cpm.cu_amd import ops
    cu = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32)).cuda()  # noqa: E731
    ins = [cu(kv), cu(new), cu(tables), cu(held), cu(stack), cu([count, 77])]
    before = [t.clone() for t in ins]
    out = ops.batch_tables(*ins, max_rows)
    torch.cuda.synchronize()
    for i in (0, 1, 3, 5):
        assert torch.equal(ins[i], before[i]), "an input has changed"
    return out, ins[2].cpu().numpy(), ins[4].cpu().numpy()


def _check_tables(torch, kv, new, tables, held, stack, count, max_rows):
    want, tables_want, stack_want = _walk(kv, new, tables, held, stack, count, max_rows)
    out, tables_got, stack_got = _run_tables(torch, kv, new, tables, held, stack, count, max_rows)
    for name, value in want.items():
        assert np.array_equal(out[name].cpu().numpy(), value), name
    assert np.array_equal(tables_got, tables_want) and np.array_equal(stack_got, stack_want)
    return want


@pytest.mark.parametrize("B, M, mean_cached, mean_new, kw, rows", [
    (1, 1, 1, 1, {}, 1), (1, 4, 300, 700, {}, 1000), (16, 512, 8000, 1, {}, 16), (16, 512, 8000, 1, dict(ended=0.3, idle=0.3), 64), (60, 8, 500, 300, dict(ended=0.1), 20001),
    (64, 3, 256, 256, dict(over=0.3), 40000), (333, 16, 1000, 100, dict(ended=0.2, idle=0.2, spare=0.5), 33333), (1023, 8, 200, 5, {}, 6001), (1024, 4, 300, 20, dict(ended=0.5), 30000),
    (1025, 4, 300, 20, dict(ended=0.1, spare=0.0), 30000), (4096, 5, 400, 30, dict(ended=0.1, idle=0.5, spare=0.9), 70003), (4096, 64, 1000, 1, {}, 4096), (100, 40, 2000, 500, dict(spare=0.8), 25000),
    (3, 2000, 200000, 100000, {}, 400000), (255, 16, 900, 300, dict(ended=0.1, spare=0.7), 60001), (256, 9, 700, 3, dict(idle=0.2), 999), (257, 9, 700, 3, dict(idle=0.2), 999), (200, 9, 300, 400, dict(over=0.2), 30000), (2000, 9, 300, 100, dict(over=0.2, ended=0.1), 100000), (5, 8, 100, 100, dict(ended=1.0), 64), (5, 8, 100, 100, dict(idle=1.0), 64), (7, 8, 100, 100, {}, 0)])
def test_batch_tables_is_the_walk_through_the_requests(gpu, B, M, mean_cached, mean_new, kw, rows):
    for seed in range(3):
        _check_tables(gpu, *_batch(B * 31 + seed, B, M, mean_cached, mean_new, **kw), rows)


@pytest.mark.parametrize("B, M, mean_cached, mean_new, kw, rows", [
    (256, 16, 900, 300, dict(ended=0.1), 65537), (30, 200, 900, 5000, dict(over=0.1), 131333), (257, 40, 900, 1100, dict(ended=0.1, spare=0.9), 262145),
    (1024, 9, 100, 300, dict(idle=0.5), 300001), (1025, 9, 100, 300, dict(idle=0.2, ended=0.2), 270000), (4096, 4, 100, 80, dict(idle=0.1), 262209)])
def test_batch_tables_of_many_rows(gpu, B, M, mean_cached, mean_new, kw, rows):
    """More rows than there are threads: several runs of rows a wave."""
    _check_tables(gpu, *_batch(B * 37, B, M, mean_cached, mean_new, **kw), rows)


def test_batch_tables_by_hand(gpu):
    """Boundaries of pages, requests that do not fit (the table, the stack, the rows), and lengths that are none."""
    I = 2 ** 31 - 1
    for kv, new, held, count, rows in (
            ([0, 255, 256, 257], [256, 1, 1, 255], [0, 1, 1, 2], 8, 600),          # pages that end with a request's last row
            ([0, 0, 0], [257, 256, 1], [0, 0, 0], 3, 600),                          # the stack ends at the second request; the third is behind it
            ([0, 100, 0], [600, 1, 1], [0, 1, 0], 2, 700),                          # a request without need passes one that is refused
            ([10, 20, 30], [5, 5, 0], [1, 1, 1], 4, 9),                             # rows that end behind the last place; none of the next one
            ([10, 20, 30], [I, I, 1], [1, 1, 1], 4, 9), ([I, I, 0], [1, 0, 1], [1, 1, 1], 4, 9), ([-5, 3, -2 ** 31], [1, 1, -2 ** 31], [1, 1, 3], 4, 9),
            ([0, 0, 0], [1, 1, 1], [-3, 99, 0], 4, 9), ([0, 0, 0], [300, 300, 300], [0, 0, 0], 99, 900), ([0, 0, 0], [300, 300, 300], [0, 0, 0], -1, 900),
            ([700, 0, 100], [-1, 600, -1], [3, 0, 1], 0, 600),                      # given back and taken again in one step
            ([700, 700, 0], [-1, -1, 1], [3, 3, 0], 7, 5)):                         # more given back than the stack can hold
        tables = np.arange(12).reshape(3, 4) % 8 if len(kv) == 3 else np.arange(16).reshape(4, 4) % 8
        _check_tables(gpu, np.array(kv), np.array(new), tables, np.array(held), np.arange(8)[::-1].copy(), count, rows)
    # page numbers outside the pool give no slot
    _check_tables(gpu, np.array([0, 10]), np.array([10, 10]), np.array([[3, 3], [9, 0]]), np.array([0, 1]), np.array([5, -7, 99]), 3, 20)
    _check_tables(gpu, np.array([0, 10]), np.array([10, 10]), np.array([[3, 3], [2, 0]]), np.array([0, 1]), np.array([5, 1, 2]), 2, 20)


def test_batch_tables_into_rows_off_16_bytes(gpu):
    """Positions and slots that do not start on 16 bytes, through the C-ABI."""
    import ctypes
    torch = gpu
    from cpm.cu_amd import lib
    kv, new, tables, held, stack, count = _batch(5, 40, 8, 300, 50)
    want, _, _ = _walk(kv, new, tables, held, stack, count, 2001)
    cu = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32)).cuda()  # noqa: E731
    ins = [cu(kv), cu(new), cu(tables), cu(held), cu(stack), cu([count, 0])]
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rows = torch.full((2, 2007), -5, dtype=torch.int32, device="cuda")
    out = [torch.zeros(50, dtype=torch.int32, device="cuda") for _ in range(4)]
    lib.get().batch_tables(p(ins[0]), p(ins[1]), 40, p(ins[2]), 8, p(ins[3]), p(ins[4]), len(stack), p(ins[5]), *(p(t) for t in out), p(rows[0, 1:]), p(rows[1, 3:]), 2001,
                           ctypes.c_void_p(torch.cuda.current_stream().cuda_stream or 1))
    torch.cuda.synchronize()
    assert np.array_equal(rows[0, 1:2002].cpu(), want["positions"]) and np.array_equal(rows[1, 3:2004].cpu(), want["slots"])
    assert (rows[0, 2002:] == -5).all() and (rows[1, 2004:] == -5).all() and (rows[:, 0] == -5).all()


# ---- rotary positions ----

def _turned(torch, x, positions, inv_freq, interleaved, magnitude, transposed=False):
    """In 64 bits; and the absolute error that 32 bits may leave: |x| + |y| of the pair times its errors."""
    r = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = torch.cos(angle)[:, None] * magnitude, torch.sin(angle)[:, None] * (-magnitude if transposed else magnitude)
    t = x.double()
    u, v = (t[..., 0:r:2], t[..., 1:r:2]) if interleaved else (t[..., :r // 2], t[..., r // 2:r])
    pair = [u * c - v * s, u * s + v * c]
    # sine and cosine: 2 units in the last place and the turn's rounding to 32 bits, 2^-22; the turn's 64-bit product, 2^-51 of the angle;
    # magnitude, two products and a sum, 4 * 2^-24
    err = (u.abs() + v.abs()) * abs(magnitude) * (2.0 ** -21 + (angle.abs() * 2.0 ** -50)[:, None])
    join = lambda a, b: torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)  # noqa: E731
    return torch.cat([join(*pair), t[..., r:]], -1), torch.cat([join(err, err), torch.zeros_like(t[..., r:])], -1)


def _rows(torch, seed, dtype, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=_types(torch, dtype), device="cuda").normal_(generator=g)


def _freq(torch, half, base=10000.0):
    return torch.from_numpy((base ** (-np.arange(half) / half)).astype(np.float32)).cuda()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n, Hq, Hkv, dim, rotary", [
    (1, 32, 2, 128, 128), (60, 32, 2, 128, 128), (7, 7, 1, 128, 64), (5, 3, 3, 128, 96), (129, 16, 16, 128, 16), (1023, 32, 8, 128, 128), (3, 1, 0, 64, 32), (9, 5, 2, 256, 256), (33, 4, 4, 80, 80),
    (4, 1000, 24, 16, 16), (6, 2, 1, 128, 42), (11, 3, 2, 62, 60), (2, 1, 1, 2, 2), (17, 9, 3, 100, 100), (4097, 2, 1, 128, 128)])
def test_rope_rows(gpu, set_option, dtype, interleaved, n, Hq, Hkv, dim, rotary):
    torch = gpu
    from cpm.cu_amd import ops
    set_option("dtype", dtype)
    q, k = _rows(torch, n, dtype, n, Hq, dim), _rows(torch, n + 1, dtype, n, Hkv, dim) if Hkv else None
    positions = torch.from_numpy(synth.rng(n, 7).integers(0, 200000, n).astype(np.int32)).cuda()
    positions[0] = 2 ** 31 - 1 if n > 4 else 0
    inv_freq = _freq(torch, rotary // 2)
    h = lambda t: None if t is None else t.view(torch.float16)  # noqa: E731
    for magnitude, transposed in ((1.0, False), (1.25, True)):
        keep = [q.clone(), None if k is None else k.clone()]
        q_out, k_out = ops.rope_rows(h(q), h(k), positions, inv_freq, interleaved, magnitude, transposed)
        torch.cuda.synchronize()
        for x, was, y in ((q, keep[0], q_out), (k, keep[1], k_out)):
            if x is None:
                assert y is None
                continue
            assert torch.equal(x.view(torch.int16), was.view(torch.int16)), "an input has changed"
            ref, err = _turned(torch, x, positions, inv_freq, interleaved, magnitude, transposed)
            _close(y.view(_types(torch, dtype)), ref, dtype, err)
            assert torch.equal(y[..., rotary:].view(torch.int16), x[..., rotary:].view(torch.int16))
        # in place: the same bits
        ops.rope_rows(h(keep[0]), h(keep[1]), positions, inv_freq, interleaved, magnitude, transposed, q_out=h(keep[0]), k_out=h(keep[1]))
        torch.cuda.synchronize()
        assert torch.equal(keep[0].view(torch.int16), q_out.view(torch.int16)) and (k is None or torch.equal(keep[1].view(torch.int16), k_out.view(torch.int16)))


@pytest.mark.parametrize("offset, rotary", [(0, 128), (8, 64), (1, 128), (0, 42), (5, 20)])
def test_rope_rows_of_wider_rows_and_rows_left_out(gpu, offset, rotary):
    """Views of a fused projection's rows, on 16 bytes and off them; what lies between them, and rows of a negative position, stay."""
    torch = gpu
    from cpm.cu_amd import ops
    n, Hq, Hkv = 37, 4, 2
    width = (Hq + 2 * Hkv) * D + (8 if offset % 8 == 0 else 3)
    x = _rows(torch, 3, 0, n, width)
    view = lambda t, first, heads: t[:, offset + first * D: offset + (first + heads) * D].view(n, heads, D) if offset + (first + heads) * D <= width else None  # noqa: E731
    q, k = view(x, 0, Hq), view(x, Hq, Hkv)
    positions = torch.arange(1000, 1000 + n, dtype=torch.int32, device="cuda")
    positions[::5] = -1
    positions[1] = -2 ** 31
    out = torch.full_like(x, 7.0)
    ops.rope_rows(q, k, positions, _freq(torch, rotary // 2), q_out=view(out, 0, Hq), k_out=view(out, Hq, Hkv))
    in_place = x.clone()
    ops.rope_rows(view(in_place, 0, Hq), view(in_place, Hq, Hkv), positions, _freq(torch, rotary // 2), q_out=view(in_place, 0, Hq), k_out=view(in_place, Hq, Hkv))
    torch.cuda.synchronize()
    left = positions < 0
    for first, heads, t in ((0, Hq, q), (Hq, Hkv, k)):
        ref, err = _turned(torch, t, positions, _freq(torch, rotary // 2), False, 1.0)
        got = view(out, first, heads)
        _close(got[~left], ref[~left], 0, err[~left])
        assert (got[left] == 7.0).all()
        assert torch.equal(view(in_place, first, heads)[~left].view(torch.int16), got[~left].view(torch.int16))
        assert torch.equal(view(in_place, first, heads)[left], t[left])
    used = torch.zeros(width, dtype=torch.bool, device="cuda")
    used[offset: offset + (Hq + Hkv) * D] = True
    assert (out[:, ~used] == 7.0).all() and torch.equal(in_place[:, ~used], x[:, ~used])


def test_rope_rows_of_one_wide_row_in_any_columns(gpu):
    """q, k and their results as columns of one tensor, in place and beside each other; columns that overlap are refused."""
    torch = gpu
    from cpm.cu_amd import ops
    n, Hq, Hkv = 21, 3, 2
    x = _rows(torch, 3, 0, n, 14 * D)
    part = lambda t, at, heads: t[:, at:at + heads * D].view(n, heads, D)  # noqa: E731
    positions, freq = torch.arange(n, dtype=torch.int32, device="cuda") * 1000, _freq(torch, 64)
    want = [t.clone() for t in ops.rope_rows(part(x, 0, Hq), part(x, Hq * D, Hkv), positions, freq)]
    for q_at, k_at in ((0, Hq * D), (5 * D, Hq * D), (0, 8 * D), (5 * D, 8 * D), (11 * D, 5 * D), (9 * D, 12 * D)):
        y = x.clone()
        ops.rope_rows(part(y, 0, Hq), part(y, Hq * D, Hkv), positions, freq, q_out=part(y, q_at, Hq), k_out=part(y, k_at, Hkv))
        torch.cuda.synchronize()
        assert torch.equal(part(y, q_at, Hq), want[0]) and torch.equal(part(y, k_at, Hkv), want[1])
        written = torch.zeros(14 * D, dtype=torch.bool, device="cuda")
        written[q_at:q_at + Hq * D] = written[k_at:k_at + Hkv * D] = True
        assert torch.equal(y[:, ~written], x[:, ~written])
    for q_at, k_at in ((2 * D, Hq * D), (4 * D, Hq * D), (0, 2 * D), (5 * D, 7 * D), (0, Hq * D + 8)):
        y = x.clone()
        with pytest.raises(ValueError, match="results"):
            ops.rope_rows(part(y, 0, Hq), part(y, Hq * D, Hkv), positions, freq, q_out=part(y, q_at, Hq), k_out=part(y, k_at, Hkv))
        torch.cuda.synchronize()
        assert torch.equal(y, x)


def test_rope_gradient_is_the_transposed_rotation(gpu):
    """Against differences: for f = sum(w * rope(x)), (f(x + h e) - f(x - h e)) / 2h = rope^T(w) . e, f being linear in x.  The sums are of
    fp16 results (half a step each, 2^-11) over 2h = 2: 32 values of |w| <= 4 and |y| <= 12 leave 32 * 4 * 12 * 2^-11 / 2 in the worst case."""
    torch = gpu
    from cpm.cu_amd import ops
    n, H = 3, 2
    x, w = _rows(torch, 1, 0, n, H, 32).clamp(-4, 4), _rows(torch, 2, 0, n, H, 32).clamp(-4, 4)
    positions = torch.tensor([0, 5, 70000], dtype=torch.int32, device="cuda")
    for interleaved in (False, True):
        inv_freq = _freq(torch, 12)  # 24 of 32 values turn
        f = lambda t: (ops.rope_rows(t, None, positions, inv_freq, interleaved, 1.25)[0].double() * w.double()).sum((1, 2))  # noqa: E731
        grad, _ = ops.rope_rows(w, None, positions, inv_freq, interleaved, 1.25, transposed=True)
        ref, err = _turned(torch, w, positions, inv_freq, interleaved, 1.25, transposed=True)
        _close(grad, ref, 0, err)
        for i in range(0, 32, 3):
            e = torch.zeros_like(x)
            e[:, 1, i] = 1.0
            diff = (f((x + e)) - f((x - e))) / 2.0
            # (x + e and x - e are rounded to fp16 as well: |x| + 1 <= 5, two of them, times |rope^T w| <= 10)
            assert ((diff - grad[:, 1, i].double()).abs() <= 32 * 4 * 12 * 2.0 ** -11 / 2 + 10 * 5 * 2.0 ** -11).all(), i


# ---- append through slots ----

def _slot_case(seed, n, kind):
    """(slots, pages): rows of requests that follow each other in pages (prompts), one each (decode), or anywhere."""
    g = synth.rng(seed, 400)
    if kind == "decode":
        pages = n + 1
        return g.permutation(pages)[:n] * PAGE + g.integers(0, PAGE, n), pages
    if kind == "scattered":
        pages = n // 64 + 2
        return g.permutation(pages * PAGE)[:n], pages
    slots, pages = [], 0
    while sum(map(len, slots)) < n:
        length, first = int(g.integers(1, 700)) if kind == "prompts" else int(g.integers(1, 21)), int(g.integers(0, 1000))
        at = first + np.arange(length)
        slots.append((pages + at // PAGE - first // PAGE) * PAGE + at % PAGE)
        pages += int(at[-1] // PAGE - first // PAGE) + 1
    slots = np.concatenate(slots)[:n]
    order = g.permutation(pages)
    return order[slots // PAGE] * PAGE + slots % PAGE, pages


def _logical(torch, cache, slots):
    """Rows at these slots, out of the pools as they are documented."""
    from cpm.cu_amd.kvcache import v_slot
    page, at = slots.long() // PAGE, slots.long() % PAGE
    return cache.k[0][page, :, at], cache.v[0][page, :, :, v_slot(at)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n, Hq, Hkv, kind, rotary, interleaved", [
    (1, 32, 2, "decode", 128, False), (64, 32, 8, "decode", 128, False), (16, 4, 4, "prompts", 64, True), (17, 32, 2, "chunks", 128, False), (333, 32, 2, "prompts", 128, True), (500, 0, 1, "chunks", 0, False),
    (100, 0, 4, "scattered", 0, False), (77, 5, 3, "scattered", 96, False), (2049, 32, 2, "prompts", 128, False), (4001, 0, 4, "prompts", 0, False), (1000, 16, 16, "chunks", 16, True), (15, 0, 2, "prompts", 128, False)])
def test_kv_append_slots(gpu, set_option, dtype, n, Hq, Hkv, kind, rotary, interleaved):
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache, v_slot
    set_option("dtype", dtype)
    slots_np, pages = _slot_case(n + Hkv, n, kind)
    g = synth.rng(n, 401)
    slots_np = np.where(g.random(n) < (0.1 if n > 20 else 0.0), g.choice([-1, -2 ** 31, pages * PAGE, 2 ** 31 - 1], n), slots_np)
    slots = torch.from_numpy(slots_np.astype(np.int32)).cuda()
    positions = torch.from_numpy(g.integers(0, 100000, n).astype(np.int32)).cuda()
    if n > 20 and rotary:
        positions[3] = -1
    x = _rows(torch, n, dtype, n, (Hq + 2 * Hkv) * D)
    h = x.view(torch.float16)
    q, k, v = h[:, :Hq * D].view(n, Hq, D) if Hq else None, h[:, Hq * D:(Hq + Hkv) * D].view(n, Hkv, D), h[:, (Hq + Hkv) * D:].view(n, Hkv, D)
    cache = PagedKVCache(1, Hkv, pages)
    cache.k[0].copy_(_rows(torch, 1, 0, *cache.k[0].shape))
    cache.v[0].copy_(_rows(torch, 2, 0, *cache.v[0].shape))
    k_was, v_was = cache.k[0].clone(), cache.v[0].clone()
    inv_freq = _freq(torch, rotary // 2) if rotary else None
    q_out = torch.full((n, Hq, D), 7.0, dtype=torch.float16, device="cuda") if Hq else None
    got_q = ops.kv_append_slots(cache, 0, k, v, slots, q=q, q_out=q_out, positions=positions if rotary else None, inv_freq=inv_freq, interleaved=interleaved, magnitude=1.125 if rotary else 1.0)
    torch.cuda.synchronize()
    there = (slots >= 0) & (slots < pages * PAGE)
    if rotary:
        there &= positions >= 0
        k_want = ops.rope_rows(k, None, positions, inv_freq, interleaved, 1.125)[0]
        if Hq:
            assert got_q is q_out
            ref, err = _turned(torch, x[:, :Hq * D].view(n, Hq, D), positions, inv_freq, interleaved, 1.125)
            _close(q_out.view(_types(torch, dtype))[there], ref[there], dtype, err[there])
            assert (q_out[~there] == 7.0).all()
    else:
        k_want = k
    # every place of the pools: the rows' own, and what was there in all others
    page, at = slots[there].long() // PAGE, slots[there].long() % PAGE
    k_was[page, :, at] = k_want[there]
    v_was[page, :, :, v_slot(at)] = v[there]
    assert torch.equal(cache.k[0].view(torch.int16), k_was.view(torch.int16))
    assert torch.equal(cache.v[0].view(torch.int16), v_was.view(torch.int16))


@pytest.mark.parametrize("n", [1, 5, 200])
def test_kv_append_slots_turns_q_in_place_of_a_fused_projection(gpu, n):
    """q's results over q, between k and v of the same rows: the same as into memory of their own, k and v as they were."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    Hq, Hkv = 6, 2
    x = _rows(torch, n, 0, n, (Hq + 2 * Hkv) * D)
    slots, positions = torch.arange(n, dtype=torch.int32, device="cuda") + 100, torch.arange(n, dtype=torch.int32, device="cuda") + 70000
    freq = _freq(torch, 64)
    parts = lambda t: [y.view(n, -1, D) for y in t.split([Hkv * D, Hq * D, Hkv * D], 1)]  # noqa: E731
    one, two, y = PagedKVCache(1, Hkv, 2), PagedKVCache(1, Hkv, 2), x.clone()
    k, q, v = parts(x)
    want = ops.kv_append_slots(one, 0, k, v, slots, q=q, positions=positions, inv_freq=freq)
    k, q, v = parts(y)
    ops.kv_append_slots(two, 0, k, v, slots, q=q, q_out=q, positions=positions, inv_freq=freq)
    torch.cuda.synchronize()
    assert torch.equal(q, want) and torch.equal(one.k[0], two.k[0]) and torch.equal(one.v[0], two.v[0])
    assert torch.equal(k, parts(x)[0]) and torch.equal(v, parts(x)[2])


def test_kv_append_slots_is_kv_append_for_one_sequence(gpu):
    """Rows that follow each other in one sequence: the same cache, bit for bit."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    for P, n in ((0, 1), (250, 20), (1000, 777), (4000, 2048), (13, 300)):
        pages = (P + n) // PAGE + 2
        table = synth.rng(P, 4).permutation(pages).astype(np.int32)
        one, two = PagedKVCache(1, 2, pages, block_table=table), PagedKVCache(1, 2, pages, block_table=table)
        k, v = _rows(torch, P, 0, n, 2, D), _rows(torch, P + 1, 0, n, 2, D)
        ops.kv_append(one, 0, k, v, torch.tensor([P + n], dtype=torch.int32, device="cuda"))
        at = np.arange(P, P + n)
        ops.kv_append_slots(two, 0, k, v, torch.from_numpy((table[at // PAGE] * PAGE + at % PAGE).astype(np.int32)).cuda())
        torch.cuda.synchronize()
        assert torch.equal(one.k[0], two.k[0]) and torch.equal(one.v[0], two.v[0])


def test_kv_append_slots_far_into_a_large_pool(gpu):
    """Places whose offsets pass 32 bits (in values, and well before that in bytes)."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache, v_slot
    Hkv, pages = 8, 2 ** 31 // (8 * PAGE * D) + 3
    k_pool, v_pool = torch.zeros((pages, Hkv, PAGE, D), dtype=torch.float16, device="cuda"), torch.zeros((pages, Hkv, D, PAGE), dtype=torch.float16, device="cuda")
    cache = PagedKVCache.from_pools([k_pool], [v_pool], torch.zeros(1, dtype=torch.int32, device="cuda"))
    n = 40
    at = torch.arange(n, device="cuda") + 100
    slots = ((pages - 2) * PAGE + at).int()
    k, v = _rows(torch, 5, 0, n, Hkv, D), _rows(torch, 6, 0, n, Hkv, D)
    ops.kv_append_slots(cache, 0, k, v, slots)
    torch.cuda.synchronize()
    assert torch.equal(k_pool[pages - 2][:, at].transpose(0, 1), k)
    assert torch.equal(v_pool[pages - 2][:, :, v_slot(at)].permute(2, 0, 1), v)
    assert not k_pool[:pages - 2].any() and not v_pool[:pages - 2].any() and not k_pool[pages - 1].any()


# ---- 8-bit rows and products ----

def _quantized(torch, x):
    """In 64 bits: the quotient is a tie only where it is one exactly (else it is 2^-19 of itself away, and off by 2^-52)."""
    x = x.double().cpu()
    finite = torch.isfinite(x).all(1)
    amax = x.abs().amax(1)
    q = torch.round(x * 127.0 / amax[:, None])
    q = torch.where((finite & (amax > 0))[:, None], q, torch.zeros_like(q))
    return q.to(torch.int8), torch.where(finite, amax / 127.0, torch.full_like(amax, float("nan")))


def _check_quantized(torch, x):
    from cpm.cu_amd import ops
    n, K = x.shape
    xq, scales = ops.quantize_rows(x.view(torch.float16) if x.is_contiguous() or x.dtype == torch.float16 else x)
    torch.cuda.synchronize()
    q, s = _quantized(torch, x)
    assert xq.shape == (n, (K + 63) // 64 * 64) and torch.equal(xq[:, :K].cpu(), q) and not xq[:, K:].any()
    got = scales.double().cpu()
    assert torch.equal(got.isnan(), s.isnan())
    ok = ~s.isnan()
    assert ((got - s).abs()[ok] <= s[ok] * 2.0 ** -24 + 2.0 ** -150).all()  # one division in 32 bits (2^-150: half the smallest step)
    return xq, scales


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n, K", [(1, 1), (1, 4096), (3, 63), (7, 64), (5, 65), (60, 4096), (2, 4099), (9, 2047), (3, 16384), (2, 16385), (2, 40000), (1, 131071), (1000, 200)])
def test_quantize_rows(gpu, set_option, dtype, n, K):
    torch = gpu
    set_option("dtype", dtype)
    x = _rows(torch, n + K, dtype, n, K)
    x[0] *= 0.001
    _check_quantized(torch, x)
    if n > 1:
        x[1] = 0
        x[-1, K // 2] = float("inf") if K % 2 else float("nan")
        _check_quantized(torch, x)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n, K", [(1023, 129), (1024, 1), (1025, 64), (1026, 71), (1027, 512), (1030, 4090), (1031, 4096), (1024, 4097), (1024, 4161)])
def test_quantize_many_rows(gpu, set_option, dtype, n, K):
    """A wave a row, and rows that are just too long for one."""
    torch = gpu
    set_option("dtype", dtype)
    x = _rows(torch, n + K, dtype, n, K)
    x[0] *= 0.001
    x[1] = 0
    x[2, K // 2] = float("inf")
    x[-1, K - 1] = float("nan")
    _check_quantized(torch, x)
    _check_quantized(torch, torch.cat([x, x], 1)[:, 3 % K:3 % K + K].contiguous().view(n, K))


@pytest.mark.parametrize("dtype", [0, 1])
def test_quantize_rows_at_the_types_limits(gpu, set_option, dtype):
    """Ties, the largest and the smallest values, signed zeros, -inf and NaN of either sign."""
    torch = gpu
    set_option("dtype", dtype)
    t = _types(torch, dtype)
    big, tiny = torch.finfo(t).max, 2.0 ** -24 if dtype == 0 else 2.0 ** -133
    rows = [[127.0] + [i + 0.5 for i in range(60)], [63.5] + [(i + 0.5) / 2 for i in range(60)], [big, -big] + [big / 3, -big / 5, 1.0, tiny] * 14, [tiny, -tiny] + [0.0, -0.0] * 29, [5 * tiny, -3 * tiny] + [tiny, 2 * tiny] * 29,
            [-0.0] * 61, [float("-inf")] + [1.0] * 60, [1.0] * 60 + [float("nan")], [254.0] + [float(i) for i in range(60)], [2.0 ** -14, 2.0 ** -15] * 30 + [0.0]]
    x = torch.zeros((len(rows), 61), dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, :min(len(r), 61)] = torch.tensor(r[:61], dtype=torch.float64)
    x = x.to(t).cuda()
    x[7, 60] = -x[7, 60]
    _check_quantized(torch, x)
    _check_quantized(torch, torch.cat([x, torch.zeros((len(rows), 3), dtype=t, device="cuda")], 1))  # rows in 16-byte pieces


def test_quantize_rows_of_wider_rows(gpu):
    torch = gpu
    x = _rows(torch, 8, 0, 20, 700)
    for lo, hi in ((0, 512), (8, 648), (3, 700), (64, 65)):
        _check_quantized(torch, x[:, lo:hi])


def test_quantize_rows_at_any_address(gpu):
    torch = gpu
    for n in (20, 1100):
        x = _rows(torch, 9, 0, n, 701)
        for lo, hi in ((1, 513), (2, 642), (5, 701), (7, 71)):
            _check_quantized(torch, x[:, lo:hi])


def _int8(torch, seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def _check_product(torch, dtype, xq, x_scales, w, w_scales, K, out=None):
    from cpm.cu_amd import ops
    weight = ops.Int8Weight(w, w_scales)
    got = ops.int8_linear(xq, x_scales, weight, out=out)
    torch.cuda.synchronize()
    ref = torch.matmul(xq[:, :K].double(), w.double().t().contiguous())  # whole numbers below 2^53
    ref = ref * x_scales.double()[:, None] * w_scales.double()[None, :]
    # the sum's rounding to 32 bits, the scales' product and the last product: 3 * 2^-24 of the value
    _close(got.view(_types(torch, dtype)), ref, dtype, ref.abs() * 2.0 ** -22)
    return got


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n, V, K", [
    (1, 1, 1), (1, 16, 64), (1, 4608, 4096), (2, 17, 65), (9, 100, 127), (16, 4096, 512), (17, 33, 64), (31, 1000, 200), (33, 257, 4099), (60, 8192, 4096), (64, 64, 64), (65, 512, 1000), (100, 4096, 128),
    (128, 1024, 2048), (129, 48, 320), (255, 300, 192), (256, 256, 256), (257, 258, 259), (333, 1229, 4099), (513, 2000, 640), (1000, 1, 100), (1024, 1024, 64), (2047, 777, 1111), (4100, 512, 384)])
def test_int8_linear(gpu, set_option, dtype, n, V, K):
    torch = gpu
    set_option("dtype", dtype)
    padded = (K + 63) // 64 * 64
    xq = _int8(torch, n + K, n, padded)  # (columns behind K are noise: they do not matter)
    w = _int8(torch, V + K, V, K)
    g = torch.Generator(device="cuda").manual_seed(9)
    x_scales, w_scales = (torch.empty(m, device="cuda").uniform_(0.5, 1.0, generator=g) * s for m, s in ((n, 0.01), (V, 0.001)))
    w_scales[0] = 0.0
    got = _check_product(torch, dtype, xq, x_scales, w, w_scales, K)
    out = torch.full((n + 2, V), 7.0, dtype=torch.float16, device="cuda")
    same = _check_product(torch, dtype, xq, x_scales, w, w_scales, K, out=out[1:n + 1])
    assert same.data_ptr() == out[1:n + 1].data_ptr() and torch.equal(same.view(torch.int16), got.view(torch.int16)) and (out[0] == 7.0).all() and (out[n + 1] == 7.0).all()


@pytest.fixture
def int8_shape():
    from cpm.cu_amd import lib
    yield lambda i: lib.get().set_option(b"int8_linear_shape", i)
    lib.get().set_option(b"int8_linear_shape", -1)


@pytest.mark.parametrize("shape", range(8))
def test_int8_linear_shapes_agree(gpu, set_option, int8_shape, shape):
    """Each shape of the kernel at sizes about its tiles': odd rows, channels and steps, one step, many, and stores off 16 bytes."""
    torch = gpu
    from cpm.cu_amd import ops
    int8_shape(shape)
    names = set()
    for n, V, K, dtype in ((1, 1, 1, 0), (7, 300, 64, 1), (31, 130, 65, 0), (33, 127, 129, 0), (64, 128, 192, 1), (65, 257, 256, 0), (130, 513, 1000, 1), (255, 255, 1027, 0), (257, 259, 2048, 0), (300, 770, 4099, 1),
                           (600, 264, 640, 0), (3, 5003, 333, 0)):
        set_option("dtype", dtype)
        names.add(ops.int8_linear_plan(n, V, K)[0])
        xq, w = _int8(torch, n + K, n, (K + 63) // 64 * 64), _int8(torch, V + K, V, K)
        x_scales, w_scales = torch.rand(n, device="cuda") * 0.01, torch.rand(V, device="cuda") * 0.001
        out = torch.full((n + 1, V), 7.0, dtype=torch.float16, device="cuda")
        got = _check_product(torch, dtype, xq, x_scales, w, w_scales, K, out=out[:n])
        assert (out[n] == 7.0).all(), "written behind the last row"
        int8_shape(0)
        assert torch.equal(ops.int8_linear(xq, x_scales, ops.Int8Weight(w, w_scales)).view(torch.int16), got.view(torch.int16))
        int8_shape(shape)
    assert len(names) == 1


@pytest.mark.parametrize("shape", range(8))
def test_int8_linear_of_every_number_of_steps(gpu, int8_shape, shape):
    """1 to 20 steps of 64 columns and those about the waves' turns and the rings' lengths: whole numbers, compared with their exact products."""
    torch = gpu
    from cpm.cu_amd import ops
    n, V = 35, 70
    one = torch.ones(n, device="cuda")
    for steps in list(range(1, 21)) + [23, 24, 25, 31, 32, 33, 34, 47, 48, 49, 63, 64, 65, 66]:
        for K in (64 * steps, 64 * steps - 37):
            xq, w = _int8(torch, K, n, 64 * steps), _int8(torch, K + 1, V, K)
            ref = torch.matmul(xq[:, :K].double(), w.double().t().contiguous())
            scale = 2.0 ** -10  # sums of up to 4224 * 2^14 < 2^26.1 stay below fp16's 65504 (2^16)
            int8_shape(shape)
            got = ops.int8_linear(xq, one, ops.Int8Weight(w, torch.full((V,), scale, device="cuda")))
            torch.cuda.synchronize()
            assert torch.isfinite(ref * scale).all() and (ref.abs() * scale < 65504).all()
            _close(got, ref * scale, 0, ref.abs() * scale * 2.0 ** -24)  # the sum's one rounding to 32 bits


@pytest.mark.parametrize("n", [1, 20, 70, 200, 600])
def test_int8_linear_sums_to_the_ends_of_32_bits(gpu, n):
    """The longest rows of the largest values, and a row of scale NaN."""
    torch = gpu
    K, V = 131071, 20
    xq, w = torch.full((n, 131072), -128, dtype=torch.int8, device="cuda"), torch.full((V, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, ::2] = 127
    x_scales, w_scales = torch.full((n,), 2.0 ** -20, device="cuda"), torch.full((V,), 2.0 ** -2, device="cuda")
    _check_product(torch, 0, xq, x_scales, w, w_scales, K)
    from cpm.cu_amd import ops
    x_scales[0] = float("nan")
    got = ops.int8_linear(xq, x_scales, ops.Int8Weight(w, w_scales))
    assert got[0].isnan().all() and not got[1:].isnan().any()


@pytest.mark.parametrize("step", [1, 2])
def test_int8_weight_is_a_copy(gpu, step):
    """Neither the values nor the scales are the caller's memory, contiguous or not."""
    torch = gpu
    from cpm.cu_amd import ops
    V, K = 50, 128
    w, scales = _int8(torch, 1, V, K), torch.rand(V * step, device="cuda")[::step]
    weight = ops.Int8Weight(w, scales)
    xq, x_scales = _int8(torch, 2, 3, K), torch.rand(3, device="cuda")
    want = ops.int8_linear(xq, x_scales, weight)
    w.zero_()
    scales.fill_(5.0)
    assert torch.equal(ops.int8_linear(xq, x_scales, weight), want) and want.any()
    rows = torch.rand((V, 1), device="cuda")
    assert ops.Int8Weight(w, rows).scales.shape == (V,)


@pytest.mark.parametrize("n, shapes", [(5, (0, 1, 2)), (70, (3, 4, 5)), (300, (6, 7))])
def test_int8_linear_with_a_weight_beyond_2_gib(gpu, int8_shape, n, shapes):
    """Channels on both sides of byte 2^31 of the weight and at its ends, in every shape of the kernel."""
    torch = gpu
    from cpm.cu_amd import ops
    V, K = 131072 + 40, 16384
    w, xq = _int8(torch, 1, V, K), _int8(torch, 2, n, K)
    g = torch.Generator(device="cuda").manual_seed(3)
    x_scales, w_scales = (torch.empty(m, device="cuda").uniform_(0.5, 1.0, generator=g) * 0.001 for m in (n, V))
    weight = ops.Int8Weight(w, w_scales)
    assert weight.data.numel() > 2 ** 31
    some = torch.cat([torch.arange(0, 40), torch.arange(131072 - 300, V)]).cuda()
    ref = torch.matmul(xq.double(), w[some].double().t().contiguous()) * x_scales.double()[:, None] * w_scales.double()[some][None, :]
    for shape in (-1,) + shapes:
        int8_shape(shape)
        got = ops.int8_linear(xq, x_scales, weight)
        torch.cuda.synchronize()
        _close(got[:, some], ref, 0, ref.abs() * 2.0 ** -22)  # (as in _check_product)


@pytest.mark.parametrize("shape", [1, 4, 7])
def test_int8_linear_with_results_beyond_2_gib(gpu, int8_shape, shape):
    """Results on both sides of value 2^31 and of byte 2^31 (value 2^30), and the last ones."""
    torch = gpu
    from cpm.cu_amd import ops
    n, V, K = 32768 + 70, 65536, 64
    w, xq = _int8(torch, 1, V, K), _int8(torch, 2, n, K)
    x_scales, w_scales = torch.full((n,), 2.0 ** -8, device="cuda"), torch.full((V,), 2.0 ** -8, device="cuda")
    int8_shape(shape)
    got = ops.int8_linear(xq, x_scales, ops.Int8Weight(w, w_scales))
    torch.cuda.synchronize()
    assert got.numel() > 2 ** 31
    some = torch.cat([torch.arange(0, 20), torch.arange(16384 - 20, 16384 + 20), torch.arange(n - 100, n)]).cuda()
    ref = torch.matmul(xq[some].double(), w.double().t().contiguous()) * 2.0 ** -16
    _close(got[some], ref, 0, ref.abs() * 2.0 ** -22)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n", [1, 20, 70, 400])
def test_int8_linear_with_scales_at_the_ends_of_32_bits(gpu, set_option, dtype, n):
    """The scales' product comes first: infinite or below the smallest float it is the result's too, whatever the sum; up to there all is finite."""
    torch = gpu
    from cpm.cu_amd import ops
    set_option("dtype", dtype)
    V, K = 40, 64
    xq, w = torch.ones((n, K), dtype=torch.int8, device="cuda"), torch.ones((V, K), dtype=torch.int8, device="cuda")
    w[1] = -1
    w[2, ::2] = -1  # the sum is 0
    sums = torch.tensor([64.0, -64.0, 0.0] + [64.0] * (V - 3), device="cuda").expand(n, V)
    for s, sw, want in ((2.0 ** 100, 2.0 ** 100, sums * float("inf")), (2.0 ** -100, 2.0 ** -100, sums * 0.0), (2.0 ** 100, 2.0 ** -100, sums), (2.0 ** -126, 2.0 ** 120, sums * 2.0 ** -6), (0.0, 5.0, sums * 0.0)):
        got = ops.int8_linear(xq, torch.full((n,), s, device="cuda"), ops.Int8Weight(w, torch.full((V,), sw, device="cuda"))).view(_types(torch, dtype)).float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


def test_int8_weight_from_16_bits(gpu):
    """Weights and rows quantised here: the product is near the 16-bit one, by at most half a step of either side's 8 bits a column."""
    torch = gpu
    from cpm.cu_amd import ops
    n, V, K = 20, 300, 500
    x, w = _rows(torch, 1, 0, n, K), _rows(torch, 2, 0, V, K)
    xq, xs = ops.quantize_rows(x)
    y = ops.int8_linear(xq, xs, ops.Int8Weight.quantized(w))
    ref = x.double() @ w.double().t().contiguous()
    a, b = x.double().abs(), w.double().abs()
    sx, sw = a.amax(1, keepdim=True) / 254.0, b.amax(1) / 254.0  # half a step
    limit = sx * b.sum(1) + a.sum(1, keepdim=True) * sw + K * sx * sw
    assert ((y.double() - ref).abs() <= limit * 1.001 + ref.abs() * 2.0 ** -10).all()


# ---- together ----

def _attend(torch, q, k, v):
    """Causal attention of the last rows in 64 bits: q [T, Hq, D] behind k, v [S, Hkv, D]."""
    T, Hq, _ = q.shape
    S, Hkv, _ = k.shape
    k, v = (t.double().repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    score = torch.matmul(q.double().transpose(0, 1), k.permute(1, 2, 0).contiguous()) / D ** 0.5
    seen = torch.arange(S, device=q.device)[None, :] <= (S - T + torch.arange(T, device=q.device))[:, None]
    p = torch.softmax(score.masked_fill(~seen, float("-inf")), -1)
    return torch.matmul(p, v.transpose(0, 1).contiguous()).transpose(0, 1)


def test_a_batch_from_hidden_rows_to_attention(gpu):
    """Three requests over several steps -- prompts, chunks, decode, one that ends and gives its pages to another: hidden rows to 8 bits,
    the fused projection, rotary positions, the slots of the batch's pages, attention of each request on its table."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    H, Hq, Hkv, R, max_rows = 512, 8, 2, 3, 192
    cache = PagedKVCache(1, Hkv, 6, fill=0.0)
    batch = ops.PageBatch(cache, R, 3)
    weight = ops.Int8Weight.quantized(_rows(torch, 11, 0, (Hq + 2 * Hkv) * D, H) * 0.05)
    inv_freq, magnitude = ops.rope_frequencies(D, 10000.0, dict(type="yarn", factor=4.0, original=128))
    inv_freq = inv_freq.cuda()
    history = {r: [] for r in range(R)}
    for step, new in enumerate([[100, 60, 0], [100, 1, 30], [60, 1, 1], [1, -1, 1], [1, 100, 1], [1, 100, 1]]):
        hidden = _rows(torch, 20 + step, 0, max_rows + 80, H)[:max_rows]
        where = batch.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), max_rows + 80)
        rows = sum(max(n, 0) for n in new)
        assert batch.counts[1].item() == 0 and where["row_offsets"][-1].item() == rows
        n = max_rows + 80
        xq, scales = ops.quantize_rows(torch.cat([hidden, hidden[:80]]))
        qkv = ops.int8_linear(xq, scales, weight)
        q, k, v = qkv[:, :Hq * D].view(n, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(n, Hkv, D), qkv[:, (Hq + Hkv) * D:].view(n, Hkv, D)
        q_rot = ops.kv_append_slots(cache, 0, k, v, where["slots"], q=q, positions=where["positions"], inv_freq=inv_freq, magnitude=magnitude)
        offsets = where["row_offsets"].tolist()
        for r in range(R):
            if new[r] < 0:
                history[r] = []
                continue
            if new[r] == 0:
                continue
            at = slice(offsets[r], offsets[r + 1])
            start = sum(t[0].shape[0] for t in history[r])
            positions = torch.arange(start, start + new[r], dtype=torch.int32, device="cuda")
            assert torch.equal(where["positions"][at], positions)
            history[r].append((_turned(torch, k[at], positions, inv_freq, False, magnitude)[0], v[at].clone()))
            out = ops.tree_attention(q_rot[at], batch.cache_of(r), 0, batch.kv_lens[r:r + 1], start + new[r])
            keys, values = (torch.cat([t[i] for t in history[r]]) for i in (0, 1))
            ref = _attend(torch, _turned(torch, q[at], positions, inv_freq, False, magnitude)[0], keys, values)
            torch.cuda.synchronize()
            # keys, queries, probabilities and results in fp16: the attention's own tolerance
            assert (out.double() - ref).abs().max() <= 2e-2
    # page 0 of the stack is never lost: what is held and what is free are all pages, once each
    held, free = batch.held.tolist(), batch.counts[0].item()
    pages = [p for r in range(R) for p in batch.block_tables[r, :held[r]].tolist()] + batch.free_pages[:free].tolist()
    assert sorted(pages) == list(range(6))


def _attention_and_limit(torch, q, k, v, seen):
    """Attention of q [T, Hq, D] on keys and values as they lie in the cache [S, Hkv, D] in 64 bits, and how far the kernel's may be off:
    the probabilities and the splits' sums are rounded to fp16 (2^-11 each, of a sum of magnitudes; their sum in the denominator as well), the
    result once more; what underflows there is below 2^-25; a score is a sum of 128 products in 32 bits with two factors, and shows
    in its probability, in the largest one's and in their sum; the products' sum has S terms."""
    S, group = k.shape[0], q.shape[1] // k.shape[1]
    q, k, v = q.double().transpose(0, 1), k.double().repeat_interleave(group, 1).transpose(0, 1), v.double().repeat_interleave(group, 1).transpose(0, 1).contiguous()
    kt = k.transpose(1, 2).contiguous()
    p = torch.softmax((torch.matmul(q, kt) / D ** 0.5).masked_fill(~seen, float("-inf")), -1)
    delta = (torch.matmul(q.abs(), kt.abs()) / D ** 0.5).amax(-1, keepdim=True) * (128 + 4) * 2.0 ** -24
    ref, weight = torch.matmul(p, v), torch.matmul(p, v.abs())
    limit = weight * (3 * 2.0 ** -11 + 4 * delta + S * 2.0 ** -24) + ref.abs() * 2.0 ** -11 + 2.0 ** -25 * (torch.matmul(seen.double(), v.abs()) + 2)
    return ref.transpose(0, 1), limit.transpose(0, 1)


def test_prompts_longer_than_an_attention_call(gpu):
    """Two prompts and their next chunks, planned and appended whole, attended in pieces of up to 128 rows whose length is their last row's
    position + 1."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    Hq, Hkv, max_rows = 8, 2, 512
    cache = PagedKVCache(1, Hkv, 7)
    batch = ops.PageBatch(cache, 2, 4)
    inv_freq, past = _freq(torch, 64), [0, 0]
    for step, new in enumerate(([300, 129], [200, 1], [1, 257])):
        x = _rows(torch, step, 0, max_rows, (Hq + 2 * Hkv) * D)
        q, k, v = (t.view(max_rows, -1, D) for t in x.split([Hq * D, Hkv * D, Hkv * D], 1))
        where = batch.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), max_rows)
        q_rot = ops.kv_append_slots(cache, 0, k, v, where["slots"], q=q, positions=where["positions"], inv_freq=inv_freq)
        k_rot = ops.rope_rows(k, None, where["positions"], inv_freq)[0]
        first = 0
        for r, n in enumerate(new):
            end, view, out = first + n, batch.cache_of(r), torch.full((n, Hq, D), float("nan"), dtype=torch.float16, device="cuda")
            for a in range(first, end, 128):
                b = min(a + 128, end)
                ops.tree_attention(q_rot[a:b], view, 0, where["positions"][b - 1:b] + 1, past[r] + b - first, out=out[a - first:b - first])
            torch.cuda.synchronize()
            keys, values = view.read_logical(0, 0, past[r] + n)
            assert torch.equal(keys[past[r]:], k_rot[first:end]) and torch.equal(values[past[r]:], v[first:end])
            seen = torch.arange(past[r] + n, device="cuda")[None, :] <= torch.arange(past[r], past[r] + n, device="cuda")[:, None]
            ref, limit = _attention_and_limit(torch, q_rot[first:end], keys, values, seen)
            assert ((out.double() - ref).abs() <= limit).all()
            past[r] += n
            first = end
    assert batch.kv_lens.tolist() == past == [501, 387]


def test_trees_on_a_batch_and_rows_that_are_not_accepted(gpu, orc):
    """Two requests, each with a draft tree a step: rows in places that follow each other, rotary positions by depth, masked attention, acceptance,
    compaction in the request's table, and the length set back to what was accepted before the next plan."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    Hq, Hkv, max_rows, vocab = 8, 2, 300, 1000
    cache = PagedKVCache(1, Hkv, 6)
    batch = ops.PageBatch(cache, 2, 3)
    inv_freq = _freq(torch, 64)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    history = [(torch.empty((0, Hkv, D), dtype=torch.float16, device="cuda"),) * 2 for _ in range(2)]

    def append(seed, new, positions=None):
        x = _rows(torch, seed, 0, max_rows, (Hq + 2 * Hkv) * D)
        q, k, v = (t.view(max_rows, -1, D) for t in x.split([Hq * D, Hkv * D, Hkv * D], 1))
        where = batch.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), max_rows)
        positions = where["positions"] if positions is None else positions
        q_rot = ops.kv_append_slots(cache, 0, k, v, where["slots"], q=q, positions=positions, inv_freq=inv_freq)
        return where, q_rot, ops.rope_rows(k, None, positions, inv_freq)[0], v

    _, _, k_rot, v = append(1, [40, 250])
    history = [(k_rot[:40], v[:40]), (k_rot[40:290], v[40:290])]
    accepted = []
    for step in range(4):
        past = [h[0].shape[0] for h in history]
        trees = [synth.random_tree(T, 10 * step + r, max_children=3, max_depth=6) for r, T in enumerate((7, 20))]
        cached = batch.kv_lens.clone()  # (the plan counts the trees' rows)
        positions = np.full(max_rows, -1, np.int32)
        positions[:27] = np.concatenate([t.positions(P) for t, P in zip(trees, past)])
        where, q_rot, k_rot, v = append(10 + step, [7, 20], dev(positions))
        assert where["positions"][:27].tolist() == [P + i for t, P in zip(trees, past) for i in range(t.T)]
        for r, (tree, first) in enumerate(zip(trees, (0, 7))):
            T, rows, view, mask = tree.T, slice(first, first + tree.T), batch.cache_of(r), dev(tree.mask.view(np.int64))
            out = ops.tree_attention(q_rot[rows], view, 0, batch.kv_lens[r:r + 1], past[r] + T, mask)
            torch.cuda.synchronize()
            keys, values = view.read_logical(0, 0, past[r] + T)
            assert torch.equal(keys, torch.cat([history[r][0], k_rot[rows]])) and torch.equal(values, torch.cat([history[r][1], v[rows]]))
            bits = (tree.mask.reshape(T, -1)[:, :1] >> np.arange(T, dtype=np.uint64)[None, :]) & np.uint64(1)
            seen = torch.cat([torch.ones((T, past[r]), dtype=torch.bool), torch.from_numpy(bits.astype(bool))], 1).cuda()
            ref, limit = _attention_and_limit(torch, q_rot[rows], keys, values, seen)
            assert ((out.double() - ref).abs() <= limit).all()
            gt = synth.rng(step, 60 + r).integers(0, vocab, T).astype(np.int32)
            ids, _ = synth.draft_ids_for_accept(tree, gt, min(step, int(tree.depth.max())), vocab, 100 * step + r)
            a, _, path = orc.tree_accept(ids, gt, tree.positions(past[r]), past[r], tree.mask, tree.parent)
            pred = dev(ids.astype(np.int32))
            best = ops.tree_accept(pred, dev(gt), dev(tree.positions(past[r])), cached[r:r + 1], mask, dev(tree.parent))
            ops.kv_compact(view, pred, dev(gt), cached[r:r + 1], best, T)
            batch.kv_lens[r:r + 1] = cached[r:r + 1] + best[:1]
            torch.cuda.synchronize()
            assert int(best[0]) == a
            accepted.append(a)
            history[r] = tuple(torch.cat([h, new[rows][torch.from_numpy(np.asarray(path[:a], np.int64)).cuda()]]) for h, new in zip(history[r], (k_rot, v)))
            assert batch.kv_lens[r].item() == past[r] + a
            keys, values = view.read_logical(0, 0, past[r] + a)
            assert torch.equal(keys, history[r][0]) and torch.equal(values, history[r][1])
    assert min(accepted) == 1 and max(accepted) >= 3 and batch.held.tolist() == [1, 2]
    pages = [p for r in range(2) for p in batch.block_tables[r, :batch.held[r]].tolist()] + batch.free_pages[:batch.counts[0]].tolist()
    assert sorted(pages) == list(range(6))


def test_batch_operators_in_a_graph(gpu):
    """A captured step on static buffers, replayed with other lengths and rows, between eager calls: each replay as the eager call."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    H, Hq, Hkv, R, max_rows, pages = 256, 4, 2, 5, 128, 40
    weight = ops.Int8Weight.quantized(_rows(torch, 11, 0, (Hq + 2 * Hkv) * D, H) * 0.05)
    inv_freq = _freq(torch, 32)

    def fresh():
        cache = PagedKVCache(1, Hkv, pages)
        return cache, ops.PageBatch(cache, R, 8)

    def step(batch, new, hidden, q_out):
        where = batch.plan(new, max_rows)
        xq, scales = ops.quantize_rows(hidden)
        qkv = ops.int8_linear(xq, scales, weight)
        q, k, v = qkv[:, :Hq * D].view(-1, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(-1, Hkv, D), qkv[:, (Hq + Hkv) * D:].view(-1, Hkv, D)
        ops.kv_append_slots(batch.cache, 0, k, v, where["slots"], q=q, q_out=q_out, positions=where["positions"], inv_freq=inv_freq, interleaved=True)
        return where

    cache, batch = fresh()
    new, hidden = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros((max_rows, H), dtype=torch.float16, device="cuda")
    q_out = torch.zeros((max_rows, Hq, D), dtype=torch.float16, device="cuda")
    step(batch, new, hidden, q_out)  # (loads the kernels outside the capture; a step of no rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        where = step(batch, new, hidden, q_out)
    cache2, batch2 = fresh()
    q_out2 = torch.zeros_like(q_out)
    for i, lens in enumerate([[30, 1, 0, 50, 7], [1, 1, 1, 1, 1], [1, 1, -1, 1, 60], [0, 0, 0, 0, 0], [1, -1, 20, 1, 100]]):
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        hidden.copy_(_rows(torch, i, 0, max_rows, H))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(batch2, new, hidden, q_out2)
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(where[name], eager[name]), name
        assert torch.equal(cache.k[0], cache2.k[0]) and torch.equal(cache.v[0], cache2.v[0]) and torch.equal(q_out, q_out2)
        assert torch.equal(batch.block_tables, batch2.block_tables) and torch.equal(batch.kv_lens, batch2.kv_lens)
    # 30 + 1 + 1 + 0 + 1; ended; ended, then 0 + 20; 50 + 1 + 1 + 0 + 1; 7 + 1 + 60 + 0 + 100; never more than max_rows rows or the stack's pages
    assert batch.counts[1].item() == 0 and batch.kv_lens.tolist() == [33, 0, 20, 53, 168]


def test_batch_operators_on_another_stream(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    x, w = _rows(torch, 1, 0, 300, 1000), ops.Int8Weight.quantized(_rows(torch, 2, 0, 500, 1000))
    positions = torch.arange(300, dtype=torch.int32, device="cuda")
    calls = lambda: (ops.int8_linear(*ops.quantize_rows(x), w), *ops.rope_rows(x[:, :896].view(300, 7, 128), x[:, :128].view(300, 1, 128), positions, _freq(torch, 64)))  # noqa: E731
    want = calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2000000)  # (what the side stream still has to do when the host is done with the calls)
        x.neg_()
        got = calls()
    side.synchronize()
    assert torch.equal(got[0], -want[0]) and torch.equal(got[1], -want[1]) and torch.equal(got[2], -want[2])


def test_batch_operators_in_two_graphs_at_once(gpu):
    """Two captured steps on data of their own, replayed side by side on two streams and between eager calls: they share no memory."""
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    Hq, Hkv, R, n = 4, 2, 3, 700
    weight = ops.Int8Weight.quantized(_rows(torch, 3, 0, (Hq + 2 * Hkv) * D, 900) * 0.05)
    inv_freq = _freq(torch, 64)

    class Step:
        def __init__(self, seed):
            self.cache = PagedKVCache(1, Hkv, 12, fill=0.0)
            self.batch = ops.PageBatch(self.cache, R, 4)
            self.hidden = _rows(torch, seed, 0, n, 900)
            self.new = torch.tensor([100 + seed, 200, 300 - seed], dtype=torch.int32, device="cuda")
            self.q = torch.zeros((n, Hq, D), dtype=torch.float16, device="cuda")
            self.free = self.batch.free_pages.clone()

        def again(self):
            self.batch._state.zero_()
            self.batch._state[0] = 12
            self.batch.free_pages.copy_(self.free)

        def run(self):
            where = self.batch.plan(self.new, n)
            qkv = ops.int8_linear(*ops.quantize_rows(self.hidden), weight)
            q, k, v = (x.view(n, -1, D) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
            ops.kv_append_slots(self.cache, 0, k, v, where["slots"], q=q, q_out=self.q, positions=where["positions"], inv_freq=inv_freq)

        def results(self):
            return [t.clone() for t in (self.q, self.cache.k[0], self.cache.v[0], self.batch.block_tables, self.batch.kv_lens, self.batch.counts)]

    steps, streams, graphs, want = [Step(1), Step(2)], [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    for s in steps:
        s.run()
        want.append(s.results())
        s.again()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run()
        graphs.append(graph)
    for turn in range(4):
        for s in steps:
            s.again()
            s.q.zero_()
            s.cache.k[0].zero_()
            s.cache.v[0].zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        other = ops.int8_linear(*ops.quantize_rows(steps[turn % 2].hidden), weight)
        torch.cuda.synchronize()
        assert torch.isfinite(other).all()
        for s, w in zip(steps, want):
            for got, ref in zip(s.results(), w):
                assert torch.equal(got, ref)


def test_no_rows_at_all(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    h = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda")  # noqa: E731
    none, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda")
    cache = PagedKVCache(1, 2, 2, fill=3.0)
    assert ops.rope_rows(h(0, 4, D), h(0, 2, D), none, f)[1].shape == (0, 2, D)
    assert ops.rope_rows(h(3, 0, D), None, torch.zeros(3, dtype=torch.int32, device="cuda"), f)[0].shape == (3, 0, D)
    assert ops.kv_append_slots(cache, 0, h(0, 2, D), h(0, 2, D), none) is None
    assert ops.kv_append_slots(cache, 0, h(0, 2, D), h(0, 2, D), none, q=h(0, 4, D), positions=none, inv_freq=f).shape == (0, 4, D)
    xq, scales = ops.quantize_rows(h(0, 100))
    assert xq.shape == (0, 128) and scales.shape == (0,)
    assert ops.int8_linear(xq, scales, ops.Int8Weight(torch.ones((5, 100), dtype=torch.int8, device="cuda"), f[:5])).shape == (0, 5)
    torch.cuda.synchronize()
    assert (cache.k[0] == 3.0).all() and (cache.v[0] == 3.0).all()


def test_wrong_tensors_are_refused(gpu):
    torch = gpu
    from cpm.cu_amd import ops
    from cpm.cu_amd.kvcache import PagedKVCache
    h, i, f = torch.zeros((4, 2, D), dtype=torch.float16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda")
    cache = PagedKVCache(1, 2, 2)
    w = ops.Int8Weight(torch.zeros((16, 64), dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda"))
    b = torch.zeros((4, 64), dtype=torch.int8, device="cuda")
    for call in (lambda: ops.rope_rows(h.float(), None, i, f), lambda: ops.rope_rows(h, None, i.long(), f), lambda: ops.rope_rows(h, None, i[:3], f), lambda: ops.rope_rows(h, None, i, f.double()),
                 lambda: ops.rope_rows(h, h[:3], i, f), lambda: ops.rope_rows(h.transpose(0, 1), None, i[:2], f), lambda: ops.rope_rows(h, None, i, f, q_out=h[:, :1]), lambda: ops.rope_rows(h[..., ::2], None, i, f[:32]),
                 lambda: ops.kv_append_slots(cache, 0, h, h[:, :1], i), lambda: ops.kv_append_slots(cache, 0, h, h, i[:3]), lambda: ops.kv_append_slots(cache, 0, h, h, i, positions=i),
                 lambda: ops.kv_append_slots(cache, 0, h[..., :64], h[..., :64], i), lambda: ops.kv_append_slots(cache, 0, h, h, i, q=h[:2], positions=i, inv_freq=f),
                 lambda: ops.quantize_rows(h), lambda: ops.quantize_rows(torch.zeros((4, 64), device="cuda")), lambda: ops.quantize_rows(h[:, 0].t()), lambda: ops.quantize_rows(h[:, 0, :0]),
                 lambda: ops.int8_linear(b[:, :32], f[:4], w), lambda: ops.int8_linear(b, f[:3], w), lambda: ops.int8_linear(b, f[:4], w, out=h[:, 0]), lambda: ops.int8_linear(b.short(), f[:4], w),
                 lambda: ops.batch_tables(i, i[:3], i.view(4, 1), i, i, i[:2], 4), lambda: ops.batch_tables(i, i, i, i, i, i[:2], 4), lambda: ops.batch_tables(i, i, i.view(4, 1), i, i, i[:3], 4),
                 lambda: ops.batch_tables(i.long(), i, i.view(4, 1), i, i, i[:2], 4)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(ValueError, match="q is rotated here"):
        ops.kv_append_slots(cache, 0, h, h, i, q=h)
    with pytest.raises(ValueError, match="closer"):
        ops.rope_rows(h[:1].expand(4, 2, D), None, i, f)
    with pytest.raises(ValueError, match="neither in place"):
        x = torch.zeros((5, 2, D), dtype=torch.float16, device="cuda")
        ops.rope_rows(x[:4], None, i, f, q_out=x[1:])
