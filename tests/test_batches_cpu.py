"""Batches on the CPU: what the operators refuse before any device call, and the rotary frequencies of long contexts."""
import ctypes
import math

import numpy as np
import pytest

P = ctypes.c_void_p
A, B, C, D, E, F = (P(1 << 20 << i) for i in range(6))  # never looked at: far apart, on 16 bytes


def _lib():
    from cpm.cu_amd import lib
    return lib.get()


def _tables(**kw):
    a = dict(kv=P(1 << 32), new=P(2 << 32), n=4, tables=P(3 << 32), blocks=8, held=P(4 << 32), free=P(5 << 32), pages=64, counts=P(6 << 32), kv_out=P(7 << 32), held_out=P(8 << 32),
             counts_out=P(9 << 32), offsets=P(10 << 32), positions=P(11 << 32), slots=P(12 << 32), rows=100)
    a.update(kw)
    _lib().batch_tables(a["kv"], a["new"], a["n"], a["tables"], a["blocks"], a["held"], a["free"], a["pages"], a["counts"], a["kv_out"], a["held_out"], a["counts_out"], a["offsets"],
                        a["positions"], a["slots"], a["rows"], None)


@pytest.mark.parametrize("kw, match", [
    (dict(kv=None), "null"), (dict(counts_out=None), "null"), (dict(positions=None), "null"), (dict(slots=None), "null"),
    (dict(n=0), "0 requests"), (dict(n=4097), "4097 requests"), (dict(blocks=0), "max_blocks=0"), (dict(blocks=(1 << 18) + 1), "max_blocks"),
    (dict(pages=0), "num_pages=0"), (dict(pages=1 << 23), "num_pages"), (dict(rows=-1), "max_rows=-1"), (dict(rows=(1 << 29) + 1), "max_rows"),
    (dict(kv_out=P(1 << 32)), "memory of an input"), (dict(held_out=P((4 << 32) + 12)), "memory of an input"), (dict(counts_out=P(6 << 32)), "memory of an input"),
    (dict(slots=P((3 << 32) + 4 * 4 * 8 - 4)), "memory of an input"), (dict(positions=P((5 << 32) - 396)), "memory of an input")])
def test_batch_tables_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _tables(**kw)


@pytest.mark.parametrize("kw, match", [
    (dict(kv=P(3 << 32)), "tables or the stack share"), (dict(held=P((3 << 32) + 4 * 4 * 8 - 4)), "tables or the stack share"), (dict(new=P((3 << 32) - 12)), "tables or the stack share"),
    (dict(counts=P((5 << 32) + 4 * 63)), "tables or the stack share"), (dict(kv=P((5 << 32) - 4)), "tables or the stack share"), (dict(free=P(3 << 32)), "tables or the stack share"),
    (dict(free=P((3 << 32) - 4 * 63)), "tables or the stack share"), (dict(held_out=P(7 << 32)), "two outputs share"), (dict(counts_out=P((7 << 32) + 12)), "two outputs share"),
    (dict(offsets=P((8 << 32) - 16)), "two outputs share"), (dict(slots=P(11 << 32)), "two outputs share"), (dict(slots=P((11 << 32) - 4)), "two outputs share")])
def test_batch_tables_refuses_memory_that_is_shared(kw, match):
    """What one workgroup writes another one would read, or write too."""
    with pytest.raises(ValueError, match=match):
        _tables(**kw)


def _rope(**kw):
    a = dict(pos=A, freq=B, rotary=128, il=0, m=1.0, tr=0, q=P(1 << 32), qs=4096, qo=P(2 << 32), qos=4096, hq=32, k=P(3 << 32), ks=256, ko=P(4 << 32), kos=256, hkv=2, dim=128, n=60)
    a.update(kw)
    _lib().rope_rows(a["pos"], a["freq"], a["rotary"], a["il"], ctypes.c_float(a["m"]), a["tr"], a["q"], a["qs"], a["qo"], a["qos"], a["hq"], a["k"], a["ks"], a["ko"], a["kos"], a["hkv"], a["dim"], a["n"], None)


@pytest.mark.parametrize("kw, match", [
    (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(q=None), "null"), (dict(ko=None), "null"), (dict(rotary=0), "rotary_dim=0"), (dict(rotary=127), "rotary_dim=127"),
    (dict(rotary=130), "rotary_dim=130"), (dict(dim=127), "head_dim=127"), (dict(dim=258), "head_dim=258"), (dict(n=-1), "n=-1"), (dict(hq=1025, qs=1 << 20, qos=1 << 20), "1025 heads of q"),
    (dict(hkv=-1), "-1 heads of k"), (dict(qs=4095), "rows of q closer"), (dict(kos=255), "rows of k closer"), (dict(qo=P((1 << 32) + 256)), "results of q"),
    (dict(qo=P(1 << 32), qos=8192), "results of q"), (dict(ko=P((3 << 32) + 2 * 60 * 256 - 16)), "results of k"), (dict(m=math.inf), "magnitude"), (dict(m=math.nan), "magnitude")])
def test_rope_rows_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _rope(**kw)


Q, K = 1 << 32, 3 << 32  # where _rope has q and k, 60 rows of 4096 and of 256 values


@pytest.mark.parametrize("kw", [
    dict(qo=P(K), qos=4096), dict(qo=P(K - 2 * 59 * 4096)), dict(qo=P(K + 2 * (59 * 256 + 255)), qos=4096), dict(ko=P(Q)), dict(ko=P(Q + 2 * (59 * 4096 + 4095))), dict(qo=P(5 << 32), ko=P(5 << 32)),
    dict(k=P(Q + 2 * 4095), ks=4352, qs=4352, qo=P(Q), qos=4352, ko=P(7 << 32)),      # the last value of each row of q is the first of k's
    dict(k=P(Q + 2 * 4097), ks=4352, qs=4352, qo=P(Q), qos=4352, ko=P(7 << 32)),      # the last of k's the first of the next row of q
    dict(qo=P(5 << 32), qos=4352, ko=P((5 << 32) + 2 * 4000), kos=4352), dict(qo=P(5 << 32), qos=5000, ko=P((5 << 32) + 2 * 4096), kos=5001)])
def test_rope_rows_refuses_results_in_the_other_rows(kw):
    """Workgroups would read rows that others have turned already, or write the same memory."""
    with pytest.raises(ValueError, match="rope_rows: results lie in the memory of the other rows"):
        _rope(**kw)


def test_empty_calls_are_no_calls():
    """No rows or heads: nothing to do, and no device is asked for."""
    _rope(n=0)
    _rope(hq=0, hkv=0)
    _append(n=0)
    _append(n=0, k=None, v=None, slots=None, q=None, qo=None, pos=None)
    _lib().quantize_rows(A, 64, 0, 64, B, C, None)
    _lib().int8_linear(A, B, C, D, 0, 16, 64, E, None)


def _append(**kw):
    a = dict(kp=P(1 << 32), vp=P(2 << 32), pages=4, slots=A, k=P(3 << 32), ks=256, v=P(4 << 32), vs=256, n=60, hkv=2, pos=B, freq=C, rotary=128, il=0, m=1.0, q=P(5 << 32), qs=4096, qo=P(6 << 32), qos=4096, hq=32)
    a.update(kw)
    _lib().kv_append_slots(a["kp"], a["vp"], a["pages"], a["slots"], a["k"], a["ks"], a["v"], a["vs"], a["n"], a["hkv"], a["pos"], a["freq"], a["rotary"], a["il"], ctypes.c_float(a["m"]), a["q"], a["qs"],
                           a["qo"], a["qos"], a["hq"], None)


@pytest.mark.parametrize("kw, match", [
    (dict(kp=None), "null"), (dict(slots=None), "null"), (dict(v=None), "null"), (dict(q=None), "null"), (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(pages=0), "num_pages=0"),
    (dict(pages=1 << 23), "num_pages"), (dict(n=-1), "n=-1"), (dict(hkv=0), "Hkv=0"), (dict(rotary=24), "multiple of 16"), (dict(rotary=144), "rotary_dim=144"), (dict(pos=None, freq=None), "q is rotated here"),
    (dict(ks=255), "closer"), (dict(vs=248), "closer"), (dict(k=P((3 << 32) + 8)), "16 bytes"), (dict(vs=260), "16 bytes"), (dict(qs=4100), "16 bytes"), (dict(vp=P((2 << 32) + 2)), "16 bytes"), (dict(m=math.inf), "magnitude")])
def test_kv_append_slots_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


@pytest.mark.parametrize("kw, match", [
    (dict(qo=P(3 << 32)), "results of q lie in the memory of k or v"), (dict(qo=P((4 << 32) - 2 * 59 * 4096)), "results of q lie in the memory of k or v"),
    (dict(qo=P((4 << 32) + 2 * (59 * 256 + 248))), "results of q lie in the memory of k or v"),
    # a fused projection in place, its k one piece too early, its v one too late for the row
    (dict(q=P(5 << 32), qo=P(5 << 32), qs=4608, qos=4608, k=P((5 << 32) + 2 * 4088), ks=4608), "results of q lie in the memory of k or v"),
    (dict(q=P(5 << 32), qo=P(5 << 32), qs=4608, qos=4608, v=P((5 << 32) + 2 * 4360), vs=4608), "results of q lie in the memory of k or v"),
    (dict(vp=P(1 << 32)), "pool share memory"), (dict(vp=P((1 << 32) + 4 * 2 * 256 * 128 * 2 - 16)), "pool share memory"), (dict(kp=P((2 << 32) + 16)), "pool share memory")])
def test_kv_append_slots_refuses_memory_that_is_shared(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


def test_int8_operators_refuse():
    L = _lib()
    for args in ((None, 64, 1, 64, B, C), (A, 64, 1, 64, None, C), (A, 64, 1, 64, B, None), (A, 64, -1, 64, B, C), (A, 64, 0, 0, B, C), (A, 64, 1, 0, B, C), (A, 1 << 20, 1, 131072, B, C), (A, 63, 1, 64, B, C),
                 (A, 64, 1, 64, P(24), C), (A, 64, 1 << 24, 64, B, C)):
        with pytest.raises(ValueError, match="quantize_rows"):
            L.quantize_rows(*args, None)
    for args in ((None, 16, 64, B), (A, 16, 64, None), (A, 16, 64, A), (A, 0, 64, B), (A, 16, 0, B), (A, 16, 131072, B), (A, 16, 64, P(8))):
        with pytest.raises(ValueError, match="int8_weight_tile"):
            L.int8_weight_tile(*args, None)
    for args in ((None, B, C, D, 1, 16, 64, E), (A, None, C, D, 1, 16, 64, E), (A, B, None, D, 1, 16, 64, E), (A, B, C, None, 1, 16, 64, E), (A, B, C, D, 1, 16, 64, None), (A, B, C, D, -1, 16, 64, E),
                 (A, B, C, D, 1, 0, 64, E), (A, B, C, D, 1, 16, 0, E), (A, B, C, D, 1, 16, 131072, E), (P(8), B, C, D, 1, 16, 64, E), (A, B, P(8), D, 1, 16, 64, E)):
        with pytest.raises(ValueError, match="int8_linear"):
            L.int8_linear(*args, None)
    assert L.raw.cpmcu_int8_weight_bytes(17, 65) == 2 * 2 * 1024 and L.raw.cpmcu_int8_weight_bytes(0, 65) == 0


@pytest.mark.parametrize("xq, scales", [(1 << 32, 9 << 32), ((1 << 32) + 2 * (9 * 200 + 100) - 16, 9 << 32), ((1 << 32) - 10 * 128 + 16, 9 << 32), (8 << 32, 1 << 32), (8 << 32, (1 << 32) - 36),
                                        (8 << 32, 8 << 32), (8 << 32, (8 << 32) + 1276), ((9 << 32) + 32, 9 << 32)])
def test_quantize_rows_refuses_memory_that_is_shared(xq, scales):
    """10 rows of 100 values, 200 apart, at 1 << 32."""
    with pytest.raises(ValueError, match="quantize_rows: the results lie"):
        _lib().quantize_rows(P(1 << 32), 200, 10, 100, P(xq), P(scales), None)


@pytest.mark.parametrize("n", [1, 10, 600])
def test_int8_linear_refuses_results_over_its_inputs(n):
    V, K = 100, 100
    at, sizes = [P(i << 32) for i in (1, 2, 3, 4)], (n * 128, 4 * n, 112 * 128, 4 * V)
    for i, size in enumerate(sizes):
        for out in (i + 1 << 32, (i + 1 << 32) + size - 2, (i + 1 << 32) - 2 * n * V + 2):
            with pytest.raises(ValueError, match="int8_linear: out is the memory of an input"):
                _lib().int8_linear(*at, n, V, K, P(out), None)


def test_sizes_beyond_a_launch_are_refused():
    """Before any grid is made of them: rows, channels and their products up to the largest 32-bit numbers."""
    L, I = _lib(), 2 ** 31 - 1
    for n in (1 << 24, I - 3, I):
        with pytest.raises(ValueError, match="rope_rows: n="):
            _rope(n=n)
        with pytest.raises(ValueError, match="kv_append_slots: n="):
            _append(n=n)
        with pytest.raises(ValueError, match="quantize_rows: n="):
            L.quantize_rows(A, 64, n, 64, B, C, None)
    with pytest.raises(ValueError, match="kv_append_slots: n="):
        _append(n=(1 << 24) - 1, hkv=16, ks=2048, vs=2048)
    for n, V in ((I, 16), (16, I), ((1 << 30) + 1, 16), (16, (1 << 30) + 1), (1 << 30, 1 << 30), (1 << 24, 1 << 24)):
        with pytest.raises(ValueError, match="int8_linear: n="):
            L.int8_linear(A, B, C, D, n, V, 64, E, None)
    for V in (I, (1 << 30) + 1):
        with pytest.raises(ValueError, match="int8_weight_tile"):
            L.int8_weight_tile(A, V, 64, B, None)
        assert L.raw.cpmcu_int8_weight_bytes(V, 64) == 0
    assert L.raw.cpmcu_int8_weight_bytes(16, 131072) == 0


def test_weights_are_on_the_current_device():
    import torch
    from cpm.cu_amd import ops
    with pytest.raises(AssertionError, match="current device required"):
        ops.Int8Weight(torch.zeros((16, 64), dtype=torch.int8), torch.zeros(16))


def test_weights_of_2_gib_and_more_fit_their_sizes():
    """Sizes in 64 bits: neither is a large weight refused, nor does a tensor fit that is shorter by a multiple of 2^32 (or 2^31)."""
    import torch
    from cpm.cu_amd import ops
    fits = ops._calls().int8_weight_fits
    weight = lambda n, t=torch.int8: torch.empty(n, dtype=t, device="meta")  # noqa: E731
    for V, K in ((256000, 12288), (131072, 16384), (131088, 16384), (262144, 16448), (1 << 20, 131071), (17, 65), (1, 1)):
        size = -(-V // 16) * 16 * (-(-K // 64) * 64)
        assert ops._lib().raw.cpmcu_int8_weight_bytes(V, K) == size
        assert fits(weight(size), V, K) and not fits(weight(size, torch.uint8), V, K)
        for other in (size - 1, size + 1, size % 2 ** 32, size % 2 ** 31):
            assert other == size or not fits(weight(other), V, K)
    I = 2 ** 31 - 1
    for V, K in ((0, 64), (-16, 64), (16, 0), (16, 131072), (16, I), (I, 64), (I, I)):
        assert not fits(weight(0), V, K) and not fits(weight(1 << 30), V, K)


def test_int8_linear_plans():
    """Every shape of the kernel is somebody's, from one row to many."""
    from cpm.cu_amd import lib, ops
    seen = {}
    for n in (1, 16, 32, 60, 128, 333, 512, 1024, 2048, 8192):
        for V, K in ((512, 1000), (4608, 4096), (16384, 4096), (73448, 4096), (4096, 16384), (12289, 4099)):
            name, workgroups = ops.int8_linear_plan(n, V, K)
            seen.setdefault(name, []).append((n, V, K))
            assert workgroups >= 1
    assert len(seen) == 8
    assert "split" in ops.int8_linear_plan(1, 4608, 4096)[0] and "wide" in ops.int8_linear_plan(8192, 16384, 4096)[0]
    for args in ((0, 16, 64), (1, 0, 64), (1, 16, 131072)):
        with pytest.raises(ValueError, match="int8_linear_plan"):
            ops.int8_linear_plan(*args)
    for value in (-2, 8):
        with pytest.raises(ValueError, match="int8_linear_shape"):
            lib.get().set_option(b"int8_linear_shape", value)


def test_int8_linear_choices_against_the_times_of_every_shape():
    """What the choice costs over the best shape in the committed table of `python -m cpm.cu_amd.sweep int8`: the figures that stand beside the costs, at the
    sizes they were fitted to and at those that were not."""
    import os
    from cpm.cu_amd import ops, sweep
    lines = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "profiles", "int8_linear_shapes.txt")).read().splitlines()
    names = lines[0].split(": ")[1].split()
    over, part = dict(fitted=[], others=[]), None
    for fields in map(str.split, lines[2:]):
        if len(fields) == 1:
            part = fields[0]
            continue
        n, V, K = map(int, fields[:3])
        times = [math.inf if t == "-" else float(t) for t in fields[3:]]
        chosen = ops.int8_linear_plan(n, V, K)[0].replace("int8_linear_", "").replace("_kernel", "")
        over[part].append(((n, V, K), times[names.index(chosen)] / min(times)))
    for part, (rows, weights), mean, worst in (("fitted", sweep.INT8_FITTED, 1.009, 1.13), ("others", sweep.INT8_OTHER, 1.019, 1.52)):
        assert [size for size, _ in over[part]] == [(n, V, K) for V, K in weights for n in rows]
        assert np.mean([x for _, x in over[part]]) < mean and max(x for _, x in over[part]) < worst


def test_binding_refuses_host_tensors_and_counts_arguments():
    import torch
    from cpm.cu_amd import ops
    native = ops._calls()
    h, i, f, b = torch.zeros((4, 2, 128), dtype=torch.float16), torch.zeros(4, dtype=torch.int32), torch.zeros(64), torch.zeros((4, 64), dtype=torch.int8)
    for call in (lambda: ops.rope_rows(h, None, i, f), lambda: ops.batch_tables(i, i, i.view(4, 1), i, i, i[:2], 4), lambda: ops.quantize_rows(h.view(4, 256)),
                 lambda: native.int8_linear(b, f[:4], b, f[:16], 16, 64, None), lambda: native.kv_append_slots(h, h, h, h, i, None, None, None, None, 0, 1.0)):
        with pytest.raises(AssertionError, match="current device required"):
            call()
    for name in ("rope_rows", "batch_tables", "quantize_rows", "int8_linear", "kv_append_slots"):
        with pytest.raises(TypeError, match="arguments given"):
            getattr(native, name)(*[None] * 17)
        with pytest.raises((AssertionError, TypeError)):
            getattr(native, name)(*[None] * dict(rope_rows=9, batch_tables=7, quantize_rows=1, int8_linear=7, kv_append_slots=11)[name])


# ---- rotary frequencies: against the formulas, pair by pair ----

def test_plain_linear_and_ntk_frequencies():
    from cpm.cu_amd import ops
    for dim, base in ((128, 10000.0), (64, 500000.0), (42, 1e6)):
        plain = np.array([base ** (-2.0 * i / dim) for i in range(dim // 2)])
        for scaling, want in ((None, plain), (dict(type="linear", factor=4.0), plain / 4), (dict(type="ntk", factor=8.0), [(base * 8.0 ** (dim / (dim - 2.0))) ** (-2.0 * i / dim) for i in range(dim // 2)])):
            freq, magnitude = ops.rope_frequencies(dim, base, scaling)
            # one rounding to 32 bits, and the powers' own in 64
            assert magnitude == 1.0 and np.allclose(freq.numpy().astype(np.float64), want, rtol=2.0 ** -24 + 1e-13, atol=0)
    # what the base is grown for: the slowest pair is stretched by the factor
    freq, _ = ops.rope_frequencies(128, 10000.0, dict(type="ntk", factor=8.0))
    assert np.isclose(float(freq[-1]) * 8.0, 10000.0 ** (-126 / 128), rtol=1e-6)


def test_yarn_frequencies():
    from cpm.cu_amd import ops
    dim, base, factor, original = 128, 10000.0, 16.0, 4096.0
    freq, magnitude = ops.rope_frequencies(dim, base, dict(type="yarn", factor=factor, original=original))
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1.0, rel=1e-12)
    low, high = (dim * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0))
    low, high = math.floor(low), math.ceil(high)
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        assert float(freq[i]) == pytest.approx(f * (1 - ramp) + f / factor * ramp, rel=1e-7)
    assert ops.rope_frequencies(dim, base, dict(type="yarn", factor=factor, original=original, magnitude=1.5))[1] == 1.5


def test_longrope_frequencies_follow_the_length():
    from cpm.cu_amd import ops
    short, long = np.linspace(1.0, 2.0, 32), np.linspace(1.0, 40.0, 32)
    scaling = dict(type="longrope", factor=32.0, original=4096, short_factor=list(short), long_factor=list(long))
    plain = 10000.0 ** (-np.arange(32) / 32)
    for length, by in ((4096, short), (4097, long)):
        freq, magnitude = ops.rope_frequencies(64, 10000.0, scaling, length=length)
        assert np.allclose(freq.numpy().astype(np.float64), plain / by, rtol=1e-7) and magnitude == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)))


@pytest.mark.parametrize("dim, scaling, length", [(7, None, None), (0, None, None), (64, dict(type="other"), None), (64, dict(type="linear", factor=0.5), None), (64, dict(type="linear", factor=math.nan), None),
                                                  (2, dict(type="ntk", factor=2.0), None), (64, dict(type="longrope", factor=2.0, original=4096, short_factor=[1.0] * 32, long_factor=[1.0] * 32), None),
                                                  (64, dict(type="longrope", factor=2.0, original=4096, short_factor=[1.0] * 31, long_factor=[1.0] * 32), 10)])
def test_rope_frequencies_refuse(dim, scaling, length):
    from cpm.cu_amd import ops
    with pytest.raises(ValueError):
        ops.rope_frequencies(dim, 10000.0, scaling, length=length)
