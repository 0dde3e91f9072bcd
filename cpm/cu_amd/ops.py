"""The operators of the verify/draft path on torch device tensors.

torch only supplies device memory and the current stream; every function here is a thin call into
``libcpmcu_amd.so`` through the C-ABI (``include/cpmcu_amd.h``), made by the native binding
``_torch_call``.  Nothing falls back to torch math.
"""
import copy
import ctypes
import math

import torch

from . import lib as _libmod
from .kvcache import HEAD_DIM

_native = None


def _lib():
    return _libmod.get()


def _calls():
    """The library's operators as native calls on tensors (csrc/torch_call.cpp), bound to the library lib.py has loaded.
    Pointer arguments are tensors (device-resident and contiguous, or AssertionError) or None; the stream is torch's current one."""
    global _native
    if _native is None:
        lib = _libmod.get()
        try:
            from . import _torch_call
        except ImportError as e:
            raise ImportError("the torch binding is not built or does not fit this torch (%s); run `python -m cpm.cu_amd.build`" % e) from e
        _torch_call.bind(lib.raw._handle)
        _native = _torch_call
    return _native


def _ptr_result(t):
    """A device tensor, or a pinned host tensor in its place: the GPU writes it through the mapped address."""
    return t if t is None or t.is_cuda else (_native or _calls()).pinned(t)


# One scratch buffer per operator family and device, handed to every call: calls that use it have to follow one another (one stream, or
# streams that wait for each other).  A call that needs more gets a buffer of at least twice the size, and the old one is
# kept, because captured launches go on writing to the addresses they were recorded with; all those kept are less than the one in use.
_workspaces = {}
_outgrown = []


def _workspace(kind, nbytes, device):
    key = (kind, device)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            if kind == "attn":
                release_attention_workspace(ws)
            if kind == "head":
                release_head_workspace(ws)
            _outgrown.append(ws)
            nbytes = max(nbytes, 2 * ws.numel())
        ws = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def release_attention_workspace(ws):
    """Before an attention workspace tensor is dropped: the library gives its merge counters to another workspace.
    The device is synchronised first (no launch on the workspace may be in flight)."""
    torch.cuda.synchronize()
    _lib().tree_attention_release_workspace(ctypes.c_void_p(ws.data_ptr()))


def release_head_workspace(ws):
    """Before a head workspace tensor is dropped: the library takes back the states its one-launch FR-Spec head
    publishes through.  The device is synchronised first (no launch on the workspace may be in flight)."""
    torch.cuda.synchronize()
    _lib().head_release_workspace(ctypes.c_void_p(ws.data_ptr()))


_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def synchronize():
    """Wait for torch's current stream."""
    (_native or _calls()).synchronize()


def mask_words(T):
    return (T + 63) // 64


def kv_append(cache, layer, k_new, v_new, kv_len):
    """copy_to_kvcache (src/model/attn.cuh:14-21): rows go to positions [*kv_len - T, *kv_len)."""
    (_native or _calls()).kv_append_rows(cache.k[layer], cache.v[layer], cache.block_table, k_new, v_new, kv_len, cache.Hkv)


def rope_table(position_ids, inv_freq):
    """(cos, sin) of float(position) * inv_freq for every tree row: [T, 64, 2] fp32 (src/model/rotary.cuh:11-17)."""
    T = position_ids.numel()
    assert position_ids.dtype == torch.int32 and inv_freq.dtype == torch.float32 and inv_freq.numel() == HEAD_DIM // 2
    out = torch.empty((T, HEAD_DIM // 2, 2), dtype=torch.float32, device=position_ids.device)
    _calls().rope_table(position_ids, inv_freq, T, out)
    return out


def rope_apply_(table, q, k):
    """In-place rotary embedding of q [T,Hq,128] and k [T,Hkv,128] (rotary_embedding_kernel, src/model/rotary.cuh:7-34)."""
    T, Hq, D = q.shape
    assert D == HEAD_DIM and k.shape[0] == T and k.shape[2] == D and table.shape[0] == T
    _calls().rope_apply(table, T, Hq, k.shape[1], q, k)


def tree_attention(q, cache, layer, kv_len, max_kv_len, mask=None, scale=None, num_splits=0, out=None,
                   k_new=None, v_new=None, mask_k_range=0, rope=None, block_window_size=0):
    """mha_fwd_kvcache with a tree mask (src/flash_attn/flash_api.hpp:292-392) on the paged cache.

    q [T, Hq, 128] fp16; kv_len int32[1] on the device = P + T; mask uint64 [T, W] or None (chain).
    k_new / v_new [T, Hkv, 128]: the tree rows' K/V; when given the kernel appends them to the cache
    itself (src/model/attn.cuh:200) instead of expecting them there.
    mask_k_range (0 = T): number of trailing keys the mask bits refer to; k*d for the drafter's layers.
    rope [T, 64, 2] fp32 from rope_table: q and k_new are taken unrotated and rotated inside the kernel.
    block_window_size (0 = none, else >= 128 tokens): the drafter layer's block sliding window
    (src/flash_attn/src/flash_blockmask.h:32): key blocks of 128 below ceil(P/128) - window/128 are skipped.
    """
    native = _native or _calls()
    if out is None:
        out = torch.empty_like(q)
    if mask is not None and not mask.is_contiguous():
        mask = mask.reshape(q.shape[0], -1)  # (a copy where the rows' order in memory is another one)
    ws = _workspaces.get(("attn", q.device))
    # (shapes and types are checked there)
    args = (q, cache.k[layer], cache.v[layer], cache.block_table, kv_len, int(max_kv_len), k_new, v_new, rope, int(block_window_size),
            mask, int(mask_k_range), cache.Hkv, _SCALE if scale is None else scale, out)
    need = native.tree_attention_rows(*args, ws, int(num_splits))
    if need is not None:
        native.tree_attention_rows(*args, _workspace("attn", need, q.device), int(num_splits))
    return out


def rope_frequencies(rotary_dim, base=10000.0, scaling=None, length=None):
    """(inv_freq fp32 [rotary_dim / 2] on the host, magnitude) for rope_rows: base ** (-2i / rotary_dim), stretched for contexts longer
    than the model was trained on.  scaling is None or a dict whose "type" is

    * "linear": positions as if factor times closer, inv_freq / factor;
    * "ntk": the base grows so that the slowest pair is stretched by factor and the fastest not at all,
      base * factor ** (rotary_dim / (rotary_dim - 2));
    * "yarn": pairs that turn more than beta_fast (32) times within original (the trained length) stay, those of fewer than beta_slow (1)
      turns are divided by factor, with a linear ramp over the pairs in between; magnitude 0.1 ln(factor) + 1 (or "magnitude");
    * "longrope": inv_freq / short_factor[i], from lengths above original on / long_factor[i] (length: the context this step works
      with); magnitude sqrt(1 + ln(factor) / ln(original)) where factor > 1 (or "magnitude").

    Computed in 64 bits."""
    half = int(rotary_dim) // 2
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim=%r is not an even number" % (rotary_dim,))
    i = torch.arange(half, dtype=torch.float64)
    freq = float(base) ** (-i / half)
    magnitude = 1.0
    if scaling is not None:
        kind = scaling.get("type")
        factor = float(scaling.get("factor", 1.0))
        if not factor >= 1.0:
            raise ValueError("scaling factor %r below 1" % (factor,))
        if kind == "linear":
            freq = freq / factor
        elif kind == "ntk":
            if half < 2:
                raise ValueError("ntk scaling of a single pair")
            freq = (float(base) * factor ** (half / (half - 1.0))) ** (-i / half)
        elif kind == "yarn":
            original = float(scaling["original"])
            # the pair (a fraction of one) that turns `turns` times within the trained length
            pair_of = lambda turns: half * math.log(original / (turns * 2.0 * math.pi)) / math.log(float(base))  # noqa: E731
            low = max(math.floor(pair_of(float(scaling.get("beta_fast", 32.0)))), 0)
            high = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1.0)))), 2 * half - 1)
            ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
            freq = freq * (1.0 - ramp) + freq / factor * ramp
            magnitude = float(scaling.get("magnitude", 0.1 * math.log(factor) + 1.0))
        elif kind == "longrope":
            original = float(scaling["original"])
            if length is None:
                raise ValueError("longrope frequencies depend on the length")
            by = torch.as_tensor(scaling["long_factor" if length > original else "short_factor"], dtype=torch.float64)
            if by.numel() != half:
                raise ValueError("%d factors for %d pairs" % (by.numel(), half))
            freq = freq / by
            magnitude = float(scaling.get("magnitude", math.sqrt(1.0 + math.log(factor) / math.log(original))))
        else:
            raise ValueError("rotary scaling of type %r" % (kind,))
    return freq.float(), magnitude


def rope_rows(q, k, positions, inv_freq, interleaved=False, magnitude=1.0, transposed=False, q_out=None, k_out=None):
    """Rotary positions of q [n, Hq, D] and k [n, Hkv, D] (or None): (q_out, k_out), new tensors unless given (q and k themselves: in place).

    positions int32 [n] (rows of a negative one are left out: a new tensor has no values there), inv_freq fp32 [rotary_dim / 2] (see rope_frequencies): the first rotary_dim
    values of each head turn, in pairs (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1).  Rows may be views of wider ones (a fused
    projection's output).  transposed: gradients of the results back to q and k.
    """
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    (_native or _calls()).rope_rows(q, k, positions, inv_freq, 1 if interleaved else 0, magnitude, 1 if transposed else 0, q_out, k_out)
    return q_out, k_out


def batch_tables(kv_lens, new_lens, block_tables, held, free_pages, counts, max_rows):
    """Pages and slots of a batch's new rows, from the requests' lengths, in one launch (int32 device tensors).

    kv_lens [B] cached and new_lens [B] new tokens of each request (negative: it has ended and gives its pages back); block_tables
    [B, max_blocks], of which the first held[r] entries of row r are request r's pages; free_pages, a stack of which counts[0] are free.
    Returns dict(kv_lens [B], held [B], counts [2] = (free pages, refused requests), row_offsets [B + 1], positions [max_rows], slots
    [max_rows]), which the next step takes in place of the inputs; block_tables and free_pages change in place.  Rows without a slot
    (refused requests', and behind the last one) have slot and position -1.  Once a request lacks pages every later one that needs any
    is refused as well, and a refused request's rows keep their range of the batch.  See PageBatch for an object that keeps all this.
    """
    lens, held, counts, offsets, positions, slots, _ = (_native or _calls()).batch_tables(kv_lens, new_lens, block_tables, held, free_pages, counts, int(max_rows))
    return dict(kv_lens=lens, held=held, counts=counts, row_offsets=offsets, positions=positions, slots=slots)


def kv_append_slots(cache, layer, k, v, slots, q=None, q_out=None, positions=None, inv_freq=None, interleaved=False, magnitude=1.0):
    """Rows k, v [n, Hkv, 128] of several requests to slots[t] = page * 256 + place of the cache (rows without a slot: left out).

    With positions and inv_freq, as rope_rows takes them, k is rotated on its way, and q [n, Hq, 128] (if given) into q_out, which is
    returned; rows left out keep what q_out held (a new tensor has no values there)."""
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    (_native or _calls()).kv_append_slots(cache.k[layer], cache.v[layer], k, v, slots, q, q_out, positions, inv_freq, 1 if interleaved else 0, magnitude)
    return q_out


class PageBatch:
    """The pages of up to max_requests requests on one paged cache, kept on the device: tables, lengths and the stack of free pages.

    ``plan(new_lens, max_rows)`` gives every request room for its new rows and returns where they go (batch_tables); ``kv_lens[r:r + 1]`` and
    ``block_tables[r]`` are then what tree_attention takes for request r (through ``cache_of``), with a max_kv_len of at most max_blocks * 256.

    Rows that turn out not to be wanted (nodes of a draft tree that are not accepted) are given up by writing the shorter length to
    ``kv_lens[r]``, in place: the next plan goes on from there, in pages that the request keeps.  A request that is refused has the length
    that it had; its rows have slot -1, and there is nothing to attend with."""

    def __init__(self, cache, max_requests, max_blocks, num_pages=None):
        self.cache = cache
        pages = cache.num_pages if num_pages is None else int(num_pages)
        assert 1 <= pages <= cache.num_pages
        self.max_requests, padded = int(max_requests), (int(max_requests) + 3) // 4 * 4
        self.block_tables = torch.zeros((self.max_requests, max_blocks), dtype=torch.int32, device=cache.device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=cache.device)
        # one tensor, laid out as batch_tables' results are, so that a step is taken by one copy: views of it, and launches captured with them, see the new values
        self._state = torch.zeros(4 + 2 * padded, dtype=torch.int32, device=cache.device)
        self.counts, self.held, self.kv_lens = self._state[:2], self._state[4:4 + self.max_requests], self._state[4 + padded:4 + padded + self.max_requests]
        self._state[0] = pages

    def plan(self, new_lens, max_rows):
        """new_lens int32 [max_requests]: rows of this step, -1 for a request that has ended.  The step is taken: lengths and pages
        are those with the new rows from here on (counts[1] says how many requests were refused)."""
        lens, held, counts, offsets, positions, slots, state = (_native or _calls()).batch_tables(self.kv_lens, new_lens, self.block_tables, self.held, self.free_pages,
                                                                                                  self.counts, int(max_rows))
        self._state.copy_(state)
        return dict(kv_lens=lens, held=held, counts=counts, row_offsets=offsets, positions=positions, slots=slots)

    def attention(self, q, layer, where, single=False, scale=None, out=None):
        """Every row of a plan (``where``) over its request's pages, behind the appends: prompt_attention, or, where no request has more than one row,
        decode_attention (single).  The tables go whole: where a bound on the requests' lengths is known, these with its columns are faster for short ones."""
        if single:
            return decode_attention(q, self.cache, layer, self.block_tables, where["positions"], where["row_offsets"], scale, out)
        return prompt_attention(q, self.cache, layer, self.block_tables, where["row_offsets"], where["positions"], scale, out)

    def cache_of(self, r):
        """Request r's view of the cache, for tree_attention."""
        view = copy.copy(self.cache)
        view.block_table = self.block_tables[r]
        return view


def quantize_rows(x):
    """16-bit rows [n, K] to 8 bits: (xq int8 [n, K rounded up to 64], zeros behind K; scales fp32 [n] = max |x| / 127)."""
    return (_native or _calls()).quantize_rows(x)


class Int8Weight:
    """8-bit weights [V, K] with a scale for each channel, in matrix-operand order: built once."""

    def __init__(self, w, scales):
        """w int8 [V, K], scales fp32 [V]: the weight of channel c is w[c] * scales[c].  Both are copied: what is written to them later
        does not change the weight."""
        assert w.dtype == torch.int8 and w.dim() == 2 and scales.dtype == torch.float32 and scales.numel() == w.shape[0]
        assert w.is_cuda and w.device == scales.device and w.device.index == torch.cuda.current_device(), "weights and scales on the current device required"
        self.V, self.K = w.shape
        self.shape = (self.V, self.K)
        self.scales = scales.detach().reshape(self.V).clone(memory_format=torch.contiguous_format)
        w = w.contiguous()
        self.data = torch.empty(_lib().raw.cpmcu_int8_weight_bytes(self.V, self.K), dtype=torch.int8, device=w.device)
        _calls().int8_weight_tile(w, self.V, self.K, self.data)

    @classmethod
    def quantized(cls, w):
        """From 16-bit weights [V, K]: each channel to 8 bits as quantize_rows does a row."""
        wq, scales = quantize_rows(w)
        return cls(wq[:, :w.shape[1]], scales)


def int8_linear(xq, x_scales, weight, out=None):
    """[n, V] = (xq . weight^T in 32-bit integers) * x_scales * weight.scales, in 16 bits; xq and x_scales from quantize_rows."""
    return (_native or _calls()).int8_linear(xq, x_scales, weight.data, weight.scales, weight.V, weight.K, out)


def prompt_attention(q, cache, layer, block_tables, row_offsets, positions, scale=None, out=None):
    """Causal attention of the new rows q [n, Hq, 128] of several requests over their pages, in any mixture: prompts, chunks, single rows.

    block_tables int32 [B, max_blocks], row_offsets int32 [B + 1] and positions int32 [n] as batch_tables gives them: request r's rows are
    [row_offsets[r], row_offsets[r + 1]), the first at positions[row_offsets[r]], each sees the tokens of its request up to its own, which have been appended
    (kv_append_slots).  Rows of refused requests, and behind the last one, keep what out held (a new tensor has no values there).  q and out may be
    parts of wider rows; out may be q.  How many columns the tables have decides the launches and the workspace (about 120 MB where they have room for long
    requests): columns that no request reaches are best left out (block_tables[:, :columns]).  See PageBatch.attention.
    """
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    (_native or _calls()).prompt_attention(q, cache.k[layer], cache.v[layer], block_tables, row_offsets, positions, _SCALE if scale is None else scale, out)
    return out


def decode_attention(q, cache, layer, block_tables, positions, row_offsets=None, scale=None, out=None):
    """prompt_attention for requests of one new row each (a step of decoding): row r of q is request r's, or row row_offsets[r] where it has one; requests of
    no row or of several are left out."""
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    (_native or _calls()).decode_attention(q, cache.k[layer], cache.v[layer], block_tables, row_offsets, positions, _SCALE if scale is None else scale, out)
    return out


def adjust_logits(logits, penalties=None, tokens=None, lens=None, requests=None, bias_ids=None, bias_values=None, allowed=None, draft_ids=None, tree_mask=None,
                  out=None, want_ids=True):
    """Penalties for repeated tokens, biases and masks on rows of logits [n, V], and their arg-max: (out, ids int32 [n] or None).

    Of a token that stands c > 0 times in the text of its row's request the logit z becomes (z / repetition if z > 0 else z * repetition) - frequency * c -
    presence; then its bias is added, and what is not allowed becomes minus infinity.  ids is the lowest index of a row's largest result, -1 where nothing is left.

    penalties fp32 [R, 3]: (repetition, presence, frequency) of each request.  tokens int32 [R, L up to 2^20], of which lens int32 [R] count.  requests int32 [n]: each
    row's request (-1: none); left out, row t is request t's, or all are of the only one.  bias_ids int32 / bias_values fp32 [R, up to 1024] (-1: not used).
    allowed int32 [n, ceil(V / 32)]: bit v % 32 of word v / 32 (``mask.expand(n, -1)``: one for all rows).  draft_ids int32 [n] / tree_mask int64
    [n, words]: the rows are the nodes of one request's draft tree, and the drafts on a node's way, its own among them, stand behind the request's tokens.
    All three penalties count the same text.  out may be logits (in place).
    """
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    ids = (_native or _calls()).adjust_logits(logits, penalties, tokens, lens, requests, bias_ids, bias_values, allowed, draft_ids, tree_mask, out, want_ids)
    return out, ids


def gather_rows(src, remap):
    """remap_copy (src/model/tree_drafter.cuh:79-86): dst[r] = src[remap[r]]."""
    assert src.dtype == torch.float16 and remap.dtype == torch.int32
    dst = torch.empty((remap.numel(), src.shape[1]), dtype=torch.float16, device=src.device)
    _calls().gather_rows(src, remap, remap.numel(), src.shape[1], dst)
    return dst


W_ROW_MAJOR, W_TILED = 0, 1
COMMIT_ADVANCE_LENGTH = 1
COMMIT_NEXT_ROOT = 2


class TiledWeight:
    """A head weight matrix in MFMA operand order (CPMCU_W_TILED): built once, streamed ~20 % faster."""

    def __init__(self, data, V, H):
        self.data, self.V, self.H = data, int(V), int(H)
        self.shape = (self.V, self.H)


def tile_head_weight(w, row_remap=None):
    """[*, H] row-major fp16 -> TiledWeight of V rows; with row_remap (int32 [V]) row r is w[row_remap[r]]
    (remap_copy, src/model/tree_drafter.cuh:79-86, fused with the re-tiling)."""
    assert w.dtype == torch.float16 and w.is_contiguous()
    H = w.shape[1]
    V = w.shape[0] if row_remap is None else row_remap.numel()
    out = torch.empty(_lib().raw.cpmcu_head_weight_tiled_bytes(V, H) // 2, dtype=torch.float16, device=w.device)
    _calls().head_weight_tile(w, row_remap, V, H, out)
    return TiledWeight(out, V, H)


def _weight(w):
    if isinstance(w, TiledWeight):
        return w.data, W_TILED, w.V
    return w, W_ROW_MAJOR, w.shape[0]


def frspec_head_topk(hidden, w, token_id_remap, k):
    """FR-Spec draft head: logits -> log-softmax -> top-k -> full-vocabulary ids.

    Returns dict(logits [n,V] f16 raw, row_stats [n,2] f32 (max, ln sum), val [n,k] f16, pos [n,k] i32, ids [n,k] i32).
    """
    n, H = hidden.shape
    w, layout, V = _weight(w)
    native = _native or _calls()
    logits, stats, val, pos, ids = native.empty(hidden, "h", n, V, "f", n, 2, "h", n, k, "i", n, k, "i", n, k)
    ws = _workspace("head", native.head_workspace_bytes(n, V), hidden.device)
    native.frspec_head_topk(hidden, w, layout, token_id_remap, n, V, H, k, logits, stats, val, pos, ids, ws, ws.numel())
    return dict(logits=logits, row_stats=stats, val=val, pos=pos, ids=ids)


def frspec_head_plan(n, w, k):
    """Kernel name(s) of a frspec_head_topk call with n hidden rows on matrix w: the one-launch kernel when the shape
    allows it and the library has a publication state for the head workspace, else GEMM + top-k."""
    w_, layout, V = _weight(w)
    H = w.H if isinstance(w, TiledWeight) else w.shape[1]
    gemm = head_plan(n, w)[0]
    ws = _workspace("head", _lib().raw.cpmcu_head_workspace_bytes(n, V), w_.device)
    if _lib().raw.cpmcu_frspec_head_mode(ctypes.c_void_p(ws.data_ptr()), layout, n, V, H, k) == 1:
        nb, fp, kc = gemm[gemm.index("<") + 1:-1].split(",")
        return "frspec_head_topk_kernel<%s,%s>" % (fp, kc)
    # the row kernel: on the whole row up to 32768 elements (in its short form up to 8192), on slices of it beyond
    slices = (V + 8191) // 8192
    short = V <= 8192 or (V > 32768 and n * slices <= 512 and slices * k <= 256)
    return gemm + ("+topk_short_row_kernel<true>" if short else "+topk_row_kernel<true>") + ("" if V <= 32768 else "+topk_slice_merge_kernel<true>")


def lm_head_argmax(hidden, w, head_scale=None, want_logits=False, gt=None):
    """Target head + arg-max (src/model/linear.cuh:82-101 + torch argmax of tree_drafter.py:233)."""
    n, H = hidden.shape
    w, layout, V = _weight(w)
    native = _native or _calls()
    logits = native.empty(hidden, "h", n, V)[0] if want_logits else None
    if gt is None:
        gt = torch.empty(n, dtype=torch.int32, device=hidden.device)
    ws = _workspace("head", native.head_workspace_bytes(n, V), hidden.device)
    native.lm_head_argmax(hidden, w, layout, n, V, H, 0 if head_scale is None else 1, 1.0 if head_scale is None else head_scale, logits, gt,
                          ws, ws.numel())
    return (gt, logits) if want_logits else gt


class HeadPartials:
    """The target head's arg-max left as per-workgroup partials (cpmcu_lm_head_partials): finished by verify_tail."""

    def __init__(self, workspace, num_partials, stride, n):
        self.workspace, self.num_partials, self.stride, self.n = workspace, int(num_partials), int(stride), int(n)


def lm_head_partials(hidden, w, head_scale=None, logits=None):
    """The target head's GEMM without the launch that finishes its arg-max; see verify_tail."""
    n, H = hidden.shape
    w, layout, V = _weight(w)
    native = _native or _calls()
    ws = _workspace("head", native.head_workspace_bytes(n, V), hidden.device)
    num, stride = native.lm_head_partials(hidden, w, layout, n, V, H, 0 if head_scale is None else 1,
                                          1.0 if head_scale is None else head_scale, logits, ws, ws.numel())
    return HeadPartials(ws, num, stride, n)


def verify_tail(cache, draft_ids, gt, position_ids, cache_length, attn_mask, tree_parent, hidden=None, prev_hidden=None,
                gt_out=None, best=None, path=None, accepted_ids=None, next_position_ids=None, result=None):
    """The whole tail of verify() in one launch (src/model/minicpm4/minicpm4_eagle.cuh:398-418): arg-max finish
    when `gt` is a HeadPartials, acceptance, compaction of every layer, accepted ids, hidden-row gather.
    draft_ids is read only; results go to best (a, node), path [T], accepted_ids [T], gt_out [T], ..."""
    T = draft_ids.numel()
    W = attn_mask.numel() // T
    parts = gt if isinstance(gt, HeadPartials) else None
    hidden_dim = 0 if hidden is None else hidden.shape[-1]
    (_native or _calls()).verify_tail(
        cache.k_ptrs, cache.v_ptrs, cache.num_layers, cache.block_table, cache.Hkv, T, draft_ids, None if parts else gt,
        parts.workspace if parts else None, parts.num_partials if parts else 0, parts.stride if parts else 0, position_ids, cache_length,
        attn_mask, W, tree_parent, hidden, hidden_dim, prev_hidden, gt_out, best, path, accepted_ids, next_position_ids, _ptr_result(result))


def verify_tail_inplace(best, accepted_ids, pred=None, cache_length=None, kv_len=None, position_ids=None, advance_length=False,
                        next_root=False):
    """The in-place updates behind verify_tail: pred[:a] <- ids (or pred[0] <- last id), lengths and positions += a."""
    flags = (COMMIT_ADVANCE_LENGTH if advance_length else 0) | (COMMIT_NEXT_ROOT if next_root else 0)
    _calls().verify_tail_inplace(best, accepted_ids, accepted_ids.numel(), pred, cache_length, kv_len, position_ids, flags)


def log_softmax_(x):
    """In place (src/model/eagle.cuh:29-89); returns row_stats [n,2] (max, ln sum)."""
    n, dim = x.shape
    native = _native or _calls()
    # (the slices' few bytes are the call's own, as the outputs are: calls on several streams or threads, and captured ones, share nothing)
    stats, ws = native.empty(x, "f", n, 2, "f", native.log_softmax_workspace_bytes(n, dim) // 4, 0)
    native.log_softmax_sliced(x, n, dim, stats, ws, ws.nbytes)
    return stats


def topk(x, top):
    """TopK::prefill (src/model/topk.cuh:255-288): value descending, ties -> lower index."""
    n, dim = x.shape
    native = _native or _calls()
    val, pos = native.empty(x, "h", n, top, "i", n, top)
    ws = _workspace("topk", native.topk_workspace_bytes(n, dim, top), x.device)
    native.topk(x, n, dim, top, val, pos, ws, ws.numel())
    return val, pos


def remap(pos, token_id_remap):
    out = torch.empty_like(pos)
    _calls().remap(pos, pos.numel(), token_id_remap, out)
    return out


def tree_accept(pred, gt, position_ids, cache_length, attn_mask, tree_parent, best=None):
    """verify_kernel (src/model/tree_drafter.cuh:5-46). pred is overwritten with the path; returns best[2]."""
    T = pred.numel()
    if best is None:
        best = torch.empty(2, dtype=torch.int32, device=pred.device)
    W = attn_mask.numel() // T
    _calls().tree_accept(T, pred, gt, position_ids, cache_length, attn_mask, W, tree_parent, best)
    return best


def kv_compact(cache, pred, gt, cache_length, best, max_accept):
    """fix_kv_cache (src/model/tree_drafter.cuh:48-77) on every layer of the paged cache."""
    _calls().kv_compact(cache.k_ptrs, cache.v_ptrs, cache.num_layers, cache.block_table, cache.Hkv, pred, gt, cache_length, best, int(max_accept))


def accept_commit(cache, pred, gt, cache_length, best, max_accept, hidden=None, prev_hidden=None,
                  next_position_ids=None, result=None, advance_length=False, next_root=False, kv_len=None):
    """The rest of verify() after the acceptance (src/model/minicpm4/minicpm4_eagle.cuh:398-418): compaction,
    accepted ids, gather of the accepted hidden rows, next position ids, packed (a, ids) result and the
    device-side advance of cache_length, in two launches with the accept length staying on the device."""
    flags = (COMMIT_ADVANCE_LENGTH if advance_length else 0) | (COMMIT_NEXT_ROOT if next_root else 0)
    hidden_dim = 0 if hidden is None else hidden.shape[-1]
    _calls().accept_commit(cache.k_ptrs, cache.v_ptrs, cache.num_layers, cache.block_table, cache.Hkv, pred, gt, cache_length, kv_len, best,
                           int(max_accept), hidden, hidden_dim, prev_hidden, next_position_ids, _ptr_result(result), flags)


class DraftTree:
    """Tree bookkeeping of the drafter (src/model/minicpm4/minicpm4_eagle.cuh:319-393) on the device.

    One object per draft model; ``begin`` / ``extend`` / ``finish`` are one kernel each and never
    synchronise, so a whole draft can be enqueued (or graph-captured) without a host round trip.
    """

    def __init__(self, k, num_iter, token_id_remap=None, device="cuda"):
        self.k, self.num_iter = int(k), int(num_iter)
        self.remap = token_id_remap
        nbytes = _lib().raw.cpmcu_draft_tree_state_bytes(self.k, self.num_iter)
        self.state = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
        self.next_ids = torch.empty(self.k, dtype=torch.int32, device=device)
        self.parent_rows = torch.empty(self.k, dtype=torch.int32, device=device)
        self.draft_mask = torch.empty(self.k, dtype=torch.int64, device=device)

    def begin(self, topk_val, topk_pos):
        """topk_val fp16[k], topk_pos int32[k] (first row). Returns next_ids [k]."""
        assert topk_val.dtype == torch.float16 and topk_pos.dtype == torch.int32 and topk_val.numel() == self.k
        (_native or _calls()).draft_tree_begin(self.state, self.k, self.num_iter, topk_val, topk_pos, self.remap, self.next_ids, self.draft_mask)
        return self.next_ids

    def extend(self, d, topk_val, topk_pos):
        """topk_val fp16[k,k] (cumulated in place), topk_pos int32[k,k] of iteration d >= 1.
        Returns (next_ids [k], parent_rows [k], draft_mask [k])."""
        assert topk_val.dtype == torch.float16 and topk_pos.dtype == torch.int32 and topk_val.numel() == self.k * self.k
        (_native or _calls()).draft_tree_extend(self.state, self.k, self.num_iter, int(d), topk_val, topk_pos, self.remap, self.next_ids,
                                                self.parent_rows, self.draft_mask)
        return self.next_ids, self.parent_rows, self.draft_mask

    def finish(self, tree_size, cache_length, tree_draft_ids=None):
        """cache_length int32[1] on the device = P.  Returns (ids [T] -- entry 0 untouched --, positions [T],
        mask [T, W] as int64 bit patterns, parent [T])."""
        native, T = _native or _calls(), int(tree_size)
        W = mask_words(T)
        if tree_draft_ids is not None:
            pos, mask, parent = native.empty(self.state, "i", T, 0, "l", T, W, "i", T, 0)
            native.draft_tree_finish(self.state, self.k, self.num_iter, T, cache_length, self.remap, tree_draft_ids, pos, mask, parent)
        else:
            tree_draft_ids, pos, mask, parent = native.empty(self.state, "i", T, 0, "i", T, 0, "l", T, W, "i", T, 0)
            native.draft_tree_finish_root(self.state, self.k, self.num_iter, T, cache_length, self.remap, -1, tree_draft_ids, pos, mask, parent)
        return tree_draft_ids, pos, mask, parent


def attention_plan(T, Hq, Hkv, max_kv_len, rope=False, block_window_size=0, num_splits=0):
    """(kernel names, KV splits, KV groups per workgroup, workgroups) of a tree-attention call of this shape."""
    buf = ctypes.create_string_buffer(160)
    ns, g, wg = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    _lib().tree_attention_plan(T, Hq, Hkv, int(max_kv_len), 1 if rope else 0, int(block_window_size), int(num_splits), buf, 160,
                               ctypes.byref(ns), ctypes.byref(g), ctypes.byref(wg))
    return buf.value.decode(), ns.value, g.value, wg.value


def head_plan(n, w):
    """(GEMM kernel name, workgroups) of a head call with n hidden rows on weight matrix w."""
    _, layout, V = _weight(w)
    H = w.H if isinstance(w, TiledWeight) else w.shape[1]
    buf = ctypes.create_string_buffer(96)
    wg = ctypes.c_int(0)
    _lib().head_plan(n, V, H, layout, buf, 96, ctypes.byref(wg))
    return buf.value.decode(), wg.value


def int8_linear_plan(n, V, K):
    """(kernel name, workgroups) of an int8_linear call of n rows on a weight [V, K]."""
    buf, wg = ctypes.create_string_buffer(96), ctypes.c_int(0)
    _lib().int8_linear_plan(int(n), int(V), int(K), buf, 96, ctypes.byref(wg))
    return buf.value.decode(), wg.value
