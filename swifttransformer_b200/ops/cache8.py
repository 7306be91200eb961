"""Caches in 8 bits, attention over them, and attention for batches that share a prefix.

An 8-bit cache is a pair of tensors: ``pool`` [pages, layers, 2, kv heads, page size, head size] of ``torch.int8`` or
``torch.float8_e4m3fn`` and ``scales`` [pages, layers, 2, kv heads, page size] of float32.  An element stands for its code times
its row's scale.  A row x is stored with the scale max(max|x| / M, 2^-126), M = 127 for int8 and 448 for e4m3, and the codes
x / scale rounded to the nearest number of the form, ties to even; a row with a NaN or an infinity has the scale NaN.  The reference
keeps its cache in the type of its activations (src/csrc/kernel/kvcache_mgmt.cu:29-80).

Against bfloat16 a cache takes 0.53 (head size 64) or 0.52 (128) of the memory, and a decode step reads that much less.  int8
stores a row's elements to 1 / 254 of its largest, e4m3 every element to 1 / 16 of itself.

The attention multiplies codes in half precision with weights p_j vs_j in half precision (float queries: both in two halves): exact
codes, weights to 2^-11 (2^-22), as long as the value scales of a row's keys lie within 2^20 of one another; smaller ones lose bits, and from
2^110 on the softmax's sum does.  Keys of magnitude 2^100 and more may overflow.

All functions take the index tensors of the other paged operations: ``positions`` and ``seq_of_token`` per token, ``slots`` per
request, ``block_table`` [slots, pages], int32 on the device.  A token whose position is negative is padding and left out.
``status`` (int32, by default a word that ``ops.kernel_status`` reads) is set to 1 when a key that a query needs has no page; such
keys count as absent, and a query without any key gets zeros.  Calls launch on the current stream and keep no state of their own.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional, Sequence

import numpy as np
import torch

from . import KernelError, _check, _current_device, _stream, _tc_status_word, lib

CACHE8_TYPES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_FORMS = {torch.int8: 0, torch.float8_e4m3fn: 1, torch.bfloat16: 2, torch.float32: 3}
_ACTS = {torch.float32: 0, torch.bfloat16: 1}
_I32 = torch.int32
# the library's: query rows of a tile, keys of a chunk, places of a (tile, key head) beside its chunks (csrc/attention_rows.cuh)
ROWS_PER_TILE = 128
ROWS_CHUNK = 64
ROWS_UNIT = 3
MAX_KEYS = 0x7fff0000            # of a request: positions and a few runs of keys behind them stay in an int (c8_reach in csrc/cache8.cuh)


def cache8_pool(num_pages: int, n_layers: int, nkv: int, page_size: int, d: int, dtype: torch.dtype, device):
    """An empty 8-bit cache (pool, scales): every row reads back as zeros."""
    if dtype not in CACHE8_TYPES:
        raise KernelError(f"an 8-bit cache is int8 or float8_e4m3fn, not {dtype}")
    shape = (num_pages, n_layers, 2, nkv, page_size)
    return (torch.zeros(shape + (d,), dtype=torch.int8, device=device).view(dtype),
            torch.zeros(shape, dtype=torch.float32, device=device))


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise KernelError(what)


# The checks below run in every call of a decode step's layers: they name what is wrong only once something is.
def _same_device(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """All tensors on one CUDA device, the current one: the launch goes there."""
    index = tensors[0].get_device()
    if index < 0:
        raise KernelError("this engine runs on a CUDA device only; got a CPU tensor")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise KernelError(f"{what}: tensors on different devices")
    if index != _current_device():
        raise KernelError(f"{what}: tensors on cuda:{index}, but the current device is cuda:{_current_device()}")


def _index(what: str, positions, seq_of_token, slots, block_table, n: int) -> None:
    """int32, contiguous, a position and a request for each of n tokens."""
    for t in (positions, seq_of_token, slots, block_table):
        if t is not None and not (t.dtype is _I32 and t.is_contiguous() and t.dim() == (2 if t is block_table else 1)):
            raise KernelError(f"{what}: positions, seq_of_token, slots (one dimension) and block_table (two) are contiguous int32 tensors")
    if positions.numel() < n or (seq_of_token is not None and seq_of_token.numel() < n):
        raise KernelError(f"{what}: a position and a request for every token")


def _pool8(what: str, pool: torch.Tensor, scales: Optional[torch.Tensor], layer: int, only8: bool):
    """The pool's sizes (pages, layers, kv heads, page size, head size) and its form."""
    shape, form = pool.shape, _FORMS.get(pool.dtype)
    if len(shape) != 6 or shape[2] != 2 or not pool.is_contiguous():
        raise KernelError(f"{what}: the pool is a contiguous [pages, layers, 2, kv heads, page size, head size]")
    if form is None or (only8 and form > 1):
        raise KernelError(f"{what}: unsupported cache type {pool.dtype}")
    if form <= 1:
        if scales is None or scales.dtype is not torch.float32 or not scales.is_contiguous() or scales.shape != shape[:5]:
            raise KernelError(f"{what}: an 8-bit pool comes with contiguous float32 scales [pages, layers, 2, kv heads, page size]")
    elif scales is not None:
        raise KernelError(f"{what}: scales belong to 8-bit pools")
    pages, layers, _, nkv, page_size, d = shape
    if not 0 <= layer < layers:
        raise KernelError(f"{what}: the pool has no layer {layer}")
    return pages, layers, nkv, page_size, d, form


_WRITE = struct.Struct("=11Q12i")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def qkv_to_cache8(qkv: torch.Tensor, bias: Optional[torch.Tensor], q_out: Optional[torch.Tensor], pool: torch.Tensor,
                  scales: torch.Tensor, layer: int, positions: torch.Tensor, seq_of_token: torch.Tensor, slots: torch.Tensor,
                  block_table: torch.Tensor, nh: int, nkv: int, d: int, status: Optional[torch.Tensor] = None,
                  write_kv: bool = True) -> None:
    """q_out = q + bias; the rows k + bias and v + bias (float32 sums) quantised into an 8-bit cache at each token's position.

    ``qkv`` [tokens, (nh + 2 nkv) d] float32 or bfloat16; ``bias`` float32 or None; ``q_out`` [tokens, nh d] of qkv's type, or None: the
    queries stay where they are.  ``write_kv`` False: only the queries move.  Head sizes up to 256.  No two tokens of a call have
    the same request and position."""
    what = "qkv_to_cache8"
    _same_device(what, qkv, bias, q_out, pool, scales, positions, seq_of_token, slots, block_table, status)
    act, cols = _ACTS.get(qkv.dtype), (nh + 2 * nkv) * d
    if act is None or qkv.dim() != 2 or qkv.shape[1] != cols or not qkv.is_contiguous():
        raise KernelError(f"{what}: qkv is a contiguous [tokens, (nh + 2 nkv) d] of float32 or bfloat16")
    n = qkv.shape[0]
    if bias is not None and (bias.dtype is not torch.float32 or bias.numel() != cols or not bias.is_contiguous()):
        raise KernelError(f"{what}: the bias is contiguous float32, one number per column")
    if q_out is not None and (q_out.dtype is not qkv.dtype or q_out.shape != (n, nh * d) or not q_out.is_contiguous()):
        raise KernelError(f"{what}: q_out is a contiguous [tokens, nh d] of qkv's type")
    pages, layers, pool_kv, page_size, pool_d, form = _pool8(what, pool, scales, layer, True)
    if pool_kv != nkv or pool_d != d:
        raise KernelError(f"{what}: the pool has other heads or sizes")
    _index(what, positions, seq_of_token, slots, block_table, n)
    st = status if status is not None else _tc_status_word(qkv.device)
    call = _WRITE.pack(qkv.data_ptr(), _ptr(bias), _ptr(q_out), pool.data_ptr(), scales.data_ptr(), positions.data_ptr(),
                       seq_of_token.data_ptr(), slots.data_ptr(), block_table.data_ptr(), st.data_ptr(), 0,
                       block_table.shape[1], pages, layers, layer, n, nh, nkv, d, page_size, 1 if write_kv else 0, act, form)
    _check(lib().st_qkv_to_cache8(call, _stream()), what)


def cache8_rows(pool: torch.Tensor, scales: torch.Tensor, layer: int, out: torch.Tensor, positions: torch.Tensor,
                seq_of_token: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor,
                status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = the keys of all heads, then the values of all heads, of position ``positions[t]`` of request ``seq_of_token[t]``:
    [tokens, 2 nkv d] float32 or bfloat16, code times scale.  A position without a page gives zeros."""
    what = "cache8_rows"
    _same_device(what, out, pool, scales, positions, seq_of_token, slots, block_table, status)
    pages, layers, nkv, page_size, d, form = _pool8(what, pool, scales, layer, True)
    act = _ACTS.get(out.dtype)
    if act is None or out.dim() != 2 or out.shape[1] != 2 * nkv * d or not out.is_contiguous():
        raise KernelError(f"{what}: out is a contiguous [tokens, 2 nkv d] of float32 or bfloat16")
    n = out.shape[0]
    _index(what, positions, seq_of_token, slots, block_table, n)
    st = status if status is not None else _tc_status_word(out.device)
    call = _WRITE.pack(0, 0, 0, pool.data_ptr(), scales.data_ptr(), positions.data_ptr(), seq_of_token.data_ptr(), slots.data_ptr(),
                       block_table.data_ptr(), st.data_ptr(), out.data_ptr(),
                       block_table.shape[1], pages, layers, layer, n, 0, nkv, d, page_size, 0, act, form)
    _check(lib().st_cache8_rows(call, _stream()), what)
    return out


# ------------------------------------------------------------------ plans
class RowPlan:
    """Which query rows share a pass over which keys: made on the host once per step, used by all its layers.

    ``tiles``: int32 [n_tiles, 6] on the device: first token (or place in ``items``), tokens, request (-1: that of the first
    item), first and last + 1 key, and where the tile begins in the line of all units (places per unit and per chunk of keys).  ``items``: the tokens of
    a plan for shared prefixes in the tiles' order; ``info`` [items, 3]: keys shared with the group, tile, place in the tile."""

    def __init__(self, kind: str, nh: int, nkv: int, device):
        _need(nkv > 0 and nh > 0 and nh % nkv == 0, f"{nh} heads cannot share {nkv} key/value heads")
        _need(nh // nkv <= ROWS_PER_TILE, f"at most {ROWS_PER_TILE} query heads to a key head")
        self.kind, self.nh, self.nkv, self.window = kind, nh, nkv, 0
        self.device = torch.device(device)
        self.n_tiles = self.n_items = self.total = self.max_rows = self.max_own = self.n_tokens = self.n_seqs = 0
        self.tiles = self.items = self.info = None

    @property
    def tokens_per_tile(self) -> int:
        return ROWS_PER_TILE // (self.nh // self.nkv)

    def _chunks(self, lo: int, hi: int) -> int:
        return -(-(hi - lo // ROWS_CHUNK * ROWS_CHUNK) // ROWS_CHUNK) if hi > lo else 0

    def _upload(self, tiles, items=None, info=None) -> None:
        start = 0
        rows = []
        for first, n, seq, lo, hi in tiles:
            _need(hi <= MAX_KEYS, f"a plan reaches to at most {MAX_KEYS} keys")
            rows.append((first, n, seq, lo, hi, start))
            chunks = self._chunks(lo, hi)
            start += (chunks + ROWS_UNIT) * self.nkv if chunks else 0
        _need(start < 1 << 30 and len(rows) * self.nkv < 1 << 22, "a plan of more keys than one call serves")
        self.total, self.n_tiles = start, len(rows)
        self.max_rows = max((r[1] for r in rows), default=0) * (self.nh // self.nkv)
        flat = np.asarray(rows, dtype=np.int32).reshape(-1)
        parts = [flat] + [np.asarray(x, dtype=np.int32).reshape(-1) for x in (items, info) if x is not None]
        dev = torch.from_numpy(np.concatenate(parts)).to(self.device)
        self.tiles = dev[:flat.size]
        if items is not None:
            self.items = dev[flat.size:flat.size + parts[1].size]
            self.info = dev[flat.size + parts[1].size:]
            self.n_items = parts[1].size


def portion_plan(lens: Sequence[int], starts: Sequence[int], nh: int, nkv: int, window: int = 0, device="cuda") -> RowPlan:
    """The plan of a step in which request i brings ``lens[i]`` tokens, one behind the other, and has ``starts[i]`` in the cache.  In a call
    token j of request i stands at ``starts[i] + j`` or is padding.  Making a plan waits for the current stream."""
    plan = RowPlan("portion", nh, nkv, device)
    _need(len(lens) == len(starts) and all(n >= 0 for n in lens) and all(s >= 0 for s in starts) and window >= 0,
          "portion_plan: a length and a start per request, none negative")
    plan.window, per, tiles, first = int(window), plan.tokens_per_tile, [], 0
    for seq, (n, start) in enumerate(zip(lens, starts)):
        for off in range(0, n, per):
            m, pos = min(per, n - off), start + off
            tiles.append((first + off, m, seq, max(0, pos - window + 1) if window else 0, pos + m))
        first += n
    plan.n_tokens, plan.n_seqs = first, len(lens)
    plan._upload(tiles)
    return plan


def shared_prefix_plan(groups: Sequence[Sequence[int]], shared: Sequence[int], nh: int, nkv: int, device="cuda",
                       max_own: int = 0, window: int = 0, starts: Optional[Sequence[int]] = None) -> RowPlan:
    """The plan of a step of single tokens: ``groups[i]`` lists the tokens whose requests have their first ``shared[i]`` keys in common
    (0: none).  ``max_own``: about the most keys a token has behind its shared ones (it decides how the work is spread).

    For calls with a window, ``window`` and ``starts`` leave out the shared keys that it hides: no token of ``groups[i]`` stands before
    position ``starts[i]``, neither now nor when the plan is used again.  A plan without them serves every window, and walks all keys.

    Sharing pays from about 16 thousand members x shared keys on (at 32 key heads of 64; 8 thousand at 32 of 128), as 16 requests behind
    1000 tokens; below, the single-token attention over the same pages is faster.  Making a plan waits for the current stream."""
    plan = RowPlan("shared", nh, nkv, device)
    _need(len(groups) == len(shared) and all(s >= 0 for s in shared), "shared_prefix_plan: a shared length per group, none negative")
    _need(window >= 0 and (starts is not None) == (window > 0), "shared_prefix_plan: a window, not negative, comes with starts")
    _need(starts is None or (len(starts) == len(groups) and all(s >= 0 for s in starts)),
          "shared_prefix_plan: a start per group, none negative")
    per, tiles, items, info = plan.tokens_per_tile, [], [], []
    for i, (tokens, n) in enumerate(zip(groups, shared)):
        lo = min(n, max(0, starts[i] - window + 1)) if window else 0
        for off in range(0, len(tokens), per):
            part = [int(t) for t in tokens[off:off + per]]
            tiles.append((len(items), len(part), -1, int(lo), int(n)))
            info += [(int(n), len(tiles) - 1, k) for k in range(len(part))]
            items += part
    _need(all(0 <= t < 1 << 31 for t in items) and len(set(items)) == len(items),
          "shared_prefix_plan: every token at most once, none negative")
    plan.n_tokens, plan.max_own, plan.window = max(items, default=-1) + 1, int(max_own), int(window)
    plan._upload(tiles, items, info)
    return plan


# ------------------------------------------------------------------ attention
_CALL = struct.Struct("=13Q3q15if")


@functools.lru_cache(maxsize=256)
def _single_scratch(*sizes: int) -> int:
    return lib().st_attention_single8_scratch(*sizes)


def _attend(what: str, entry, q, pool, scales, layer, out, positions, seq_of_token, slots, block_table, nh, scale, window, status, *,
            only8=True, items=None, n_items=0, plan=None, max_keys=0) -> None:
    _same_device(what, q, pool, scales, out, positions, seq_of_token, slots, block_table, status, items,
                 plan.tiles if plan is not None else None)
    pages, layers, nkv, page_size, d, form = _pool8(what, pool, scales, layer, only8)
    act = _ACTS.get(q.dtype)
    if nh <= 0 or nh % nkv:
        raise KernelError(f"{what}: {nh} heads cannot share {nkv} key/value heads")
    if act is None or out.dtype is not q.dtype or (form > 1 and pool.dtype is not q.dtype):
        raise KernelError(f"{what}: queries and results of one type, float32 or bfloat16, that of a cache that is not in 8 bits")
    width, n = nh * d, out.shape[0]
    if q.dim() != 2 or q.shape != out.shape or q.shape[1] != width or not out.is_contiguous() or (width > 1 and q.stride(1) != 1):
        raise KernelError(f"{what}: q and out are [tokens, nh d], out contiguous, q's rows contiguous")
    stride = q.stride(0) if n > 1 else width
    if not scale > 0.0 or window < 0:
        raise KernelError(f"{what}: the scale is positive, the window not negative")
    _index(what, positions, seq_of_token, slots, block_table, n)
    n_tiles = total = max_rows = 0
    tiles = info = None
    if plan is not None:
        if plan.nh != nh or plan.nkv != nkv:
            raise KernelError(f"{what}: the plan is for {plan.nh} heads over {plan.nkv}")
        if plan.n_tokens > n or plan.n_seqs > slots.numel():
            raise KernelError(f"{what}: the plan names tokens or requests that are not there")
        tiles, info, items = plan.tiles, plan.info, plan.items
        n_items, n_tiles, total, max_rows = plan.n_items, plan.n_tiles, plan.total, plan.max_rows
    elif items is not None and not (items.dtype is _I32 and items.dim() == 1 and items.is_contiguous()):
        raise KernelError(f"{what}: items is a contiguous int32 tensor of one dimension")
    if stride != width:
        if plan is None or plan.kind != "portion" or stride < width:
            raise KernelError(f"{what}: q is contiguous")
    else:
        stride = 0
    st = status if status is not None else _tc_status_word(q.device)
    reach = min(block_table.shape[1] * page_size, 1 << 30)       # a hint of more keys than the table has room for is none
    max_keys = min(max_keys, reach) if max_keys > 0 else reach
    window = min(window, 0x7fffffff)
    if 0 < window < max_keys:
        max_keys = window
    # the parts of rows that several blocks leave, and those of single tokens
    floats = lib().st_attention_rows_scratch(n_tiles, nkv, d, total, 1 if n_items else 0) if total else 0
    if n_items:
        floats += _single_scratch(n_items, nh, nkv, d, page_size, block_table.shape[1], max_keys, act, form)
    scratch = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    call = _CALL.pack(q.data_ptr(), out.data_ptr(), pool.data_ptr(), _ptr(scales), block_table.data_ptr(), positions.data_ptr(),
                      _ptr(seq_of_token), slots.data_ptr(), _ptr(items), _ptr(tiles), _ptr(info), _ptr(scratch), st.data_ptr(),
                      stride, pages, floats, block_table.shape[1], layers, layer, nh, nkv, d, page_size, window, act, form,
                      n_items, n_tiles, total, max_rows, max_keys, scale)
    _check(entry(call, _stream()), what)


def attention_cache8_single(q: torch.Tensor, pool: torch.Tensor, scales: torch.Tensor, layer: int, out: torch.Tensor,
                            items: Optional[torch.Tensor], n_items: int, positions: torch.Tensor, seq_of_token: torch.Tensor,
                            slots: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float, window: int = 0, max_kv: int = 0,
                            status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of single query tokens over an 8-bit cache: what ``attention_decode`` does over a bfloat16 one.  ``q`` and ``out``
    [tokens, nh d] float32 or bfloat16; ``items`` lists the token indices that are served (-1: none; None: tokens 0 .. n_items - 1),
    the rows of ``out`` of other tokens stay.  ``max_kv``: about the most keys a token reads (0: what the block table has room
    for); it decides how the work is spread, not the result's meaning."""
    what = "attention_cache8_single"
    if not 0 <= n_items <= (items.numel() if items is not None else out.shape[0]):
        raise KernelError(f"{what}: n_items tokens are not there")
    _attend(what, lib().st_attention_single8, q, pool, scales, layer, out, positions, seq_of_token, slots, block_table, nh, scale,
            window, status, items=items, n_items=n_items, max_keys=max_kv)
    return out


def attention_cache8_tiles(q: torch.Tensor, pool: torch.Tensor, scales: torch.Tensor, layer: int, out: torch.Tensor, plan: RowPlan,
                           positions: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor, nh: int, scale: float,
                           window: int = 0, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of portions of prompts over an 8-bit cache: what ``attention_prefill`` does over a bfloat16 one.  ``plan``: from
    ``portion_plan``, of the same heads and window.  ``q`` may be the first columns of the q|k|v product (any row stride).  The
    portions' own keys and values have been written (``qkv_to_cache8``)."""
    what = "attention_cache8_tiles"
    if plan.kind != "portion" or plan.window != window:
        raise KernelError(f"{what}: the plan is from portion_plan, for this window")
    _attend(what, lib().st_attention_tiles8, q, pool, scales, layer, out, positions, None, slots, block_table, nh, scale, window,
            status, plan=plan)
    return out


def attention_shared_prefix(q: torch.Tensor, pool: torch.Tensor, layer: int, out: torch.Tensor, plan: RowPlan,
                            positions: torch.Tensor, seq_of_token: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor,
                            nh: int, scale: float, window: int = 0, scales: Optional[torch.Tensor] = None,
                            status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of single query tokens whose requests share their first keys: the result of ``attention_decode`` for every token of
    ``plan`` (from ``shared_prefix_plan``), with a group's shared keys and values read once for the group: each by the block table of
    the request of the group's first token that sees it, so that members may stand in any order.  Keys that no member sees, as they lie
    before all windows or behind all positions, need no page.  The cache is of q's type, or an 8-bit one with its ``scales``.

    A token's position may lie anywhere, inside the shared keys too: it sees keys 0 .. its own position (``window`` > 0: the last
    ``window`` of these).  A token that sees keys before those of the plan (its ``starts``) sets the status.  A value that is not finite reaches, in bfloat16 caches, all rows of its group that share it, also those
    whose window or position hides it; in the other forms only rows that see it."""
    what = "attention_shared_prefix"
    if plan.kind != "shared" or plan.window not in (0, window):
        raise KernelError(f"{what}: the plan is from shared_prefix_plan, for this window or for any")
    _attend(what, lib().st_attention_shared, q, pool, scales, layer, out, positions, seq_of_token, slots, block_table, nh, scale,
            window, status, only8=False, plan=plan, max_keys=plan.max_own)
    return out
