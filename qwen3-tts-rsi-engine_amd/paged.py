"""Key-value cache kept in pages: storage without a capacity per request.

The slot arena gives every request as many rows as the longest one needs, and is regrown and
compacted as requests come, grow and go (``grow_arena``, ``SlotArena.move``).  Here a layer's
keys and values are pools of pages of ``page_size`` rows, ``(pages, kv_heads, page_size,
head_dim)``, and a request has a list of page numbers, its row of the page table: row j of
request b is row ``j % page_size`` of page ``page_table[b, j // page_size]``.

* ``paged_write`` - new key and value rows into their pages, one token per request or a padded
  batch of prompts (the paged counterpart of ``write`` / ``write_tokens``).
* ``paged_attention`` - grouped-query attention of one new token per request over its pages
  (the counterpart of ``decode_attention``); the pages that a whole batch begins with are read once
  for all of it (``shared_pages``).
* ``paged_read`` - rows out of their pages, the inverse of ``paged_write`` (the counterpart of
  ``copy_packed_prefix`` out of a slot).
* ``PagedArena`` / ``PagedCache`` - every layer's pools with their free pages, and the HF
  ``Cache`` over them that ``PackedAttention`` takes for one-token steps (the counterparts of
  ``SlotArena`` / ``SlotCache``, qwen3_tts_engine/continuous.py:97-169).

Pools may hold 8-bit elements, int8 or float8_e4m3fn, in place of the rows' own type: half the
memory, and half the reading of a step.  Every key (value) row of a pool then has a float32 scale, and
``scales`` is the pair of their tensors, (pages, kv_heads, page_size) each.  A row x with a = max(2^-100,
max |x|) is held, in float32 arithmetic, as

* int8: round(x * (127 / a)), ties to even, with the scale a / 127;
* e4m3: x / s rounded to the nearest e4m3 value, ties to even, with the scale s, the smallest power of two
  for which a <= 448 s;

and stands for scale times element.  A row with an infinity or a NaN in it stands for NaN.

Page numbers live on the device and are not checked on the host: a number outside the pool names
no page, rows for it are not written and keys on it do not exist.  Two rows that are written to
one place of a pool in one call leave either of the two (in 8 bits, of one the row and of the other
the scale, perhaps).  Inference only, as the rest of the attention path.
"""
from __future__ import annotations

import torch
from transformers.cache_utils import Cache

from . import _lib
from .attention import _check_out, workspace
from .rotary import _share_memory

_pack_attention = _lib.packer(_lib.PagedArgs)
_pack_write = _lib.packer(_lib.PagedWriteArgs)
_pack_read = _lib.packer(_lib.PagedReadArgs)
_pack_scales = _lib.packer(_lib.PagedScales)
_HELD = {torch.int8: _lib.Q3T_I8, torch.float8_e4m3fn: _lib.Q3T_E4M3}  # types of pools with scales
_SHARE = {None: 0, True: 1, False: 2}  # Q3T_SHARE_*
_TYPES = {torch.bfloat16: _lib.Q3T_BF16, torch.float16: _lib.Q3T_F16, torch.float32: _lib.Q3T_F32}


def _check_pools(key_pages, value_pages, page_table, positions, batch):
    """(strides of the key pages, of the value pages, of the page table, its width)."""
    if key_pages.ndim != 4 or value_pages.shape != key_pages.shape:
        raise ValueError('key and value pages must be (pages, kv_heads, page_size, head_dim) of one shape')
    ks, vs = key_pages.stride(), value_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError('rows must be unit-stride along head_dim')
    if page_table.ndim != 2 or page_table.dtype != torch.int32:
        raise ValueError('page_table must be an int32 (batch, pages) tensor')
    (rows, width), ts = page_table.shape, page_table.stride()
    if rows != batch or width < 1 or (width > 1 and ts[1] != 1):
        raise ValueError('page_table must have a unit-stride row of page numbers per request')
    if positions.dtype != torch.int64 or positions.shape != (batch,) or not positions.is_contiguous():
        raise ValueError('positions must be a contiguous int64 (batch,) tensor')
    return ks, vs, ts[0], width


def _check_scales(scales, key_pages, value_pages, dtype):
    """The fields of the scales of pools of 8 bits, as bytes; None for pools of the rows' own ``dtype``."""
    held = key_pages.dtype
    if value_pages.dtype != held or (held not in _HELD and held != dtype):
        raise ValueError('key and value pages must be of the rows\' dtype, or int8 or float8_e4m3fn')
    if (scales is None) != (held not in _HELD):
        raise ValueError('pages of int8 or float8_e4m3fn have scales, others have none')
    if scales is None:
        return None
    key_scales, value_scales = scales
    shape = key_pages.shape[:3]
    for x in (key_scales, value_scales):
        if x.dtype != torch.float32 or x.shape != shape:
            raise ValueError('scales must be two float32 (pages, kv_heads, page_size) tensors')
    _lib.gpu_index(key_pages, key_scales, value_scales)
    return _pack_scales(_HELD[held], key_scales.data_ptr(), value_scales.data_ptr(), *key_scales.stride(), *value_scales.stride())


def _check_lengths(lengths, batch, rows):
    if lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError('lengths must be a contiguous int32 (batch,) tensor')
    _lib.gpu_index(rows, lengths)


def _rows_overlap(row, count, stride, other_count, other_stride):
    """Whether any two rows of ``row`` elements at i * stride + j * other_stride, i < count, j < other_count,
    share one."""
    (inner, inner_count), (outer, outer_count) = sorted(((stride, count), (other_stride, other_count)))
    if inner_count > 1 and inner < row:
        return True
    if outer_count == 1 or outer >= (inner_count - 1) * inner + row:
        return False
    # a row i outer strides on lies between two rows of the inner dimension, or past their last
    return outer < row or inner_count > 1 and any(
        i * outer % inner < row and i * outer // inner < inner_count
        or -i * outer % inner < row and -(-i * outer // inner) < inner_count for i in range(1, outer_count))


def paged_write(keys, values, key_pages, value_pages, page_table, positions, lengths=None, *, scales=None):
    """Write the rows keys/values (B, Hkv, T, D) of every request into its pages, from row
    ``positions[b]`` on; one launch for both, bit-exact.

    key_pages/value_pages (pages, Hkv, page_size, D), by any strides with unit-stride rows;
    page_table (B, width) int32; positions (B,) int64; lengths (B,) int32: only the first
    ``lengths[b]`` of the T rows belong to request b (a right-padded batch).  bf16, fp16 or
    fp32.  Rows outside the table's ``width * page_size`` rows, or on no page of the pool, are
    skipped on the device; everything else of the pools stays as it was.  keys/values must not
    overlap the rows that are written.

    With ``scales`` the pools are int8 or float8_e4m3fn, of head_dim 64 or 128, their rows starting at
    multiples of 16 bytes, and the rows are quantised as they are written, their scales beside them."""
    if keys.ndim != 4 or values.shape != keys.shape:
        raise ValueError('Expected matching BNSD K/V')
    batch, heads, tokens, width = keys.shape
    kps, vps, ts, table_width = _check_pools(key_pages, value_pages, page_table, positions, batch)
    pages, page_heads, page_size, page_rows = key_pages.shape
    if page_heads != heads or page_rows != width:
        raise ValueError('pages must have the rows\' KV heads and head_dim')
    dtype = keys.dtype
    if dtype not in _TYPES or values.dtype != dtype:
        raise ValueError('paged K/V write supports bf16/fp16/fp32 tensors of one dtype')
    held = None
    if scales is not None or key_pages.dtype != dtype or value_pages.dtype != dtype:
        held = _check_scales(scales, key_pages, value_pages, dtype)
    ks, vs = keys.stride(), values.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError('K/V rows must be unit-stride along head_dim')
    device = _lib.gpu_index(keys, values, key_pages, value_pages, page_table, positions)
    if lengths is not None:
        _check_lengths(lengths, batch, keys)
    if batch == 0 or tokens == 0:
        return
    args = _pack_write(
        batch, heads, tokens, width, keys.element_size(), keys.data_ptr(), values.data_ptr(),
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], key_pages.data_ptr(), value_pages.data_ptr(),
        kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], pages, page_size,
        page_table.data_ptr(), table_width, ts, positions.data_ptr(), 0 if lengths is None else lengths.data_ptr())
    if held is None:
        _lib.launch('q3t_paged_write', args, device, 'paged write')
    else:
        _lib.launch('q3t_paged_write_quantized', args, device, 'paged write', _TYPES[dtype], held)


def paged_read(key_pages, value_pages, page_table, positions, tokens, lengths=None, *, scales=None, dtype=None, out=None):
    """Rows out of their pages, the inverse of ``paged_write``: (keys, values), each (B, Hkv, ``tokens``, D),
    whose row t of request b is that of position ``positions[b] + t``; one launch for both.

    Pools, page_table (B, width) int32, positions (B,) int64 and lengths (B,) int32 as there.  Rows past the
    first ``lengths[b]``, outside the table's ``width * page_size`` rows or on no page of the pool are
    zeros.  Pools of bf16, fp16 or fp32 are copied bit for bit.  With ``scales`` the pools are int8 or
    float8_e4m3fn, of head_dim 64 or 128, their rows starting at multiples of 16 bytes, and elements are scale times
    element in float32, rounded to ``dtype`` (bf16, fp16 or fp32; bf16 unless ``out`` is given).  ``out``: the
    pair of tensors to write to, by any strides with unit-stride rows that share no memory; they must not
    overlap the pools."""
    if isinstance(tokens, bool) or not isinstance(tokens, int) or tokens < 0:
        raise ValueError('tokens must be the number of rows to read')
    batch = positions.shape[0] if positions.ndim else 0
    kps, vps, ts, table_width = _check_pools(key_pages, value_pages, page_table, positions, batch)
    pages, heads, page_size, width = key_pages.shape
    if dtype is None:
        dtype = out[0].dtype if out is not None else torch.bfloat16 if scales is not None else key_pages.dtype
    if dtype not in _TYPES:
        raise ValueError('paged read supports bf16/fp16/fp32 rows')
    held = _check_scales(scales, key_pages, value_pages, dtype)
    device = _lib.gpu_index(key_pages, value_pages, page_table, positions)
    if lengths is not None:
        _check_lengths(lengths, batch, key_pages)
    shape = (batch, heads, tokens, width)
    if out is None:
        keys = torch.empty(shape, dtype=dtype, device=key_pages.device)
        values = torch.empty_like(keys)
    else:
        keys, values = out
        for x in (keys, values):
            _check_out(x, shape, dtype, key_pages.device, 'paged read')
        if _share_memory(keys) or _share_memory(values) or _share_memory(keys, values):
            raise ValueError('paged read: rows of out must not share memory')
    if batch == 0 or tokens == 0:
        return keys, values
    ks, vs = keys.stride(), values.stride()
    _lib.launch('q3t_paged_read', _pack_read(
        batch, heads, tokens, width, _TYPES[dtype], keys.data_ptr(), values.data_ptr(),
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], key_pages.data_ptr(), value_pages.data_ptr(),
        kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], pages, page_size,
        page_table.data_ptr(), table_width, ts, positions.data_ptr(), 0 if lengths is None else lengths.data_ptr()),
        device, 'paged read', held)
    return keys, values


def paged_attention(query, key_pages, value_pages, page_table, positions, *, scale=None, mask=None, out=None,
                    scales=None, shared_pages=0, read_once=None):
    """Attention of one new token per request: query (B, 1, Hq, D) over the keys
    0 ... positions[b] of request b, which its row of ``page_table`` (B, width) int32 finds in
    key_pages/value_pages (pages, Hkv, page_size, D), by any strides with unit-stride rows.
    Returns (B, 1, Hq, D); bf16, fp16 or fp32, head_dim 64 or 128, any number of query heads
    that is a multiple of the KV heads.  Rows of the pools start at multiples of 16 bytes, and
    there are at most 64512 requests times KV heads (times blocks of 16 query heads of one).  ``out``
    may be the query itself; other tensors of the call it must not overlap.

    ``mask``: SDPA-style, broadcastable to (B, 1, 1, K) with K at most ``width * page_size``:
    bool (True attends) or additive (bf16 / fp16 / fp32, added to the scaled scores in float32).
    A mask that ends in K > 1 gives a request K keys at most; without one, or with one term for all
    keys (a last dimension of 1), it has ``width * page_size``.  A position outside those attends
    nothing.  A key under -inf (or False), or on no page of the pool, does not exist, whatever its
    rows hold; a request that attends nothing gets zero rows.

    ``scales``: the pools are int8 or float8_e4m3fn, and the keys and values those that they stand for.

    ``shared_pages``: the first that many entries are the same pages in every row of ``page_table``, also in
    rows of requests that attend nothing, as where all requests have one prompt in front; only in rows that requests have
    left may all entries be numbers of no page (-1), and nothing is attended by those.  What each
    request attends is as without it, but where it saves enough (``read_once`` True or False: always, or
    never) the keys on them are read once for the whole batch, their weights then held in two parts of the queries'
    type (of 16 bits): a relative 2^-16 in bf16, 2^-22 in fp16.  Pools of 8 bits are
    attended request by request, whatever ``read_once`` says."""
    return _attend(_attention_call(query, key_pages, value_pages, page_table, positions, scale, mask, out, scales, shared_pages,
                                   read_once))


def _attention_call(query, key_pages, value_pages, page_table, positions, scale, mask, out, scales=None, shared_pages=0,
                    read_once=None):
    """An attention launch whose arguments have been checked, for ``_attend``: (query, out, device index, fields,
    bytes of workspace, scales and shared pages if any); nothing has been launched on the pools yet."""
    if query.ndim != 4 or query.shape[1] != 1:
        raise ValueError('paged attention takes one token per request, (batch, 1, heads, head_dim)')
    batch, _, q_heads, head_dim = query.shape
    kps, vps, ts, table_width = _check_pools(key_pages, value_pages, page_table, positions, batch)
    pages, kv_heads, page_size, width = key_pages.shape
    if width != head_dim or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError('head_dim mismatch or q_heads not a multiple of kv_heads')
    dtype = query.dtype
    if dtype not in _TYPES:
        raise ValueError('paged attention supports bf16, fp16 or fp32 tensors of one dtype')
    held = None
    if scales is not None or key_pages.dtype != dtype or value_pages.dtype != dtype:
        held = _check_scales(scales, key_pages, value_pages, dtype)
    if isinstance(shared_pages, bool) or not isinstance(shared_pages, int) or not 0 <= shared_pages <= table_width:
        raise ValueError('shared_pages must be a number of entries of the page table')
    if read_once not in _SHARE:
        raise ValueError('read_once must be True, False or None')
    qs = query.stride()
    if qs[3] != 1:
        raise ValueError('rows must be unit-stride along head_dim')
    device = _lib.gpu_index(query, key_pages, value_pages, page_table, positions)
    ctx = table_width * page_size
    mask_fields = (0, 0, 0, 0)
    if mask is not None:
        if getattr(mask, 'dtype', None) not in _lib.DTYPE_CODES:
            raise ValueError('attention mask must be bool, bf16, fp16 or fp32')
        if not 1 <= mask.ndim <= 4 or not 1 <= mask.shape[-1] <= ctx or any(n != 1 for n in mask.shape[-3:-1]):
            raise ValueError('the mask must be broadcastable to (batch, 1, 1, keys), its keys within the page table')
        _lib.gpu_index(query, mask)
        if mask.shape[-1] > 1:  # else one term for all keys
            ctx = mask.shape[-1]
        try:
            rows = mask.expand(batch, 1, 1, ctx)
        except RuntimeError:
            raise ValueError('the mask must be broadcastable to (batch, 1, 1, keys)') from None
        mask_fields = (mask.data_ptr(), _lib.DTYPE_CODES[mask.dtype], rows.stride(0), rows.stride(3))
        if max(mask_fields[2:]) >= 1 << 32:
            raise ValueError('paged attention: mask strides must be below 2^32 elements')
    if out is None:
        out, os = torch.empty_like(query, memory_format=torch.contiguous_format), (q_heads * head_dim, 0, head_dim)
    else:
        _check_out(out, (batch, 1, q_heads, head_dim), dtype, query.device, 'paged attention')
        os = out.stride()
        if _rows_overlap(head_dim, batch, os[0], q_heads, os[2]):
            raise ValueError('paged attention: rows of out must not share memory')
        same = out.data_ptr() == query.data_ptr() and all(n == 1 or o == s for n, o, s in zip(out.shape, os, qs))
        if not same and _share_memory(query, out):
            raise ValueError('paged attention: out must be the query itself, row by row, or lie apart from it')
    if batch == 0:
        return query, out, device, None, 0, None
    if query.data_ptr() % 16 or (qs[0] | qs[2]) * query.element_size() % 16:
        query = query.clone(memory_format=torch.contiguous_format)  # rows that 16-byte loads do not fit
        qs = query.stride()
    fields = (
        batch, q_heads, kv_heads, head_dim, _TYPES[dtype], ctx, head_dim ** -0.5 if scale is None else scale, _SHARE[read_once],
        query.data_ptr(), qs[0], qs[2], key_pages.data_ptr(), value_pages.data_ptr(),
        kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], pages, page_size,
        page_table.data_ptr(), table_width, ts, positions.data_ptr(), *mask_fields, out.data_ptr(), os[0], os[2])
    more = None
    if held is not None or shared_pages:
        # (the last row that a request may have is left to the requests)
        more = held, min(shared_pages, (ctx - 1) // page_size)
        need = _lib.packed('q3t_paged_workspace_bytes_with')(_pack_attention(*fields, 0, 0), *more)
    else:
        need = _lib.packed('q3t_paged_workspace_bytes')(_pack_attention(*fields, 0, 0))
    if need < 0:
        raise ValueError('paged attention: unsupported shape or dtype')
    return query, out, device, fields, need, more


def _attend(call):
    """Launches what ``_attention_call`` has checked; the caller keeps its tensors."""
    query, out, device, fields, need, more = call
    if fields is None:
        return out
    with _lib.on_device(device) as stream:
        ws = workspace(query.device, need, stream)
        args = _pack_attention(*fields, ws.data_ptr(), ws.numel())
        if more is None:
            status = _lib.packed('q3t_paged_attention')(args, stream)
        else:
            status = _lib.packed('q3t_paged_attention_with')(args, *more, stream)
    if status != _lib.Q3T_OK:
        _lib.check(status, 'paged attention')
    return out


class PagedArena:
    """Pages of KV storage for every talker layer, and which of them are free.

    ``packed`` is (2 * layers, pages, kv_heads, page_size, head_dim), keys first, as the slot
    arena's packed tensor is; a page number names the same page of every layer.

    ``dtype``: torch.int8 or torch.float8_e4m3fn holds the rows, of head_dim 64 or 128, in 8 bits; their scales are ``packed_scales``
    (2 * layers, pages, kv_heads, page_size), and ``scales[i]`` is layer i's pair of them (None otherwise)."""

    def __init__(self, reference, pages, page_size=16, dtype=None):
        if pages < 1 or page_size < 1:
            raise ValueError('an arena needs pages of at least one row')
        self.reference = reference
        self.pages = pages
        self.page_size = page_size
        weight, config = next(reference.parameters()), reference.config
        if dtype is not None and dtype != weight.dtype and dtype not in _HELD:
            raise ValueError('an arena holds rows of the model\'s dtype, int8 or float8_e4m3fn')
        if dtype in _HELD and config.head_dim not in (64, 128):
            raise ValueError('rows of 8 bits have a head_dim of 64 or 128')
        layers = len(reference.layers)
        shape = (2 * layers, pages, config.num_key_value_heads, page_size, config.head_dim)
        self.packed = torch.zeros(shape, device=weight.device, dtype=weight.dtype if dtype is None else dtype)
        self.packed_scales, self.scales = None, [None] * layers
        if dtype in _HELD:
            self.packed_scales = torch.zeros(shape[:4], device=weight.device)
            self.scales = list(zip(self.packed_scales[:layers].unbind(0), self.packed_scales[layers:].unbind(0)))
        self.keys = list(self.packed[:layers].unbind(0))
        self.values = list(self.packed[layers:].unbind(0))
        self._free = list(range(pages - 1, -1, -1))
        self._used = set()
        self._shares = {}  # of pages that are released more than once: times beyond the first

    @property
    def free_pages(self):
        return len(self._free)

    def pages_for(self, rows):
        """Pages that ``rows`` rows take."""
        return -(-rows // self.page_size)

    def allocate(self, count):
        """``count`` free page numbers, now in use; ValueError, and none taken, when fewer are free."""
        if not 0 <= count <= len(self._free):
            raise ValueError(f'{count} pages asked for, {len(self._free)} are free')
        taken = [self._free.pop() for _ in range(count)]
        self._used.update(taken)
        return taken

    def share(self, pages):
        """Another request has ``pages`` too, and releases them as well: a page is free again once it has
        been released as often as it was allocated and shared.  Returns the pages; ValueError, and none
        shared, unless each is in use and named once."""
        pages = list(pages)
        if len(set(pages)) != len(pages) or not self._used.issuperset(pages):
            raise ValueError('only pages in use can be shared, each once')
        for page in pages:
            self._shares[page] = self._shares.get(page, 0) + 1
        return pages

    def release(self, pages):
        """Give pages back; ValueError, and none released, unless each is in use and named once."""
        pages = list(pages)
        if len(set(pages)) != len(pages) or not self._used.issuperset(pages):
            raise ValueError('only pages in use can be released, each once')
        for page in pages:
            others = self._shares.pop(page, 0)
            if others > 1:
                self._shares[page] = others - 1
            elif others == 0:
                self._used.remove(page)
                self._free.append(page)

    def page_table(self, requests, width=None):
        """An int32 (requests, width) table on the arena's device from one list of page numbers per
        request (width: the longest list's by default); -1 past a request's pages."""
        longest = max((len(pages) for pages in requests), default=0)
        width = max(longest, 1) if width is None else width
        if longest > width:
            raise ValueError('a request has more pages than the table is wide')
        rows = [list(pages) + [-1] * (width - len(pages)) for pages in requests]
        return torch.tensor(rows, dtype=torch.int32).reshape(len(rows), width).to(self.packed.device)

    def load(self, page_table, cache, lengths, start=None):
        """Copy the rows of a prefill cache (``cache.layers[i].keys`` / ``.values``, (B, kv_heads,
        length, head_dim)) into the pages of their requests: row b's first ``lengths[b]`` (int32,
        device) positions, to positions ``start[b]`` (int64, device; 0) on."""
        if len(cache.layers) != len(self.keys):
            raise ValueError('the cache and the arena must have the same layers')
        if start is None:
            start = torch.zeros(page_table.shape[0], device=page_table.device, dtype=torch.int64)
        for layer, keys, values, scales in zip(cache.layers, self.keys, self.values, self.scales):
            paged_write(layer.keys, layer.values, keys, values, page_table, start, lengths, scales=scales)

    def read(self, page_table, tokens, lengths=None, start=None):
        """The rows of requests, the inverse of ``load``: ``tokens`` positions from ``start[b]`` (int64, device; 0) on as a
        packed cache (2 * layers, B, kv_heads, tokens, head_dim) of the model's dtype, as
        ``SlotArena.load_packed`` takes it, zeros past the first ``lengths[b]`` (int32, device) rows of request b."""
        if start is None:
            start = torch.zeros(page_table.shape[0], device=page_table.device, dtype=torch.int64)
        layers, (_, heads, _, width) = len(self.keys), self.keys[0].shape
        packed = torch.empty((2 * layers, page_table.shape[0], heads, tokens, width), device=self.packed.device,
                             dtype=next(self.reference.parameters()).dtype)
        for i in range(layers):
            paged_read(self.keys[i], self.values[i], page_table, start, tokens, lengths, scales=self.scales[i],
                       out=(packed[i], packed[layers + i]))
        return packed


class PagedCache(Cache):
    """HF ``Cache`` over a paged arena for one-token steps: ``update`` writes request b's row at
    ``positions[b]`` and returns the layer's pools; ``step`` attends over them too, as
    ``PackedAttention`` calls it.  ``page_table`` and ``positions`` are read at every step as they are
    then, so a captured step follows changes of their contents.  ``shared_pages``: entries that all rows of the
    table begin with, as ``paged_attention`` takes them (all but retired requests' rows, of -1), and its ``read_once``; no request
    may write to those pages.

    The lengths live on the device, so ``get_seq_length`` is 0: pass the model ``position_ids``, and as
    its mask None (a request then attends its keys up to its position) or one over the table's rows."""

    def __init__(self, arena, page_table, positions, shared_pages=0, read_once=None):
        super().__init__(layers=[])
        self.arena = arena
        self.page_table = page_table
        self.positions = positions
        self.shared_pages = shared_pages
        self.read_once = read_once

    def update(self, keys, values, layer_idx, cache_kwargs=None):
        if keys.shape[2] != 1:
            raise ValueError('a PagedCache takes one token per request; prompts are loaded with PagedArena.load')
        key_pages, value_pages = self.arena.keys[layer_idx], self.arena.values[layer_idx]
        paged_write(keys, values, key_pages, value_pages, self.page_table, self.positions,
                    scales=self.arena.scales[layer_idx])
        return key_pages, value_pages

    def step(self, query, keys, values, layer_idx, *, scale=None, mask=None):
        """A layer's step: ``update`` with keys/values (B, Hkv, 1, D), then ``paged_attention`` of query
        (B, 1, Hq, D).  A call that the attention refuses writes nothing.

        The mask must end in the key dimension: the one that transformers' ``create_causal_mask``
        builds ends in a single key, since it cannot know the lengths, and is refused."""
        if getattr(mask, 'shape', ())[-1:] == (1,) and self.page_table.shape[1] * self.arena.page_size > 1:
            raise ValueError('the mask of a paged step must end in the key dimension')
        call = _attention_call(query, self.arena.keys[layer_idx], self.arena.values[layer_idx], self.page_table,
                               self.positions, scale, mask, None, self.arena.scales[layer_idx], self.shared_pages,
                               *(() if self.read_once is None else (self.read_once,)))
        self.update(keys, values, layer_idx)
        return _attend(call)

    def get_seq_length(self, layer_idx=0):
        return 0  # the lengths are per request and live on the device: positions + 1
