"""Key-value cache kept in pages: storage without a capacity per request.

The slot arena gives every request as many rows as the longest one needs, and is regrown and
compacted as requests come, grow and go (``grow_arena``, ``SlotArena.move``).  Here a layer's
keys and values are pools of pages of ``page_size`` rows, ``(pages, kv_heads, page_size,
head_dim)``, and a request has a list of page numbers, its row of the page table: row j of
request b is row ``j % page_size`` of page ``page_table[b, j // page_size]``.

* ``paged_write`` - new key and value rows into their pages, one token per request or a padded
  batch of prompts (the paged counterpart of ``write`` / ``write_tokens``).
* ``paged_attention`` - grouped-query attention of one new token per request over its pages
  (the counterpart of ``decode_attention``).
* ``PagedArena`` / ``PagedCache`` - every layer's pools with their free pages, and the HF
  ``Cache`` over them that ``PackedAttention`` takes for one-token steps (the counterparts of
  ``SlotArena`` / ``SlotCache``, qwen3_tts_engine/continuous.py:97-169).

Page numbers live on the device and are not checked on the host: a number outside the pool names
no page, rows for it are not written and keys on it do not exist.  Two rows that are written to
one place of a pool in one call leave either of the two.  Inference only, as the rest of the
attention path.
"""
from __future__ import annotations

import torch
from transformers.cache_utils import Cache

from . import _lib
from .attention import _check_out, workspace
from .rotary import _share_memory

_pack_attention = _lib.packer(_lib.PagedArgs)
_pack_write = _lib.packer(_lib.PagedWriteArgs)
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


def paged_write(keys, values, key_pages, value_pages, page_table, positions, lengths=None):
    """Write the rows keys/values (B, Hkv, T, D) of every request into its pages, from row
    ``positions[b]`` on; one launch for both, bit-exact.

    key_pages/value_pages (pages, Hkv, page_size, D), by any strides with unit-stride rows;
    page_table (B, width) int32; positions (B,) int64; lengths (B,) int32: only the first
    ``lengths[b]`` of the T rows belong to request b (a right-padded batch).  bf16, fp16 or
    fp32.  Rows outside the table's ``width * page_size`` rows, or on no page of the pool, are
    skipped on the device; everything else of the pools stays as it was.  keys/values must not
    overlap the rows that are written."""
    if keys.ndim != 4 or values.shape != keys.shape:
        raise ValueError('Expected matching BNSD K/V')
    batch, heads, tokens, width = keys.shape
    kps, vps, ts, table_width = _check_pools(key_pages, value_pages, page_table, positions, batch)
    pages, page_heads, page_size, page_rows = key_pages.shape
    if page_heads != heads or page_rows != width:
        raise ValueError('pages must have the rows\' KV heads and head_dim')
    dtype = keys.dtype
    if dtype not in _TYPES or values.dtype != dtype or key_pages.dtype != dtype or value_pages.dtype != dtype:
        raise ValueError('paged K/V write supports bf16/fp16/fp32 tensors of one dtype')
    ks, vs = keys.stride(), values.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError('K/V rows must be unit-stride along head_dim')
    device = _lib.gpu_index(keys, values, key_pages, value_pages, page_table, positions)
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous():
            raise ValueError('lengths must be a contiguous int32 (batch,) tensor')
        _lib.gpu_index(keys, lengths)
    if batch == 0 or tokens == 0:
        return
    _lib.launch('q3t_paged_write', _pack_write(
        batch, heads, tokens, width, keys.element_size(), keys.data_ptr(), values.data_ptr(),
        ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], key_pages.data_ptr(), value_pages.data_ptr(),
        kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], pages, page_size,
        page_table.data_ptr(), table_width, ts, positions.data_ptr(), 0 if lengths is None else lengths.data_ptr()),
        device, 'paged write')


def paged_attention(query, key_pages, value_pages, page_table, positions, *, scale=None, mask=None, out=None):
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
    rows hold; a request that attends nothing gets zero rows."""
    return _attend(_attention_call(query, key_pages, value_pages, page_table, positions, scale, mask, out))


def _attention_call(query, key_pages, value_pages, page_table, positions, scale, mask, out):
    """An attention launch whose arguments have been checked, for ``_attend``: (query, out, device index, fields,
    bytes of workspace); nothing has been launched on the pools yet."""
    if query.ndim != 4 or query.shape[1] != 1:
        raise ValueError('paged attention takes one token per request, (batch, 1, heads, head_dim)')
    batch, _, q_heads, head_dim = query.shape
    kps, vps, ts, table_width = _check_pools(key_pages, value_pages, page_table, positions, batch)
    pages, kv_heads, page_size, width = key_pages.shape
    if width != head_dim or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError('head_dim mismatch or q_heads not a multiple of kv_heads')
    dtype = query.dtype
    if dtype not in _TYPES or key_pages.dtype != dtype or value_pages.dtype != dtype:
        raise ValueError('paged attention supports bf16, fp16 or fp32 tensors of one dtype')
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
        return query, out, device, None, 0
    if query.data_ptr() % 16 or (qs[0] | qs[2]) * query.element_size() % 16:
        query = query.clone(memory_format=torch.contiguous_format)  # rows that 16-byte loads do not fit
        qs = query.stride()
    fields = (
        batch, q_heads, kv_heads, head_dim, _TYPES[dtype], ctx, head_dim ** -0.5 if scale is None else scale, 0,
        query.data_ptr(), qs[0], qs[2], key_pages.data_ptr(), value_pages.data_ptr(),
        kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], pages, page_size,
        page_table.data_ptr(), table_width, ts, positions.data_ptr(), *mask_fields, out.data_ptr(), os[0], os[2])
    need = _lib.packed('q3t_paged_workspace_bytes')(_pack_attention(*fields, 0, 0))
    if need < 0:
        raise ValueError('paged attention: unsupported shape or dtype')
    return query, out, device, fields, need


def _attend(call):
    """Launches what ``_attention_call`` has checked; the caller keeps its tensors."""
    query, out, device, fields, need = call
    if fields is None:
        return out
    with _lib.on_device(device) as stream:
        ws = workspace(query.device, need, stream)
        status = _lib.packed('q3t_paged_attention')(_pack_attention(*fields, ws.data_ptr(), ws.numel()), stream)
    if status != _lib.Q3T_OK:
        _lib.check(status, 'paged attention')
    return out


class PagedArena:
    """Pages of KV storage for every talker layer, and which of them are free.

    ``packed`` is (2 * layers, pages, kv_heads, page_size, head_dim), keys first, as the slot
    arena's packed tensor is; a page number names the same page of every layer."""

    def __init__(self, reference, pages, page_size=16):
        if pages < 1 or page_size < 1:
            raise ValueError('an arena needs pages of at least one row')
        self.reference = reference
        self.pages = pages
        self.page_size = page_size
        weight, config = next(reference.parameters()), reference.config
        layers = len(reference.layers)
        self.packed = torch.zeros((2 * layers, pages, config.num_key_value_heads, page_size, config.head_dim),
                                  device=weight.device, dtype=weight.dtype)
        self.keys = list(self.packed[:layers].unbind(0))
        self.values = list(self.packed[layers:].unbind(0))
        self._free = list(range(pages - 1, -1, -1))
        self._used = set()

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

    def release(self, pages):
        """Give pages back; ValueError, and none released, unless each is in use and named once."""
        pages = list(pages)
        if len(set(pages)) != len(pages) or not self._used.issuperset(pages):
            raise ValueError('only pages in use can be released, each once')
        self._used.difference_update(pages)
        self._free.extend(pages)

    def page_table(self, requests, width=None):
        """An int32 (requests, width) table on the arena's device from one list of page numbers per
        request (width: the longest list's by default); -1 past a request's pages."""
        longest = max((len(pages) for pages in requests), default=0)
        width = max(longest, 1) if width is None else width
        if longest > width:
            raise ValueError('a request has more pages than the table is wide')
        rows = [list(pages) + [-1] * (width - len(pages)) for pages in requests]
        return torch.tensor(rows, dtype=torch.int32).reshape(len(rows), width).to(self.packed.device)

    def load(self, page_table, cache, lengths):
        """Copy the rows of a prefill cache (``cache.layers[i].keys`` / ``.values``, (B, kv_heads,
        length, head_dim)) into the pages of their requests: row b's first ``lengths[b]`` (int32,
        device) positions, to positions 0 on."""
        if len(cache.layers) != len(self.keys):
            raise ValueError('the cache and the arena must have the same layers')
        start = torch.zeros(page_table.shape[0], device=page_table.device, dtype=torch.int64)
        for layer, keys, values in zip(cache.layers, self.keys, self.values):
            paged_write(layer.keys, layer.values, keys, values, page_table, start, lengths)


class PagedCache(Cache):
    """HF ``Cache`` over a paged arena for one-token steps: ``update`` writes request b's row at
    ``positions[b]`` and returns the layer's pools; ``step`` attends over them too, as
    ``PackedAttention`` calls it.  ``page_table`` and ``positions`` are read at every step as they are
    then, so a captured step follows changes of their contents.

    The lengths live on the device, so ``get_seq_length`` is 0: pass the model ``position_ids``, and as
    its mask None (a request then attends its keys up to its position) or one over the table's rows."""

    def __init__(self, arena, page_table, positions):
        super().__init__(layers=[])
        self.arena = arena
        self.page_table = page_table
        self.positions = positions

    def update(self, keys, values, layer_idx, cache_kwargs=None):
        if keys.shape[2] != 1:
            raise ValueError('a PagedCache takes one token per request; prompts are loaded with PagedArena.load')
        key_pages, value_pages = self.arena.keys[layer_idx], self.arena.values[layer_idx]
        paged_write(keys, values, key_pages, value_pages, self.page_table, self.positions)
        return key_pages, value_pages

    def step(self, query, keys, values, layer_idx, *, scale=None, mask=None):
        """A layer's step: ``update`` with keys/values (B, Hkv, 1, D), then ``paged_attention`` of query
        (B, 1, Hq, D).  A call that the attention refuses writes nothing.

        The mask must end in the key dimension: the one that transformers' ``create_causal_mask``
        builds ends in a single key, since it cannot know the lengths, and is refused."""
        if getattr(mask, 'shape', ())[-1:] == (1,) and self.page_table.shape[1] * self.arena.page_size > 1:
            raise ValueError('the mask of a paged step must end in the key dimension')
        call = _attention_call(query, self.arena.keys[layer_idx], self.arena.values[layer_idx], self.page_table,
                               self.positions, scale, mask, None)
        self.update(keys, values, layer_idx)
        return _attend(call)

    def get_seq_length(self, layer_idx=0):
        return 0  # the lengths are per request and live on the device: positions + 1
