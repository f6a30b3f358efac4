"""Problems for the paged cache in 8 bits and for prefixes that requests share, and how far results may be off.

The quantised rows are worked out here from the definition (``quantised``), on the host, in float32 where the
definition says so.  What a pool stands for is scale * element, exact in float64, so that attention over it
is ``attention64`` of tests/_paged.py over pools of float64.  Its bound counts 4 roundings of a score and 16 of
a weight; a scale adds one to each (2 to either are left for them).  Weights that meet a matrix product in
parts of fewer bits than ``attention64`` counts add, with A = sum_j w_j |v_j| and e the relative error of a
weight: to the numerator e A, and e |out| <= e A for the sum of the weights (``parts``).
"""
import math
from types import SimpleNamespace

import torch

from tests._paged import attention64

HELD = [torch.int8, torch.float8_e4m3fn]


def quantised(x, held):
    """(elements, scales) of rows x (..., D), as the definition has them."""
    x = x.detach().cpu().float()
    a = x.abs().amax(-1)
    finite = torch.isfinite(a)
    a = torch.where(finite, a, torch.ones_like(a)).clamp(min=2.0 ** -100)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    if held == torch.int8:
        inverse = torch.full_like(a, 127.0) / a  # (127 / a would be 127 times the reciprocal)
        scale, elements = a / 127, (x * inverse[..., None]).round().to(torch.int8)
    else:
        m, e = torch.frexp(a.double() / 448)  # m in [1/2, 1): a / 448 <= 2^e, and 2^(e - 1) only for m = 1/2
        scale = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).float()
        elements = (x.double() / scale.double()[..., None]).float().to(held)
    return elements, torch.where(finite, scale, torch.full_like(scale, math.nan))


def bits(x):
    return x.detach().cpu().contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def stands_for(pool, scales):
    """What a pool's rows stand for, in float64."""
    return pool.detach().cpu().float().double() * scales.detach().cpu().double()[..., None]


def parts(dtype, shared, value_pages, call, keys):
    """What weights in parts may add to a bound: bf16 in one part (2^-8), for keys of shared pages; in two (2^-16) in
    the keys of pools of 8 bits.  fp16 in one part: 2^-11, and 2^-32 of the largest weight for every key, which
    the smallest fp16 is."""
    e = 0.0
    if shared:
        e = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}[dtype]
    elif dtype != torch.float32:
        e = 2.0 ** -16
    if e == 0.0:
        return 0.0
    finite = torch.nan_to_num(value_pages, 0.0)
    a, _ = call(value_pages.abs())
    return 2 * e * a + (keys * 2.0 ** -32 * finite.abs().max() if dtype == torch.float16 and shared else 0.0)


def expected(p, mask=None, scale=None):
    """(values, tolerances) of ``run``."""
    if p.scales is None:
        keys, values = (x.detach().cpu().double() for x in (p.key_pages, p.value_pages))
    else:
        keys, values = (stands_for(x, s) for x, s in zip((p.key_pages, p.value_pages), p.scales))
    query, size = p.query, scale
    if scale is not None and scale < 0:  # (attention64's bound is for positive ones)
        query, size = -query, -scale
    call = lambda v: attention64(query, keys, v, p.table, p.positions, mask=mask, scale=size)  # noqa: E731
    out, tol = call(values)
    return out, tol + parts(p.query.dtype, p.shared > 0, values, call, p.table.shape[1] * p.page)


def run(pkg, p, **kwargs):
    if p.shared:
        kwargs.setdefault('read_once', True)
    return pkg.paged_attention(p.query, p.key_pages, p.value_pages, p.table, p.positions, scales=p.scales,
                               shared_pages=p.shared, **kwargs)


def problem(device, lengths, *, held=None, shared=0, q_heads=16, kv_heads=8, width=128, page=16, dtype=torch.bfloat16,
            seed=0, layout='hnd', spare=3, table_width=None, query_scale=1.5):
    """Requests of ``lengths`` keys (0: a position of -1) over randomly ordered pages, the first ``shared`` of all of
    them; pool rows that belong to nobody, and table entries past a request's pages, are poisoned.  ``held``:
    the type of pools of 8 bits."""
    gen = torch.Generator().manual_seed(seed)
    counts = [max(0, -(-n // page) - shared) for n in lengths]
    total = sum(counts) + shared
    pages = total + spare
    order = torch.randperm(pages, generator=gen)[:total].to(torch.int32)
    widest = max(shared + max(counts, default=0), 1)
    table = torch.full((len(lengths), widest if table_width is None else table_width), -7, dtype=torch.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for b, n in enumerate(counts):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    shape = (pages, kv_heads, page, width)
    pools = [torch.randn(shape, generator=gen).to(dtype) for _ in range(2)]
    pools[0][..., 3::17] *= 3
    owned = torch.zeros(pages, page, dtype=torch.bool)
    owned[order[:shared].long()] = True
    for b, n in enumerate(lengths):
        j = torch.arange(shared * page, max(n, shared * page))
        owned[table[b].long()[j // page], j % page] = True
    scales = None
    if held is not None:
        pools, scales = zip(*(quantised(x, held) for x in pools))
        for pool, scale in zip(pools, scales):
            scale.masked_fill_(~owned[:, None], math.nan)
            pool.view(torch.uint8).masked_fill_(~owned[:, None, :, None], 0x7f)  # NaN as e4m3
    else:
        for pool in pools:
            pool.masked_fill_(~owned[:, None, :, None], math.nan)

    def placed(x):
        if layout == 'nhd':  # (pages, page, heads, ...) in memory
            return x.transpose(1, 2).contiguous().to(device).transpose(1, 2)
        return x.to(device)
    query = (torch.randn(len(lengths), 1, q_heads, width, generator=gen) * query_scale).to(dtype)
    positions = torch.tensor([n - 1 for n in lengths], dtype=torch.int64).reshape(-1)
    return SimpleNamespace(query=query.to(device), key_pages=placed(pools[0]), value_pages=placed(pools[1]), table=table.to(device),
                           scales=None if scales is None else tuple(placed(s) for s in scales), positions=positions.to(device),
                           lengths=list(lengths), page=page, shared=shared)
