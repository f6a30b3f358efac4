"""Problems for the paged cache and the float64 values that its operators are held to.

``attention64`` computes softmax attention of one token per request from the definition, on the
host in float64, and with it how far a result may be off.  With u = 2^-24 (float32's rounding) and,
per (request, head), s_j the scaled scores, w the weights and A = sum_j w_j |v_j|:

* a score: D products and sums in float32 and a few roundings after, each at most 2 u (matrix
  instructions may truncate): ds <= 2 (D + 4) u max_j scale sum_i |q_i k_ji| + 4 u max_j |s_j|
  (the largest |s_j| includes the mask's finite terms above half the type's lowest);
* a weight: exp moves by 2 ds and some units of exp2 and of the parts it is split into: 2 ds + 16 u
  (+ 2^-21 for 16-bit types, whose weights are kept in parts of 22 bits or more);
* the sums over the keys: a chain of at most L/16 + 64 additions: 2 (L/16 + 64) u A;
* both numerator and denominator carry these, so an element may be off by
  A (2 (2 ds + 16 u + 2^-21) + 4 (L/16 + 64) u), and by the output's rounding, half a step of it:
  eps/2 |out| (and half the smallest subnormal, for fp16).
"""
import math
from types import SimpleNamespace

import torch

U = 2.0 ** -24


def problem(device, lengths, *, q_heads=16, kv_heads=8, width=128, page=16, dtype=torch.bfloat16, seed=0,
            layout='hnd', spare=3, table_width=None, query_scale=2.0):
    """Requests of ``lengths`` keys (0: a position of -1) over randomly ordered pages; pool rows that
    belong to nobody, and table entries past a request's pages, are poisoned."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen)[:sum(counts)].to(torch.int32)
    widest = max(max(counts, default=1), 1)
    table = torch.full((len(lengths), widest if table_width is None else table_width), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv_heads, page, width)
    pools = [torch.randn(shape, generator=gen).to(dtype) for _ in range(2)]
    owned = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        owned[table[b].long()[j // page], j % page] = True
    for pool in pools:
        pool.masked_fill_(~owned[:, None, :, None], math.nan)
    if layout == 'nhd':  # (pages, page, heads, width) in memory
        pools = [p.transpose(1, 2).contiguous().to(device).transpose(1, 2) for p in pools]
    else:
        pools = [p.to(device) for p in pools]
    query = (torch.randn(len(lengths), 1, q_heads, width, generator=gen) * query_scale).to(dtype)
    positions = torch.tensor([n - 1 for n in lengths], dtype=torch.int64).reshape(-1)
    return SimpleNamespace(query=query.to(device), key_pages=pools[0], value_pages=pools[1], table=table.to(device),
                           positions=positions.to(device), lengths=list(lengths), page=page)


def attention64(query, key_pages, value_pages, table, positions, mask=None, scale=None):
    """(values, tolerances) in float64, (B, 1, Hq, D)."""
    dtype = query.dtype
    q, table, positions = query.detach().cpu().double(), table.cpu().long(), positions.cpu()
    kp, vp = key_pages.detach().cpu(), value_pages.detach().cpu()
    pages, kv_heads, page, width = kp.shape
    batch, _, q_heads, _ = q.shape
    group = q_heads // kv_heads
    scale = width ** -0.5 if scale is None else scale
    ctx = table.shape[1] * page if mask is None else mask.shape[-1]
    mask = None if mask is None else mask.cpu().expand(batch, 1, 1, ctx)[:, 0, 0]
    out, tol = torch.zeros(batch, 1, q_heads, width, dtype=torch.float64), torch.zeros(batch, 1, q_heads, width, dtype=torch.float64)
    for b in range(batch):
        length = int(positions[b]) + 1 if 0 <= int(positions[b]) < ctx else 0
        j = torch.arange(length)
        at = table[b][j // page]
        keep = (at >= 0) & (at < pages)
        term = torch.zeros(length, dtype=torch.float64)
        if mask is not None:
            row = mask[b, :length]
            keep &= row if row.dtype == torch.bool else row != -math.inf
            if row.dtype != torch.bool:
                term = row.double()
        j, at, term = j[keep], at[keep], term[keep]
        if j.numel() == 0:
            continue
        k, v = kp[at, :, j % page].double(), vp[at, :, j % page].double()  # (keys, heads, width)
        for h in range(kv_heads):
            rows = q[b, 0, h * group:(h + 1) * group]
            s = scale * rows @ k[:, h].T + term
            w = torch.softmax(s, -1)
            out[b, 0, h * group:(h + 1) * group] = w @ v[:, h]
            a = w @ v[:, h].abs()
            size = scale * (rows.abs() @ k[:, h].abs().T).amax(-1, keepdim=True)
            finite = torch.where(s.abs() < 1e30, s.abs(), torch.zeros_like(s)).amax(-1, keepdim=True)
            ds = 2 * (width + 4) * U * size + 4 * U * finite
            split = 0.0 if dtype == torch.float32 else 2.0 ** -21
            tol[b, 0, h * group:(h + 1) * group] = a * (2 * (2 * ds + 16 * U + split) + 4 * (j.numel() / 16 + 64) * U)
    tol += torch.finfo(dtype).eps / 2 * out.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    return out, tol


def assert_within(actual, expected, tol):
    actual = actual.detach().cpu().double()
    assert actual.shape == expected.shape
    assert torch.isfinite(actual).all(), 'not finite'
    over = ((actual - expected).abs() - tol).max().item()
    assert over <= 0, f'off by {over:.3e} more than the bound'


def run(pkg, p, **kwargs):
    return pkg.paged_attention(p.query, p.key_pages, p.value_pages, p.table, p.positions, **kwargs)


def expected(p, **kwargs):
    return attention64(p.query, p.key_pages, p.value_pages, p.table, p.positions, **kwargs)
