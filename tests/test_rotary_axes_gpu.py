"""``rotary_axes`` against the definition in float64.

Bound, per element, with u = 2^-24: cos and sin are off by what the fraction of a turn loses in
float32 (pi u), by a few units of sincospi (4 u) and, from the float64 angle, by |turns| 2^-52
2 pi; a product and a sum round by u each: |x1| + |x2| times (8 + 3) u + 2 pi |turns| 2^-52, and half a
step of the output, eps/2 |y| (and half the smallest subnormal, for fp16).  ``scaling`` multiplies both
and rounds once more (u)."""
import importlib
import math

import pytest
import torch

from tests._paged import assert_within, attention64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _axis(i, sections, interleaved):
    if interleaved:
        a = i % len(sections)
        return a if i < len(sections) * sections[a] else 0
    for axis, n in enumerate(sections):
        if i < n:
            return axis
        i -= n


def rotated64(x, positions, sections, interleaved=False, theta=1e6, inv_freq=None, scaling=1.0):
    half, x64 = sum(sections), x.detach().cpu().double()
    frequency = (float(theta) ** -(torch.arange(half, dtype=torch.float64) / half)) if inv_freq is None else inv_freq.cpu().double()
    axes = torch.tensor([_axis(i, sections, interleaved) for i in range(half)])
    angle = (positions.cpu().double()[axes].permute(1, 2, 0) * frequency)[:, :, None]
    c, s = angle.cos() * scaling, angle.sin() * scaling
    a, b = x64[..., :half], x64[..., half:2 * half]
    y = torch.cat([a * c - b * s, b * c + a * s, x64[..., 2 * half:]], -1)
    each = (a.abs() + b.abs()) * abs(scaling) * (12 * U + angle.abs() * 2.0 ** -52)
    tol = torch.cat([each, each, torch.zeros_like(x64[..., 2 * half:])], -1)
    rounding = torch.finfo(x.dtype).eps / 2 * (y.abs() + tol) + (2.0 ** -25 if x.dtype == F16 else 0.0)
    rounding[..., 2 * half:] = 0  # copies
    return y, tol + rounding


def _rows(device, batch, tokens, heads, width, dtype, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(batch, tokens, heads, width, generator=gen, device=device).to(dtype)


def _positions(device, axes, batch, tokens, far, seed=1):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, far, (axes, batch, tokens), generator=gen, device=device)


def _check(pkg, q, k, positions, sections, **kwargs):
    got = pkg.rotary_axes(q, k, positions, sections, **kwargs)
    for x, y in zip((q, k), got):
        if x is not None:
            assert y.is_contiguous() and y.dtype == x.dtype
            assert_within(y, *rotated64(x, positions, sections, **kwargs))
    return got


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('width,sections', [(128, (24, 20, 20)), (128, (16, 24, 24)), (64, (8, 12, 12)), (64, (8, 4, 4)),
                                            (128, (64,)), (96, (10, 7)), (20, (1, 0, 2, 3)), (2, (1,)), (130, (33, 32)),
                                            (256, (0, 64, 64)), (100, (5, 5, 5))], ids=str)
def test_types_widths_and_sections(pkg, device, dtype, interleaved, width, sections):
    q, k = _rows(device, 2, 5, 6, width, dtype), _rows(device, 2, 5, 2, width, dtype, seed=2)
    _check(pkg, q, k, _positions(device, len(sections), 2, 5, 900), sections, interleaved=interleaved)


@pytest.mark.parametrize('batch,tokens', [(1, 1), (64, 1), (1, 63), (3, 1000), (2, 2049)])
def test_sizes(pkg, device, batch, tokens):
    q, k = _rows(device, batch, tokens, 16, 128, BF16), _rows(device, batch, tokens, 8, 128, BF16, seed=3)
    _check(pkg, q, k, _positions(device, 3, batch, tokens, 500), (24, 20, 20), interleaved=True)


def test_many_short_rows(pkg, device):
    """More tokens than one workgroup's angles hold, with odd groups at the end."""
    q = _rows(device, 1, 20011, 2, 20, F32)
    _check(pkg, q, None, _positions(device, 2, 1, 20011, 100), (3, 2))


def test_far_and_negative_positions(pkg, device):
    """Angles of millions of turns keep their place on the circle; a negative position turns back."""
    q = _rows(device, 1, 6, 4, 64, F32)
    positions = torch.tensor([1 << 24, (1 << 31) - 1, 1 << 40, -5, -(1 << 33), 0], device=device).view(1, 1, 6)
    _check(pkg, q, None, positions, (32,))
    back, _ = pkg.rotary_axes(pkg.rotary_axes(q, None, positions, (32,))[0], None, -positions, (32,))
    assert (back - q).abs().max() <= 24 * U * 2 * q.abs().max()


def test_frequencies_and_scaling_of_the_callers(pkg, device):
    q, k = _rows(device, 2, 7, 4, 128, BF16), _rows(device, 2, 7, 4, 128, BF16, seed=4)
    positions = _positions(device, 3, 2, 7, 3000)
    _check(pkg, q, k, positions, (24, 20, 20), theta=1e4, scaling=1.3)
    for dtype in (F32, torch.float64):
        inv = (torch.rand(64, device=device, dtype=dtype) + 0.01)
        _check(pkg, q, k, positions, (24, 20, 20), inv_freq=inv)


def test_equal_axes_are_plain_rotary(pkg, device):
    """With one position on all axes the sections do not matter, and float32 rows agree with ``rotary`` on
    its tables up to the tables' float32 angles."""
    q = _rows(device, 2, 9, 4, 128, F32)
    positions = torch.randint(0, 64, (1, 2, 9), device=device).expand(3, 2, 9)
    got, _ = pkg.rotary_axes(q, None, positions, (24, 20, 20))
    for interleaved in (False, True):
        assert torch.equal(pkg.rotary_axes(q, None, positions, (64, 0, 0), interleaved=interleaved)[0], got)
    cos, sin = pkg.rope_tables(positions[0].contiguous(), 128, dtype=F32)
    assert (pkg.rotary(q, cos, sin) - got).abs().max() <= 64 * 2 * U * 2 * q.abs().max() + 16 * U * q.abs().max()


def test_strides_and_views(pkg, device):
    fused = _rows(device, 3, 5, 28, 128, BF16)
    q, k = fused[:, :, :16], fused[:, :, 16:24]
    positions = _positions(device, 3, 3, 5, 700)
    want = _check(pkg, q, k, positions, (24, 20, 20))
    # heads first in memory; positions with their axes last; elements that only fit one by one
    bnsd = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]
    axes_last = positions.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device=device)[1:].view(q.shape).copy_(q)
    for a, b, p in ((*bnsd, positions), (q, k, axes_last), (odd, k, positions)):
        got = pkg.rotary_axes(a, b, p, (24, 20, 20))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    shared = q[:, :, :1].expand(3, 5, 16, 128)
    got, _ = pkg.rotary_axes(shared, None, positions, (24, 20, 20))
    assert torch.equal(got, pkg.rotary_axes(shared.contiguous(), None, positions, (24, 20, 20))[0])


@pytest.mark.parametrize('sections', [(24, 20, 20), (8, 4, 4)], ids=str)
def test_in_place(pkg, device, sections):
    """The given rows are rotated where they are, and nothing else of their tensor changes."""
    fused = _rows(device, 3, 5, 28, 128, BF16)
    positions = _positions(device, 3, 3, 5, 700)
    want = pkg.rotary_axes(fused[:, :, :16], fused[:, :, 16:24], positions, sections)
    rest = fused[:, :, 24:].clone()
    q, k = fused[:, :, :16], fused[:, :, 16:24]
    got = pkg.rotary_axes(q, k, positions, sections, inplace=True)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, :, 24:], rest)
    with pytest.raises(ValueError):
        pkg.rotary_axes(q[:, :, :1].expand(3, 5, 16, 128), k, positions, sections, inplace=True)


@pytest.mark.parametrize('views', [lambda f: (f[:, :, :16], f[:, :, 8:16]), lambda f: (f, f), lambda f: (f[:, :, :16], f[:, :, 15:20]),
                                   lambda f: (f[:, :, :1].expand(3, 5, 16, 128), None)], ids=['part', 'same', 'one row', 'expanded'])
def test_in_place_refuses_rows_that_overlap(pkg, device, views):
    fused = _rows(device, 3, 5, 28, 128, BF16)
    before = fused.clone()
    q, k = views(fused)
    positions = _positions(device, 3, 3, 5, 700)
    with pytest.raises(ValueError):
        pkg.rotary_axes(q, k, positions, (24, 20, 20), inplace=True)
    assert torch.equal(fused, before)
    got = pkg.rotary_axes(q, k, positions, (24, 20, 20))  # (fresh outputs: any views are fine)
    assert torch.equal(got[0], pkg.rotary_axes(q.contiguous(), None, positions, (24, 20, 20))[0])


def test_no_rows(pkg, device):
    q = torch.empty(0, 5, 4, 128, device=device)
    got, none = pkg.rotary_axes(q, None, torch.empty(3, 0, 5, dtype=torch.int64, device=device), (24, 20, 20))
    assert got.shape == q.shape and none is None


def test_special_values(pkg, device):
    """Infinities and NaN stay in their pairs of elements."""
    q = _rows(device, 1, 2, 2, 64, BF16)
    positions = _positions(device, 1, 1, 2, 50) + 1
    want, tol = rotated64(q, positions, (32,))
    q[0, 0, 1, 5], q[0, 1, 0, 40] = math.inf, math.nan
    got = pkg.rotary_axes(q, None, positions, (32,))[0].cpu().double()
    bad = torch.zeros(got.shape, dtype=torch.bool)
    bad[0, 0, 1, [5, 37]] = bad[0, 1, 0, [8, 40]] = True
    assert not torch.isfinite(got[bad]).any() and torch.isnan(got[0, 1, 0, [8, 40]]).all()
    got[bad], want[bad] = 0, 0
    assert_within(got, want, tol)


def test_captured_call_follows_its_positions(pkg, device):
    q, k = _rows(device, 4, 1, 16, 128, BF16), _rows(device, 4, 1, 8, 128, BF16, seed=5)
    positions = _positions(device, 3, 4, 1, 100)
    pkg.rotary_axes(q, k, positions, (24, 20, 20))  # the frequencies' copy is made outside the capture
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out = pkg.rotary_axes(q, k, positions, (24, 20, 20))
    for step in range(4):
        positions.add_(step * 1000)
        q.mul_(1.1)
        want = pkg.rotary_axes(q, k, positions, (24, 20, 20))
        graph.replay()
        torch.cuda.synchronize(device)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_first_call_of_a_theta_under_capture(pkg, device):
    """A graph forms the frequencies of a theta that no call has had, and leaves nothing for later calls."""
    q = _rows(device, 4, 1, 16, 128, BF16)
    positions = _positions(device, 3, 4, 1, 100)
    table = importlib.import_module(pkg.__name__ + '.rotary')._TURNS
    kept = dict(table)
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph):
        out, _ = pkg.rotary_axes(q, None, positions, (24, 20, 20), theta=54321.5)
    assert table.keys() == kept.keys()
    for step in range(4):
        positions.add_(step * 1000)
        graph.replay()
        torch.cuda.synchronize(device)
        assert_within(out.cpu().double(), *rotated64(q, positions, (24, 20, 20), theta=54321.5))
        _check(pkg, q, q, positions, (24, 20, 20), theta=54321.5)
    for theta in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            pkg.rotary_axes(q, None, positions, (24, 20, 20), theta=theta)


def test_a_layers_step(pkg, device):
    """The three operators as a layer runs them: rotated rows into the pages, then attention over
    what the pages hold, three steps in a row."""
    page, batch, sections = 16, 3, (24, 20, 20)
    pools = [torch.full((12, 8, page, 128), math.nan, dtype=BF16, device=device) for _ in range(2)]
    table = torch.randperm(12, generator=torch.Generator().manual_seed(6))[:9].view(3, 3).to(torch.int32).to(device)
    lengths = torch.tensor([14, 31, 0], device=device)
    start = _rows(device, batch, 32, 16, 128, BF16, seed=7)
    pkg.paged_write(start[:, :, :8].transpose(1, 2), start[:, :, 8:].transpose(1, 2), *pools, table,
                    torch.zeros(3, dtype=torch.int64, device=device), lengths.int())
    for step in range(3):
        fused = _rows(device, batch, 1, 32, 128, BF16, seed=8 + step)
        q, k, v = fused[:, :, :16], fused[:, :, 16:24], fused[:, :, 24:]
        at = torch.stack([lengths, lengths // 4, lengths // 7])[..., None]
        q, k = _check(pkg, q, k, at, sections, interleaved=True)
        pkg.paged_write(k.transpose(1, 2), v.transpose(1, 2), *pools, table, lengths)
        for b in range(batch):
            j = int(lengths[b])
            for pool, rows in zip(pools, (k, v)):
                assert torch.equal(pool[int(table[b, j // page]), :, j % page], rows[b, 0])
        out = pkg.paged_attention(q, *pools, table, lengths)
        assert_within(out, *attention64(q, *pools, table, lengths))
        lengths += 1
