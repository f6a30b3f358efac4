"""Steps of ``PackedAttention`` over arenas of 8 bits and over requests that share their first pages: admission, steps, growth,
retirement and the way back to a slot, as a server runs them."""
import math

import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import HELD, bits, expected, quantised
from tests._talker import Talker
from tests._util import assert_attention_close, f64
from types import SimpleNamespace

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _model(pkg, device, dtype=BF16, layers=2):
    model = Talker(layers=layers, hidden=256, seed=3, dtype=dtype).to(device).eval()
    pkg.install_packed_attention(model, native_gqa=True, text_only_rope=True, triton_talker_rope=True)
    return model


def _step(model, cache, hidden, positions, mask=None):
    tables = model.rotary_emb(hidden, positions.expand(3, -1)[..., None])
    for layer in model.layers:
        hidden = layer(hidden, attention_mask=mask, past_key_values=cache, position_embeddings=tables)[0]
    return model.norm(hidden)


def _prefill(planes):
    """A prefill cache of (2 * layers, B, kv_heads, length, head_dim) planes."""
    layers = planes.shape[0] // 2
    return SimpleNamespace(layers=[SimpleNamespace(keys=planes[i], values=planes[layers + i]) for i in range(layers)])


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_steps_over_8_bits_and_back_to_a_slot(pkg, device, held, dtype):
    model = _model(pkg, device, dtype)
    lengths = [30, 47, 1, 16]
    gen = torch.Generator(device=device).manual_seed(4)
    prompt = torch.randn(4, 4, 8, 47, 128, generator=gen, device=device).to(dtype)
    arena = pkg.PagedArena(model, pages=24, page_size=16, dtype=held)
    arena.packed_scales.fill_(math.nan)
    owned = [arena.allocate(arena.pages_for(n)) for n in lengths]
    table = arena.page_table(owned, width=6)
    arena.load(table, _prefill(prompt), torch.tensor(lengths, dtype=torch.int32, device=device))
    positions = torch.tensor(lengths, device=device)
    cache = pkg.PagedCache(arena, table, positions)
    attention, seen, queries = model.layers[0].self_attn, [], []
    attention.reference.o_proj.register_forward_hook(lambda m, args, out: seen.append(args[0]))
    attention.reference.q_norm.register_forward_hook(lambda m, args, out: queries.append(out))
    with torch.inference_mode():
        for step in range(6):
            for b in range(4):
                if int(positions[b]) == len(owned[b]) * 16:
                    owned[b] += arena.allocate(1)
            table.copy_(arena.page_table(owned, width=6))
            hidden = torch.randn(4, 1, 256, generator=gen, device=device).to(dtype)
            _step(model, cache, hidden, positions)
            cos, sin = model.rotary_emb(hidden, positions[None, :, None])
            query = pkg.rotary(queries[-1].contiguous(), cos[0].contiguous(), sin[0].contiguous())
            p = SimpleNamespace(query=query, key_pages=arena.keys[0], value_pages=arena.values[0], scales=arena.scales[0],
                                table=table, positions=positions, shared=0, page=16)
            assert_within(seen[-1].view(4, 1, 16, 128), *expected(p))
            positions += 1
        # every prompt's rows came back from their pages as the definition has them
        back = arena.read(table, 47, torch.tensor(lengths, dtype=torch.int32, device=device))
        elements, scales = quantised(prompt, held)
        want = (elements.float() * scales[..., None]).to(dtype)
        for b, n in enumerate(lengths):
            assert torch.equal(bits(back[:, b, :, :n]), bits(want[:, b, :, :n])) and (back[:, b, :, n:] == 0).all()
        slots = pkg.SlotArena(model, 4, 96, packed_kv=True)
        slots.load_packed(2, back, row=1, length=47)
        assert torch.equal(bits(slots.packed[:, 2, :, :47]), bits(back[:, 1]))


@pytest.mark.parametrize('held', [None, *HELD], ids=str)
@pytest.mark.parametrize('once', [None, True])
def test_requests_that_share_their_prompt(pkg, device, held, once, monkeypatch):
    """Answers to one prompt of 70 rows: whole pages shared, the rest of it each request's own.  Their steps are those of requests
    that have all rows for themselves; the pages are free once the last request is gone."""
    import importlib
    if once:  # (short prompts are attended request by request otherwise)
        paged = importlib.import_module(pkg.__name__ + '.paged')
        whole = paged._attention_call
        monkeypatch.setattr(paged, '_attention_call', lambda *args: whole(*args, True))
    model = _model(pkg, device)
    batch, rows, page = 5, 70, 16
    gen = torch.Generator(device=device).manual_seed(5)
    prompt = torch.randn(4, 1, 8, rows, 128, generator=gen, device=device).to(BF16)
    arenas = [pkg.PagedArena(model, pages=60, page_size=page, dtype=held) for _ in range(2)]
    shared = rows // page
    first = arenas[0].allocate(shared)
    full = torch.tensor([shared * page], dtype=torch.int32, device=device)
    arenas[0].load(arenas[0].page_table([first]), _prefill(prompt), full)
    owned = [(arenas[0].share(first) if b else first) + arenas[0].allocate(2) for b in range(batch)]
    table = arenas[0].page_table(owned, width=8)
    rest = torch.full((batch,), rows - shared * page, dtype=torch.int32, device=device)
    arenas[0].load(table, _prefill(prompt[..., shared * page:, :].expand(4, batch, 8, -1, 128)), rest,
                   torch.full((batch,), shared * page, device=device))
    twins = [arenas[1].allocate(shared + 2) for _ in range(batch)]
    twin_table = arenas[1].page_table(twins, width=8)
    arenas[1].load(twin_table, _prefill(prompt.expand(4, batch, 8, rows, 128)), torch.full((batch,), rows, dtype=torch.int32, device=device))
    positions = torch.full((batch,), rows, device=device)
    caches = pkg.PagedCache(arenas[0], table, positions, shared_pages=shared), pkg.PagedCache(arenas[1], twin_table, positions)
    before = arenas[0].packed[:, first].view(torch.uint8).clone()
    with torch.inference_mode():
        for step in range(12):
            hidden = torch.randn(batch, 1, 256, generator=gen, device=device).to(BF16)
            out, want = (_step(model, cache, hidden, positions) for cache in caches)
            assert_attention_close(f64(out), f64(want), max_abs=2 * 3e-2, mean_abs=2 * 3e-3)
            at = rows + step  # layer 0 sees the same rows on both sides
            for b in range(batch):
                for plane in (0, 2):
                    new, twin = (bits(a.packed[plane, o[b][at // page], :, at % page]) for a, o in zip(arenas, (owned, twins)))
                    assert torch.equal(new, twin)
            positions += 1
    assert torch.equal(arenas[0].packed[:, first].view(torch.uint8), before)
    for b in range(batch):
        assert arenas[0].free_pages == 60 - shared - 2 * (batch - b)
        arenas[0].release(owned[b])
    assert arenas[0].free_pages == 60


@pytest.mark.parametrize('held', [None, HELD[0]], ids=str)
def test_captured_step_of_a_padded_batch(pkg, device, held):
    """Captured with no positions, replayed as requests take their places, against the eager step on a twin arena."""
    model = _model(pkg, device)
    arenas = [pkg.PagedArena(model, pages=40, page_size=16, dtype=held) for _ in range(2)]
    shared = arenas[0].allocate(20)
    prompt = torch.randn(4, 1, 8, 320, 128, device=device).to(BF16)
    for arena in arenas:
        arena.load(arena.page_table([shared]), _prefill(prompt), torch.tensor([320], dtype=torch.int32, device=device))
    table = arenas[0].page_table([shared + arenas[0].allocate(2) for _ in range(6)])
    positions = torch.full((6,), -1, device=device)
    caches = [pkg.PagedCache(arena, table, positions, shared_pages=20) for arena in arenas]
    hidden = torch.zeros(6, 1, 256, device=device, dtype=BF16)
    with torch.inference_mode():
        _step(model, caches[0], hidden, positions)
        torch.cuda.synchronize(device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(model, caches[0], hidden, positions)
        torch.cuda.synchronize(device)
        for step in range(6):
            positions[step] = 320 + 3 * step
            hidden.normal_()
            graph.replay()
            want = _step(model, caches[1], hidden, positions)
            torch.cuda.synchronize(device)
            assert torch.equal(out, want)
            assert torch.equal(bits(arenas[0].packed), bits(arenas[1].packed))
            positions[positions >= 0] += 1


@pytest.mark.parametrize('held', HELD, ids=str)
def test_pools_past_four_gigabytes(pkg, device, held):
    pages = (1 << 32) // (8 * 16 * 128) + 16
    pool = torch.empty(2, pages, 8, 16, 128, dtype=torch.uint8, device=device)
    pool[:, -3:] = 0
    scales = torch.zeros(2, pages, 8, 16, device=device)
    rows = [torch.randn(1, 8, 20, 128, device=device).to(BF16) for _ in range(2)]
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=device)
    start = torch.tensor([1], device=device)
    pools, pair = pool.view(held).unbind(0), tuple(scales.unbind(0))
    pkg.paged_write(*rows, *pools, table, start, scales=pair)
    back = pkg.paged_read(*pools, table, start, 20, scales=pair, dtype=F32)
    for x, got, plane in zip(rows, back, pool):
        elements, own = quantised(x, held)
        assert torch.equal(got.cpu(), elements.float() * own[..., None])
        assert (plane[-2] == 0).all() and (plane[-3, :, 5:] == 0).all() and (plane[-1, :, 0] == 0).all()
    query = torch.randn(1, 1, 16, 128, device=device).to(BF16)
    near = SimpleNamespace(query=query, key_pages=pools[0][-3:], value_pages=pools[1][-3:], table=torch.tensor([[2, 0]], dtype=torch.int32),
                           scales=tuple(x[-3:] for x in pair), positions=torch.tensor([20]), shared=0, page=16)
    out = pkg.paged_attention(query, *pools, table, torch.tensor([20], device=device), scales=pair)
    assert_within(out, *expected(near))
