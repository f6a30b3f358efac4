"""Steps of ``PagedCache`` over shared pages as a server's batch changes: requests that retire, and the row that they leave."""
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import expected
from tests._talker import Talker
from types import SimpleNamespace

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize('prefix', [16, 4096])
def test_the_first_request_retires(pkg, device, prefix):
    """Its pages are released and its row of the next table is empty.  On either side of where the library reads the prefix once."""
    batch, page = 32, 16
    model = Talker(layers=1, hidden=256, seed=3, dtype=BF16).to(device).eval()
    arena = pkg.PagedArena(model, pages=prefix // page + 2 * batch, page_size=page)
    gen = torch.Generator(device=device).manual_seed(6)
    draw = lambda *shape: torch.randn(*shape, generator=gen, device=device).to(BF16)  # noqa: E731
    shared = arena.allocate(prefix // page)
    prompt = SimpleNamespace(layers=[SimpleNamespace(keys=draw(1, 8, prefix, 128), values=draw(1, 8, prefix, 128))])
    arena.load(arena.page_table([shared]), prompt, torch.tensor([prefix], dtype=torch.int32, device=device))
    owned = [(arena.share(shared) if b else shared) + arena.allocate(2) for b in range(batch)]
    positions = torch.full((batch,), prefix, device=device)
    table = arena.page_table(owned)
    cache = pkg.PagedCache(arena, table, positions, shared_pages=len(shared))
    for step in range(4):
        if step:
            gone = (0, 1, 9)[step - 1]
            arena.release(owned[gone])
            owned[gone] = []
            table.copy_(arena.page_table(owned, width=table.shape[1]))
        query, keys, values = draw(batch, 1, 16, 128), draw(batch, 8, 1, 128), draw(batch, 8, 1, 128)
        out = cache.step(query, keys, values, 0)
        p = SimpleNamespace(query=query, key_pages=arena.keys[0], value_pages=arena.values[0], scales=None, table=table,
                            positions=positions, shared=len(shared), page=page)
        assert_within(out, *expected(p))
        assert all((out[b] == 0).all() for b in range(batch) if not owned[b])
        positions += 1


@pytest.mark.parametrize('once', [True, False])
def test_a_step_reads_as_it_is_told(pkg, device, once):
    """At a size where the library would do the other."""
    prefix, batch = (512, 6) if once else (4096, 32)
    model = Talker(layers=1, hidden=256, seed=3, dtype=BF16).to(device).eval()
    arena = pkg.PagedArena(model, pages=prefix // 16 + batch)
    arena.packed.normal_()
    shared = arena.allocate(prefix // 16)
    table = arena.page_table([shared + arena.allocate(1) for _ in range(batch)])
    positions = torch.full((batch,), prefix + 3, device=device)
    query, rows = torch.randn(batch, 1, 16, 128, device=device).to(BF16), torch.randn(batch, 8, 1, 128, device=device).to(BF16)
    out = pkg.PagedCache(arena, table, positions, len(shared), read_once=once).step(query, rows, rows, 0)
    call = lambda once: pkg.paged_attention(query, arena.keys[0], arena.values[0], table, positions, shared_pages=len(shared),  # noqa: E731
                                            read_once=once)
    assert torch.equal(out, call(once))
    assert torch.equal(call(None), call(not once)) and not torch.equal(out, call(None))
