"""Steps over a cache in pages that find no room."""
import pytest

import pages_ref as ref
from helpers import pkg
from pages_ref import Pool
from test_gpu_pages import DEV, gen, ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_a_step_without_room_leaves_the_dialogs_as_they_were(cache):
    """the step as it is documented, what was kept taken times the reservation's answer: with no page free no code, scale, table,
    count or length changes, though the last block has places left and the new rows are far larger; with one, all are written"""
    g, h, hs, t = gen(1), 2, 64, 9
    pool = Pool(1, 4, h, 64, hs, cache, g)
    tensors = pool.tensors(layers=False)
    table, lens, refs = ints([[3, -1, -1], [0, 2, -1]]), ints([60, 120]), ints([1, 1, 1, 1])
    kn, vn = (100.0 * torch.randn(2, t, h, hs, generator=g).to(DEV) for _ in range(2))
    path = torch.arange(t, dtype=torch.int32, device=DEV).repeat(2, 1)
    kept = ints([5, t])
    state = [*(x.view(torch.int8) if x.element_size() == 1 else x for x in tensors), table, lens, refs]

    def step():
        room = pkg().page_reserve(*tensors, table, refs, lens, kept, max_n=t)
        taken = kept * room[0]
        pkg().page_write(kn, vn, *tensors, table, lens, taken, path, refs)
        lens.add_(taken)
        return room

    before = [x.clone() for x in state]
    assert step().tolist() == [0, 2]
    assert all(torch.equal(a, b) for a, b in zip(before, state))
    table[1, 1], refs[2], lens[1] = -1, 0, 64  # (the second dialog goes back to its first page)
    refs[1] = 0
    assert step().tolist() == [1, 2]
    assert lens.tolist() == [65, 64 + t] and table.tolist() == [[3, 1, -1], [0, 2, -1]]


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_more_blocks_than_a_grids_row_holds(cache):
    """131073 sequences of up to 4096 rows, 8.5 million blocks: of the last one three rows, of all others none"""
    b, t, h, hs = 131073, 4096, 1, 16
    pool = Pool(1, 2, h, 64, hs, cache)
    tensors = pool.tensors(layers=False)
    table = torch.full((b, 64), -1, dtype=torch.int32, device=DEV)
    table[-1, 0] = 1
    pos, n = torch.zeros(2, b, dtype=torch.int32, device=DEV).unbind()
    n[-1] = 3
    rows = torch.randn(2, t, h, hs, generator=gen(3)).to(DEV)
    pkg().page_write(*(x.expand(b, t, h, hs) for x in rows), *tensors, table, pos, n)
    want = Pool(1, 2, h, 64, hs, cache)
    ref.write(want, *(x.cpu()[None, :3] for x in rows), [[1]], [0], [3])
    want.compare(tensors)
    # (sequences four values apart: nothing but the last one's rows is written)
    flat = torch.zeros(2, 4 * b + t * h * hs, device=DEV)
    out = [x.as_strided((b, t, h, hs), (4, h * hs, hs, 1)) for x in flat]
    pkg().page_read(*tensors, table, pos, t, n, out=out)
    got, _, _ = ref.read(want, [[1]], [0], [3], 3)
    assert torch.equal(out[0][-1, :3].cpu().double(), got[0].float().double()) and not flat[0, :4 * (b - 1)].any()
    assert not out[1][-1, 3:].any()
