"""Attention over the 8-bit cache at the edges of what its arguments allow."""
import numpy as np
import pytest
import torch

from tests import kv_ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def positions(w):
    return np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(len(w.lens))])


def missing_pages(be, w, g, dtype, lost, window=0, first=None, **rules):
    """Pages `lost` [(sequence, entry of its table)] are none of the cache's: rows that see a token of one are NaN, the others are what they are with it, bit for bit.
    Some rows of either kind share a tile."""
    from oxinfer_amd import hip
    q = torch.randn(w.rows, w.n_kv * g * w.d, device="cuda").to(dtype)
    cache, batch = w.tensors(hip, ragged=True)
    if first is not None:
        rules["first"] = torch.from_numpy(first).cuda()
    want = be.attend(cache, batch, q, window=window, **rules)
    assert not want.isnan().any()
    pages = batch.pages.clone()
    sees = np.zeros(w.rows, bool)
    pos = positions(w)
    for s, entry in lost:
        pages[s, entry] = w.n_pages
        for r in range(w.start[s], w.start[s + 1]):
            j = np.arange(pos[r] + 1)
            seen = (j > pos[r] - window if window else j >= 0) & (j >= (first[r] if first is not None else 0))
            sees[r] |= (seen & (j // w.page == entry)).any()
    tile = np.concatenate([s * 1000 + np.arange(w.n[s]) * g // 16 for s in range(len(w.lens))])
    assert any(len(set(sees[tile == t])) == 2 for t in set(tile))
    got = be.attend(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), q, window=window, **rules)
    sees = torch.from_numpy(sees).cuda()
    assert got[sees].isnan().all() and torch.equal(got[~sees], want[~sees])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("g", [1, 3])
@pytest.mark.parametrize("rules", [dict(), dict(cap=30.0)], ids=str)
def test_a_missing_page_that_part_of_a_tile_sees(be, g, dtype, rules):
    w = kv_ref.World([34, 61, 90], 2, 64, page=32, seed=3, n=[5, 9, 8])
    missing_pages(be, w, g, dtype, [(0, 1), (2, 2)], **rules)  # (positions 29 .. 33 and 82 .. 89)
    w = kv_ref.World([34, 61, 90], 2, 64, page=32, seed=3, n=[5, 9, 8])
    missing_pages(be, w, g, dtype, [(1, 0)], window=25, **rules)  # (52 .. 60 see from 28 .. 36 on)
    missing_pages(be, w, g, dtype, [(2, 1)], first=np.where(np.arange(w.rows) % 2, 64, 0).astype(np.int32) * (positions(w) >= 64).astype(np.int32), **rules)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rules", [dict(), dict(cap=30.0)], ids=str)
def test_a_missing_page_that_part_of_a_prompts_tile_sees(be, dtype, rules):
    """Rows from position 101 on, four to a wave's tile: one of these holds 157 .. 160."""
    w = kv_ref.World([400, 64], 16, 128, page=32, seed=3, n=[299, 5])
    missing_pages(be, w, 8, dtype, [(0, 5)], window=100, **rules)
