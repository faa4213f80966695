"""Attention over the 8-bit cache at the edges of what its arguments allow."""
import numpy as np
import pytest
import torch

from tests import kv_ref
from tests.test_gpu_attend import check

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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [0.0, 1e-42, 1e-25])
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("n,n_kv,d,g", [([1, 1], 2, 64, 3), ([5, 40], 2, 64, 3), ([299, 5], 16, 128, 8)], ids=["one", "few", "prompt"])
def test_scales_of_zero(be, n, n_kv, d, g, which, value, dtype):
    """Blocks whose scale is 0, or under the least one, which counts as 0: their keys score 0, their values are 0. Blocks of the first tokens, and the last, of
    which rows see a part."""
    w = kv_ref.World([90, 301] if d == 64 else [400, 64], n_kv, d, page=32, seed=5, n=n)
    for s in range(2):
        for b in (0, (w.lens[s] - 1) // 32):
            if which != "v":
                w.ks[w.table[s, b], :, 0] = value
            if which != "k":
                w.vs[w.table[s, b], :, 0] = value
    heads = None if d == 64 else [0, 60, 127]
    sequence = w.sequence
    w.sequence = lambda s: [x * (np.repeat(scales[w.table[s, : -(-w.lens[s] // 32)], :, 0], 32, 0)[: w.lens[s]] >= 2.0**-60)[..., None] for x, scales in zip(sequence(s), (w.ks, w.vs))]
    check(be, w, g, dtype, ragged=True, heads=heads)
    check(be, w, g, dtype, ragged=True, heads=heads, cap=20.0, window=70)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_new_cache_holds_zeros(be, dtype):
    from oxinfer_amd import hip
    cache = be.kv_cache(4, 2, 64)
    batch = hip.KvBatch(torch.tensor([130, 7], dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda").repeat(2, 1))
    assert (be.attend(cache, batch, torch.randn(2, 4 * 64, device="cuda").to(dtype)) == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q,scale,k", [(-90, 90, 0), (-90, 37, 53), (-140, 117, 23), (-70, 10, 60), (-64, 4, 60), (-100, 40, 60), (100, -50, -50), (50, 2, -52), (110, -110, 0), (120, -120, 0)])
@pytest.mark.parametrize("n,n_kv,d,g", [([5, 40], 2, 64, 3), ([299, 5], 16, 128, 8)], ids=["few", "prompt"])
def test_rows_scales_and_keys_of_any_size(be, n, n_kv, d, g, q, scale, k, dtype):
    """Powers of two on the rows, the scale and the keys whose product is 1."""
    w = kv_ref.World([90, 301] if d == 64 else [400, 64], n_kv, d, page=32, seed=5, n=n)
    w.ks *= np.float32(2.0**k)
    check(be, w, g, dtype, ragged=True, heads=None if d == 64 else [0, 60, 127], loud=2.0 ** (q + 1), scale=2.0 ** (scale - 3))


def one_key(be, w, g, dtype, scale, slopes=None, heads=None, loud=2.0, cached=None):
    """Scores so far apart that a row's softmax is its best key's alone, by a margin past all errors of f32 scores: the results are that key's values.
    A weight's error: the rounding to f16 (2^-11, or 2^-21 in two), and what the logarithm and exponentials of the value scale leave, 16 u of 84."""
    from oxinfer_amd import hip
    rng = np.random.default_rng(11)
    n_q = w.n_kv * g
    cache, batch = w.tensors(hip, ragged=True)
    q = torch.from_numpy(loud * rng.normal(size=(w.rows, n_q * w.d))).to("cuda", dtype)
    up = None if slopes is None else torch.from_numpy(np.asarray(slopes, np.float32)).cuda()
    got = be.attend(cache, batch, q, scale=scale, slopes=up).double().cpu().numpy().reshape(w.rows, n_q, w.d)
    hq, pos = q.double().cpu().numpy().reshape(w.rows, n_q, w.d), positions(w)
    half = dtype == torch.bfloat16
    rel = (2.0**-11 if half else 2.0**-21) + 2 * 8 * 84 * 2.0**-24 + (2.0**-8 if half else 2.0**-24)
    checked = 0
    for s in range(len(w.lens)):
        k, v = w.sequence(s)
        for r in range(w.start[s], w.start[s + 1]):
            for h in range(n_q) if heads is None else heads:
                j = np.arange(pos[r] + 1)
                score = scale * (k[j, h // g] @ hq[r, h])
                mass = abs(scale) * (np.abs(k[j, h // g]) @ np.abs(hq[r, h])).max()
                if slopes is not None:
                    bias = float(np.float32(slopes[h])) * (pos[r] - j)
                    score, mass = score - bias, mass + bias.max()
                best = np.argsort(score)[-2:]
                if len(best) == 2 and score[best[1]] - score[best[0]] < 2.0**-16 * mass + 100:
                    continue
                checked += 1
                want = v[best[-1], h // g]
                assert (np.abs(got[r, h] - want) <= rel * np.abs(want)).all(), (r, h)
    assert checked >= w.rows * (n_q if heads is None else len(heads)) // 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0**14, 2.0**19, 2.0**22, -(2.0**22), 2.0**30, 2.0**39, 2.0**60, -(2.0**100)])
@pytest.mark.parametrize("n,n_kv,d,g", [([1, 1], 2, 64, 3), ([5, 40], 2, 64, 3), ([299, 5], 16, 128, 8)], ids=["one", "few", "prompt"])
def test_scores_far_from_zero(be, n, n_kv, d, g, scale, dtype):
    w = kv_ref.World([90, 301] if d == 64 else [400, 64], n_kv, d, page=32, seed=5, n=n)
    one_key(be, w, g, dtype, scale, heads=None if d == 64 else [0, 60, 127])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("slope", [1e3, 1e7, 1e9, 1e20, 1e35])
@pytest.mark.parametrize("n,n_kv,d,g", [([1, 1], 2, 64, 3), ([5, 40], 2, 64, 3), ([299, 5], 16, 128, 8)], ids=["one", "few", "prompt"])
def test_steep_slopes(be, n, n_kv, d, g, slope, dtype):
    """A row's own key is what is left."""
    w = kv_ref.World([90, 301] if d == 64 else [400, 64], n_kv, d, page=32, seed=5, n=n)
    one_key(be, w, g, dtype, d**-0.5, slopes=np.full(n_kv * g, slope), heads=None if d == 64 else [0, 60, 127])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0**22, 2.0**39, -(2.0**60)])
def test_scores_far_from_zero_in_parts_that_meet(be, scale, dtype):
    """Sequences whose blocks several workgroups share."""
    one_key(be, kv_ref.World([9000, 4500], 2, 64, page=64, seed=5), 3, dtype, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("slope", [1e7, 1e30])
def test_steep_slopes_in_parts_that_meet(be, slope, dtype):
    w = kv_ref.World([9000, 4500], 2, 64, page=64, seed=5)
    one_key(be, w, 3, dtype, 0.125, slopes=np.full(6, slope))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales_of_zero_in_parts_that_meet(be, dtype):
    """Most blocks of one sequence, and all of the other, hold zeros."""
    w = kv_ref.World([9000, 4500], 2, 64, page=64, seed=5)
    at = np.concatenate([w.table[0, 3:140], w.table[1, : -(-4500 // 64)]])
    w.vs[at] = 0.0
    w.ks[at[::2]] = 0.0
    check(be, w, 3, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,n_kv", [([5, 3], 2), ([300, 5], 16)], ids=["few", "prompt"])
@pytest.mark.parametrize("factor", [2.0**20, 2.0**40, 2.0**-40, 0.0])
def test_a_rows_bits_beside_rows_of_another_size(be, n, n_kv, factor, dtype):
    """Rows whose scores are far from zero, or all alike, leave the rows of their tile as they are; blocks without values among them."""
    from oxinfer_amd import hip
    w = kv_ref.World([900, 64], n_kv, 128, page=32, seed=3, n=n)
    w.vs[w.table[0, 7]] = 0.0
    cache, batch = w.tensors(hip)
    q = torch.randn(w.rows, n_kv * 8 * 128, device="cuda").to(dtype)
    for rules in (dict(), dict(cap=1e12)):
        want = be.attend(cache, batch, q, **rules)
        for part in (slice(0, None, 3), slice(1, None, 2)):
            other = q.clone()
            other[part] *= factor
            kept = torch.ones(w.rows, dtype=torch.bool)
            kept[part] = False
            got = be.attend(cache, batch, other, **rules)
            assert torch.equal(got[kept], want[kept]) and got.isfinite().all() and not torch.equal(got, want)
