"""Attention of a batch whose sequences begin with the same tokens, against the same in 64 bits (kv_ref over the tokens that each sequence then has)."""
import threading

import numpy as np
import pytest
import torch

from tests import kv_ref
from tests.lists_ref import Shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def handles(w, hip, ragged=None, extra=0):
    cache, batch = w.tensors(hip, ragged=ragged, extra_rows=extra)
    return cache, batch, hip.KvShared(torch.from_numpy(w.group_start).cuda(), torch.from_numpy(w.common).cuda())


def positions(w):
    return np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(len(w.lens))])


def check(be, w, g, dtype="f32", scale=None, seed=5, strided=False, odd=False, ragged=None, loud=2.0, **rules):
    from oxinfer_amd import hip
    rng = np.random.default_rng(seed)
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n_q = w.n_kv * g
    ragged = (w.n != 1).any() if ragged is None else ragged
    extra = 3 if ragged else 0
    width = n_q * w.d
    cache, batch, shared = handles(w, hip, ragged, extra)
    stride = width + (8 if strided else 0) + (1 if odd else 0)
    q = torch.from_numpy(loud * rng.normal(size=(w.rows + extra, stride))).to("cuda", tt)
    flat = torch.full(((w.rows + extra) * stride + 1,), 7.5, dtype=tt, device="cuda")
    out = flat[1 if odd else 0 :][: (w.rows + extra) * stride].view(w.rows + extra, stride)
    scale = w.d**-0.5 if scale is None else scale
    up = {k: torch.from_numpy(np.ascontiguousarray(v)).to("cuda") if isinstance(v, np.ndarray) else v for k, v in rules.items()}
    if "first" in up:
        up["first"] = torch.cat([up["first"], torch.zeros(extra, dtype=torch.int32, device="cuda")])
    be.attend_shared(cache, batch, shared, q[:, :width], scale=scale, out=out[:, :width], **up)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want, tol = kv_ref.attend(w, q[: w.rows, :width].double().cpu().numpy().reshape(w.rows, n_q, w.d), g, scale, half=dtype == "bf16", **rules)
    assert (got[w.rows :] == 7.5).all() and (got[:, width:] == 7.5).all(), "what is not the call's was written"
    off = np.abs(got[: w.rows, :width].reshape(want.shape) - want)
    assert (off <= tol).all(), f"{np.max(off / np.maximum(tol, 1e-300)):.2f} times the bound"
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_head_sizes(be, d, dtype):
    check(be, Shared([397, 365, 401], [0, 3], [360], 2, d, page=64, seed=d), 4, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [1, 2, 3, 5, 8, 9, 15, 16, 17, 33])
def test_groups_of_heads(be, g, dtype):
    check(be, Shared([70, 73, 200, 90, 71], [0, 5], [67], 3, 64, page=32, seed=g), g, dtype)
    check(be, Shared([70, 73, 200, 90, 71], [0, 2, 4], [60, 85], 1, 64, page=32, seed=g, n=[2, 5, 3, 0, 4]), g, dtype)


@pytest.mark.parametrize("common", [0, 1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1023, 2049, 4097])
@pytest.mark.parametrize("page", [32, 256])
def test_lengths_of_the_prefix(be, common, page):
    """Prefixes that end inside blocks and pages, or at their ends; sequences that end with the prefix, one token behind it, or a little further."""
    check(be, Shared([common + 1, common + 40, max(common, 1), common + 2, common + 65], [0, 5], [common], 2, 128, page=page, seed=common), 4)


def test_a_long_prefix(be):
    check(be, Shared([70001, 70300, 70010], [0, 3], [69999], 1, 64, page=128, seed=3), 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_several_groups(be, dtype):
    """Tiles that hold rows of several groups, groups of one sequence, groups that share nothing, sequences before and behind all groups."""
    lens = [50, 130, 140, 90, 95, 99, 300, 64, 31, 200, 70]
    for start, common in (([1, 3, 6, 7, 8], [100, 33, 250, 0]), ([0, 11], [31]), ([2, 2, 5, 5, 9], [7, 70, 3, 20]), ([0, 1, 2, 3], [5, 6, 7]), ([11, 11], [40]), ([20, 25], [40])):
        check(be, Shared(lens, start, common, 2, 64, page=32, seed=4), 3, dtype)
        check(be, Shared(lens, start, common, 1, 96, page=64, seed=4, n=[1, 3, 0, 2, 7, 1, 1, 5, 2, 1, 4]), 2, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,lens,common", [([5, 2], [40, 39], 37), ([17, 0, 3], [40, 90, 300], 20), ([70, 1, 33], [100, 60, 100], 45), ([0, 0, 4], [7, 3, 4], 2), ([30, 30, 30], [30, 30, 30], 20), ([130, 64], [400, 410], 390)])
def test_rows_of_ragged_sequences(be, n, lens, common, dtype):
    """Also rows that lie inside the shared tokens themselves."""
    for g, d in ((1, 64), (4, 128), (3, 96), (20, 32)):
        check(be, Shared(lens, [0, len(lens)], [common], 2, d, page=64, seed=sum(n), n=n), g, dtype, ragged=True)


def test_more_rows_than_tokens(be):
    got = check(be, Shared([40, 3, 0], [0, 3], [2], 2, 64, seed=1, n=[4, 7, 2]), 2, ragged=True)
    assert (got[4:8, :256] == 0).all() and (got[11:13, :256] == 0).all()


@pytest.mark.parametrize("n_seqs", [1, 63, 64, 65, 200])
def test_many_sequences(be, n_seqs):
    """Also long runs of sequences without rows between those that share a tile."""
    rng = np.random.default_rng(n_seqs)
    n = rng.integers(0, 4, n_seqs)
    n[n_seqs // 4 : n_seqs // 4 * 3] = 0
    n[-1] = 2
    start = np.unique(rng.integers(0, n_seqs + 1, 5))
    if len(start) < 2:
        start = np.array([0, n_seqs])
    check(be, Shared(n + 40 + rng.integers(0, 90, n_seqs), start, rng.integers(0, 40, len(start) - 1), 1, 64, seed=n_seqs, n=n), 5, ragged=True)
    check(be, Shared(41 + rng.integers(0, 90, n_seqs), start, rng.integers(0, 40, len(start) - 1), 1, 64, seed=n_seqs), 3)


RULES = [dict(window=1), dict(window=33), dict(window=100), dict(window=10**6), dict(cap=5.0), dict(slopes=True), dict(prefix=[20, 0, 700, 80, 3]), dict(prefix=[-3, 64, 33, 100, 101]), dict(window=20, prefix=[10, 130, 4, 0, 110]),
         dict(first="docs"), dict(first="none"), dict(window=40, cap=30.0, slopes=True, prefix=[5, 100, 0, 64, 7], first="docs")]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rules", RULES, ids=str)
@pytest.mark.parametrize("n", [[1, 1, 1, 1, 1], [3, 70, 35, 0, 6]], ids=["one", "many"])
def test_masks_caps_and_biases(be, rules, n, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    w = Shared([190, 150, 300, 110, 170], [0, 3, 5], [101, 75], 2, 64, page=32, seed=9, n=n)
    g = 3
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-np.arange(1, 7)).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.array(rules["prefix"], np.int32)
    pos = positions(w)
    if rules.get("first") == "docs":
        rules["first"] = (pos * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    elif rules.get("first") == "none":  # every other row sees nothing at all
        rules["first"] = np.where(np.arange(w.rows) % 2, 0, np.where(np.arange(w.rows) % 4, pos + 1, 2**31 - 1)).astype(np.int32)
    check(be, w, g, dtype, loud=4.0, **rules)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 4.0])
def test_scales(be, scale):
    check(be, Shared([100, 137], [0, 2], [90], 2, 64, seed=2), 4, scale=scale, window=30)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_addresses(be, dtype):
    for n in ([1, 1], [20, 3]):
        w = Shared([85, 100], [0, 2], [50], 2, 96, seed=3, n=n)
        check(be, w, 2, dtype, strided=True)
        check(be, w, 2, dtype, strided=True, odd=True)


@pytest.mark.parametrize("n", [[1, 1, 1], [5, 9, 2]])
def test_scales_of_zero_and_values_far_apart(be, n):
    """A cache holds scales of zero, and scales at either end, in shared blocks as in own ones."""
    w = Shared([150, 170, 180], [0, 3], [90], 2, 64, page=32, seed=6, n=n)
    for s, page, value in ((0, 0, 0.0), (0, 1, 2.0**60), (0, 2, 2.0**-60), (1, 3, 0.0), (1, 4, 2.0**59), (2, 3, 2.0**-60)):
        w.vs[w.table[s, page]] = value
    w.ks[w.table[0, 1]] = w.ks[w.table[2, 4]] = 0.0
    check(be, w, 3)


@pytest.mark.parametrize("n,n_kv,d,g", [([5, 9], 2, 64, 3), ([299, 5], 16, 128, 8)], ids=["few", "prompt"])
def test_values_of_zero_before_huge_ones(be, n, n_kv, d, g):
    """Of `attend` as well: weights of blocks whose scale is 0, or the least, count for the sum although blocks of the largest scale come behind them."""
    from oxinfer_amd import hip
    w = kv_ref.World([400, 330], n_kv, d, page=32, seed=6, n=n)
    w.vs[w.table[:, :3]] = 0.0
    w.vs[w.table[:, 3:5]] = 2.0**-60
    w.vs[w.table[:, 5]] = 2.0**60
    cache, batch = w.tensors(hip, ragged=True)
    q = 2 * torch.randn(w.rows, n_kv * g * d, device="cuda")
    heads = None if d == 64 else [0, 60, 127]
    want, tol = kv_ref.attend(w, q.double().cpu().numpy().reshape(w.rows, n_kv * g, d), g, d**-0.5, heads=heads)
    off = np.abs(be.attend(cache, batch, q).double().cpu().numpy().reshape(want.shape) - want)
    off, tol = (off, tol) if heads is None else (off[:, heads], tol[:, heads])
    assert (off <= tol).all(), f"{np.max(off / np.maximum(tol, 1e-300)):.2f} times the bound"


def test_pages_outside_the_cache(be):
    """Rows that would see a token of such a page are NaN, the others of their tile what they are."""
    from oxinfer_amd import hip
    for n in ([1, 1, 1, 1], [5, 3, 2, 6]):
        w = Shared([140, 100, 150, 130], [0, 3, 4], [97, 20], 2, 64, page=32, seed=3, n=n)
        q = torch.randn(w.rows, 4 * 64, device="cuda")
        cache, batch, shared = handles(w, hip)
        want = be.attend_shared(cache, batch, shared, q, window=50)
        pos, seq = positions(w), np.repeat(np.arange(4), w.n)
        # a shared page of the first three; the page of the second where the prefix ends; an own page of the first; pages that nobody is to read
        for s, entry, sees in ((0, 2, (seq < 3) & (pos - 49 <= 95)), (1, 3, (seq == 1) & (pos >= 97)), (0, 3, (seq < 3) & (pos >= 96) & (pos - 49 <= np.where(seq == 0, 127, 96))), (0, 4, (seq == 0) & (pos >= 128)), (1, 0, pos < 0), (2, 2, pos < 0)):
            pages = batch.pages.clone()
            pages[s, entry] = w.n_pages
            got = be.attend_shared(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), shared, q, window=50)
            assert got[torch.from_numpy(sees).cuda()].isnan().all()
            assert torch.equal(got[torch.from_numpy(~sees).cuda()], want[torch.from_numpy(~sees).cuda()]), (s, entry)


def test_infinite_and_nan_queries_stay_in_their_rows(be):
    from oxinfer_amd import hip
    w = Shared([77, 80, 90], [0, 3], [70], 2, 64, seed=6)
    q = torch.randn(3, 2 * 2 * 64, device="cuda")
    cache, batch, shared = handles(w, hip)
    want = be.attend_shared(cache, batch, shared, q)
    bad = q.clone()
    bad[1, 70] = float("nan")
    bad[2, 5] = float("inf")
    got = be.attend_shared(cache, batch, shared, bad)
    same = torch.ones(3, 4, dtype=torch.bool)
    same[1, 1] = same[2, 0] = False
    assert torch.equal(got.view(3, 4, 64)[same], want.view(3, 4, 64)[same])
    assert got.view(3, 4, 64)[1, 1].isnan().all() and got.view(3, 4, 64)[2, 0].isnan().all()


def test_unsound_numbers_stay_inside_the_arrays(be):
    """Lengths, row numbers and groups that do not hold together: nothing outside the tensors is read or written, and the next call is right."""
    from oxinfer_amd import hip
    w = Shared([64, 64, 64], [0, 3], [40], 1, 64, seed=3, wild=False, n=[2, 1, 3])
    cache, batch, shared = handles(w, hip, True)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(8, 64, device="cuda")
    out = torch.full((16, 64), 7.0, device="cuda")
    want = be.attend_shared(cache, batch, shared, q)[:6].clone()
    zeros = torch.zeros_like(batch.pages)
    big = 2**31 - 1
    for lens, start, groups, common in (((big, 64, -5), (0, 2, 3, 6), (0, 3), (40,)), ((64, 64, 64), (0, 2, 3, 9000), (0, 3), (40,)), ((64, 64, 64), (-7, 2, 3, 6), (0, 3), (40,)), ((64, 64, 64), (6, 3, 2, 0), (0, 3), (40,)),
                                        ((64, 64, 64), (0, 0, 0, 0), (0, 3), (40,)), ((64, 64, 64), (0, 2, 3, 6), (-4, 99), (big,)), ((64, 64, 64), (0, 2, 3, 6), (3, 0), (big,)), ((64, 3, 64), (0, 2, 3, 6), (1, 3), (big,)),
                                        ((64, 64, 64), (0, 2, 3, 6), (0, 2, 1, 3), (-1, -(2**31), 50)), ((0, 0, 0), (0, 2, 3, 6), (0, 3), (64,))):
        b = hip.KvBatch(i32(*lens), zeros, rows=6, row_start=i32(*start))
        be.attend_shared(cache, b, hip.KvShared(i32(*groups), i32(*common)), q, out=out[4:12])
        torch.cuda.synchronize()
        assert (out[:4] == 7).all() and (out[10:] == 7).all()
        assert torch.equal(be.attend_shared(cache, batch, shared, q)[:6], want)


# ---- groups of many entries, in tables with room for thousands of tokens: several tiles a group, several parts a tile ----


def broad(w):
    """w with tables for 8192 tokens at least, no page of the cache in what is added."""
    add = max(0, 8192 // w.page - w.table.shape[1])
    w.table = np.concatenate([w.table, np.full((len(w.lens), add), w.n_pages, np.int32)], 1)
    return w


def crowd(n_seqs, common, *args, n=None, starts=None, seed=0, **kwargs):
    rng = np.random.default_rng(seed)
    starts, common = ([0, n_seqs] if starts is None else starts), np.atleast_1d(common)
    least = np.zeros(n_seqs, int)
    for i, c in enumerate(common):
        least[starts[i] : starts[i + 1]] = c
    lens = least + rng.integers(0, 70, n_seqs) + (1 if n is None else np.asarray(n))
    return broad(Shared(lens, starts, common, *args, n=n, seed=seed, **kwargs))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_many_entries_of_head_sizes(be, d, dtype):
    check(be, crowd(37, 360, 2, d, page=64, seed=d), 4, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [1, 2, 3, 5, 7, 8, 12, 16, 17, 33])
def test_many_entries_of_groups_of_heads(be, g, dtype):
    n = 130 // g + 3
    check(be, crowd(n, 67, 3, 64, page=32, seed=g), g, dtype)
    check(be, crowd(n, 130, 1, 64, page=32, seed=g, n=np.random.default_rng(g).integers(1, 4, n)), g, dtype)


@pytest.mark.parametrize("common", [0, 1, 31, 32, 33, 64, 511, 512, 513, 1300])
def test_many_entries_and_lengths_of_the_prefix(be, common):
    check(be, crowd(33, common, 1, 64, page=128, seed=common), 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_entries_of_several_groups(be, dtype):
    """Groups that end inside a tile and between tiles, groups of one sequence or without shared tokens, sequences of no group."""
    for starts, common in (([0, 20, 70, 101], [50, 90, 33]), ([3, 4, 9, 90], [64, 0, 70]), ([0, 64, 96], [100, 40]), ([0, 1, 2, 3, 101], [9, 9, 70, 69])):
        check(be, crowd(101, common, 2, 64, page=32, seed=4, starts=starts), 4, dtype)
        n = np.random.default_rng(len(starts)).integers(0, 9, 101)
        check(be, crowd(101, common, 1, 96, page=64, seed=4, starts=starts, n=n), 1 if dtype == "f32" else 3, dtype, ragged=True)


def test_many_entries_of_groups_of_a_row(be):
    """Many groups of a row each, beside a group of many sequences."""
    starts = [*range(64), 200, 9000]
    check(be, broad(Shared(60 + np.arange(200), starts, [40 + i % 20 for i in range(64)] + [3], 1, 32, page=32, seed=5)), 50)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rules", RULES, ids=str)
@pytest.mark.parametrize("n", [1, 3], ids=["one", "many"])
def test_many_entries_with_masks_caps_and_biases(be, rules, n, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    w = crowd(60, [101, 75], 2, 64, page=32, seed=9, starts=[0, 36, 60], n=None if n == 1 else rng.integers(0, 7, 60))
    g = 5
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-np.arange(1, 11)).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.tile(np.array(rules["prefix"], np.int32), 12)
    pos = positions(w)
    if rules.get("first") == "docs":
        rules["first"] = (pos * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    elif rules.get("first") == "none":
        rules["first"] = np.where(np.arange(w.rows) % 2, 0, np.where(np.arange(w.rows) % 4, pos + 1, 2**31 - 1)).astype(np.int32)
    check(be, w, g, dtype, loud=4.0, **rules)


def test_many_entries_and_more_rows_than_tokens(be):
    n = [4, 7, 2, 60, 70]
    got = check(be, broad(Shared([40, 3, 0, 90, 65], [0, 5], [2], 2, 64, seed=1, n=n)), 2, ragged=True)
    assert (got[4:8] == 0).all() and (got[11:13] == 0).all() and (got[73:78] == 0).all()


def test_many_entries_of_a_long_prefix(be):
    """More than 64 blocks of a wave."""
    w = broad(Shared([40100, 40040, 40037, 40020], [0, 4], [40003], 16, 32, page=256, seed=3, n=[20, 16, 12, 16]))
    from oxinfer_amd import hip
    cache, batch, shared = handles(w, hip)
    for dtype, half in ((torch.float32, False), (torch.bfloat16, True)):
        q = (2 * torch.randn(w.rows, 128 * 32, device="cuda")).to(dtype)
        heads = [0, 60, 127]
        want, tol = kv_ref.attend(w, q.double().cpu().numpy().reshape(w.rows, 128, 32), 8, 32**-0.5, heads=heads, half=half)
        off = np.abs(be.attend_shared(cache, batch, shared, q).double().cpu().numpy().reshape(want.shape) - want)[:, heads]
        assert (off <= tol[:, heads]).all(), f"{np.max(off / np.maximum(tol[:, heads], 1e-300)):.2f} times the bound"


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 4.0])
def test_many_entries_and_scales(be, scale):
    check(be, crowd(33, 90, 2, 64, seed=2), 4, scale=scale, window=30)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_entries_with_strides_and_addresses(be, dtype):
    for n in (None, [4] * 44):
        w = crowd(44, 50, 2, 96, seed=3, n=n)
        check(be, w, 3, dtype, strided=True)
        check(be, w, 3, dtype, strided=True, odd=True)


@pytest.mark.parametrize("n", [1, 5])
def test_many_entries_with_scales_of_zero_and_values_far_apart(be, n):
    w = broad(Shared([190] + [175 + i for i in range(47)], [0, 48], [160], 2, 64, page=32, seed=6, n=[n] * 48))
    for s, page, value in ((0, 0, 0.0), (0, 1, 2.0**60), (0, 2, 2.0**-60), (0, 4, 0.0), (1, 5, 0.0), (2, 5, 2.0**-60), (3, 5, 2.0**60)):
        w.vs[w.table[s, page]] = value
    w.ks[w.table[0, 3]] = w.ks[w.table[4, 5]] = 0.0
    check(be, w, 3)


def test_many_entries_with_pages_outside_the_cache(be):
    from oxinfer_amd import hip
    n = np.array([2] * 40)
    w = broad(Shared(140 + np.arange(40), [0, 30, 40], [97, 20], 2, 64, page=32, seed=3, n=n))
    q = torch.randn(w.rows, 16 * 64, device="cuda")
    cache, batch, shared = handles(w, hip)
    want = be.attend_shared(cache, batch, shared, q, window=60)
    assert want.isfinite().all()
    pos, seq = positions(w), np.repeat(np.arange(40), 2)
    for s, entry, sees in ((0, 2, (seq < 30) & (pos - 59 <= 95)), (1, 3, (seq == 1) & (pos >= 97)), (0, 3, (seq < 30) & (pos >= 96) & (pos - 59 <= np.where(seq == 0, 127, 96))), (30, 0, (seq >= 30) & (pos - 59 <= np.where(seq == 30, 31, 19))), (5, 0, pos < 0)):
        pages = batch.pages.clone()
        pages[s, entry] = w.n_pages
        got = be.attend_shared(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), shared, q, window=60)
        assert got[torch.from_numpy(sees).cuda()].isnan().all()
        assert torch.equal(got[torch.from_numpy(~sees).cuda()], want[torch.from_numpy(~sees).cuda()]), (s, entry)


def test_many_entries_and_queries_that_are_no_numbers(be):
    from oxinfer_amd import hip
    w = crowd(40, 70, 2, 64, seed=6)
    q = torch.randn(40, 2 * 4 * 64, device="cuda")
    cache, batch, shared = handles(w, hip)
    want = be.attend_shared(cache, batch, shared, q)
    bad = q.clone()
    bad[1, 70] = float("nan")
    bad[33, 5] = float("inf")
    got = be.attend_shared(cache, batch, shared, bad)
    same = torch.ones(40, 8, dtype=torch.bool)
    same[1, 1] = same[33, 0] = False
    assert torch.equal(got.view(40, 8, 64)[same], want.view(40, 8, 64)[same])
    assert got.view(40, 8, 64)[1, 1].isnan().all() and got.view(40, 8, 64)[33, 0].isnan().all()


def test_many_entries_and_unsound_numbers(be):
    from oxinfer_amd import hip
    w = broad(Shared([64, 64, 64], [0, 3], [40], 1, 64, seed=3, wild=False, n=[20, 10, 30]))
    cache, batch, shared = handles(w, hip, True)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(62, 5 * 64, device="cuda")
    out = torch.full((70, 5 * 64), 7.0, device="cuda")
    want = be.attend_shared(cache, batch, shared, q)[:60].clone()
    zeros = torch.zeros_like(batch.pages)
    big = 2**31 - 1
    for lens, start, groups, common in (((big, 64, -5), (0, 20, 30, 60), (0, 3), (40,)), ((64, 64, 64), (0, 20, 30, 9000), (0, 3), (40,)), ((64, 64, 64), (-7, 20, 30, 60), (0, 3), (40,)), ((64, 64, 64), (60, 30, 20, 0), (0, 3), (40,)),
                                        ((64, 64, 64), (0, 0, 0, 0), (0, 3), (40,)), ((64, 64, 64), (0, 20, 30, 60), (-4, 99), (big,)), ((64, 64, 64), (0, 20, 30, 60), (3, 0), (big,)), ((64, 3, 64), (0, 20, 30, 60), (1, 3), (big,)),
                                        ((64, 64, 64), (0, 20, 30, 60), (0, 3), (-(2**31),)), ((0, 0, 0), (0, 20, 30, 60), (0, 3), (64,))):
        b = hip.KvBatch(i32(*lens), zeros, rows=60, row_start=i32(*start))
        be.attend_shared(cache, b, hip.KvShared(i32(*groups), i32(*common)), q[:60], out=out[4:64])
        torch.cuda.synchronize()
        assert (out[:4] == 7).all() and (out[64:] == 7).all()
        assert torch.equal(be.attend_shared(cache, batch, shared, q)[:60], want)


def test_many_entries_give_the_same_bits_every_time(be):
    from oxinfer_amd import hip
    w = crowd(40, 6000, 2, 128, page=64, seed=3)
    cache, batch, shared = handles(w, hip)
    q = torch.randn(40, 8 * 128, device="cuda")
    want = be.attend_shared(cache, batch, shared, q).clone()
    for _ in range(20):
        assert torch.equal(be.attend_shared(cache, batch, shared, q), want)


def test_many_entries_in_a_recorded_plan(be):
    """The lengths and the shared tokens are the device's at each replay, down to none; eager calls on another stream run beside it."""
    from oxinfer_amd import hip
    w = crowd(40, 5000, 2, 128, page=64, seed=3)
    cache, batch, shared = handles(w, hip)
    q, out = torch.randn(40, 8 * 128, device="cuda"), torch.zeros(40, 8 * 128, device="cuda")
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        be.attend_shared(cache, batch, shared, q, out=out)
        stream.synchronize()
        plan = be.plan_record(lambda: be.attend_shared(cache, batch, shared, q, out=out))
        full = batch.kv_len.clone()
        for common in (5000, 37, 0, 5000, 4097):
            shared.common.fill_(common)
            batch.kv_len.copy_(torch.minimum(full, torch.full_like(full, max(common, 1))) if common < 5000 else full)
            q.normal_()
            out.fill_(7)
            stream.synchronize()
            plan.replay()
            with torch.cuda.stream(other):
                want = be.attend_shared(cache, batch, shared, q)
            torch.cuda.synchronize()
            assert torch.equal(out, want), common
    del plan


def test_tables_that_name_the_shared_pages_fit_both_calls(be):
    """As appending sequences have them: whole shared pages in all tables. The results are attend's within both calls' bounds."""
    from oxinfer_amd import hip
    w = kv_ref.World([200, 210, 330, 250], 2, 128, page=64, seed=8)
    w.table[1:, :3] = w.table[0, :3]  # 192 tokens
    q = torch.randn(4, 8 * 128, device="cuda")
    cache, batch = w.tensors(hip)
    shared = hip.KvShared(torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.tensor([192], dtype=torch.int32, device="cuda"))
    want, tol = kv_ref.attend(w, q.double().cpu().numpy().reshape(4, 8, 128), 4, 128**-0.5)
    for got in (be.attend(cache, batch, q), be.attend_shared(cache, batch, shared, q)):
        assert (np.abs(got.double().cpu().numpy().reshape(want.shape) - want) <= tol).all()


def test_nothing_to_do(be):
    from oxinfer_amd import hip
    w = Shared([64], [0, 1], [10], 1, 64, seed=3, n=[0])
    cache, batch, shared = handles(w, hip, True)
    assert be.attend_shared(cache, batch, shared, torch.empty(0, 64, device="cuda")).shape == (0, 64)


def test_the_same_bits_every_time_and_whatever_the_rows_beside(be):
    from oxinfer_amd import hip
    for dt in (torch.float32, torch.bfloat16):
        w = Shared([9000, 9050, 9100, 8990, 9001], [0, 5], [8970], 1, 128, page=64, seed=3)
        cache, batch, shared = handles(w, hip)
        q = torch.randn(5, 4 * 128, device="cuda").to(dt)
        a = be.attend_shared(cache, batch, shared, q)
        for _ in range(20):
            assert torch.equal(a, be.attend_shared(cache, batch, shared, q))
        other = q.clone()
        other[1::2] *= 64
        got = be.attend_shared(cache, batch, shared, other)
        assert torch.equal(got[::2], a[::2]) and not torch.equal(got, a)


def test_a_recorded_plan_follows_the_lengths(be):
    """Recorded once, replayed for other lengths and other groups, with eager calls between: every replay is the eager result."""
    from oxinfer_amd import hip
    w = Shared([3000, 2900, 2950], [0, 3], [2800], 2, 128, page=64, seed=3)
    cache, batch, shared = handles(w, hip)
    q, out = torch.randn(3, 8 * 128, device="cuda"), torch.empty(3, 8 * 128, device="cuda")
    states = [([3000, 2900, 2950], [0, 3], 2800), ([2801, 2802, 2803], [0, 3], 2800), ([2999, 5, 33], [0, 1], 2990), ([64, 699, 64], [1, 3], 64), ([3000, 2900, 2950], [0, 3], 2800)]
    want = []

    def set_to(lens, groups, common):
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        shared.group_start.copy_(torch.tensor(groups, dtype=torch.int32))
        shared.common.fill_(common)

    for s in states:
        set_to(*s)
        want.append(be.attend_shared(cache, batch, shared, q))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be.attend_shared(cache, batch, shared, q, out=out)
        stream.synchronize()
        plan = be.plan_record(lambda: be.attend_shared(cache, batch, shared, q, out=out))
        for s, expect in zip(states, want):
            set_to(*s)
            out.fill_(9)
            plan.replay()
            stream.synchronize()
            assert torch.equal(out, expect), s
            assert torch.equal(be.attend_shared(cache, batch, shared, q), expect)
    del plan


def test_streams_and_threads(be):
    from oxinfer_amd import hip
    worlds = [Shared([4000 + 900 * i, 4010 + 900 * i, 3990], [0, 3], [3970], 2, 128, page=64, seed=i) for i in range(4)]
    made = [(handles(w, hip), torch.randn(3, 8 * 128, device="cuda")) for w in worlds]
    want = [be.attend_shared(*c, q) for c, q in made]
    torch.cuda.synchronize()
    wrong = []

    def go(i):
        c, q = made[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                out = be.attend_shared(*c, q)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_recording_without_scratch_is_refused(be):
    from oxinfer_amd import hip
    w = Shared([300, 310], [0, 2], [200], 1, 64, seed=3)
    cache, batch, shared = handles(w, hip)
    q, out = torch.randn(2, 64, device="cuda"), torch.empty(2, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()), pytest.raises(RuntimeError, match="plan"):
        be.plan_record(lambda: be.attend_shared(cache, batch, shared, q, out=out))


def test_the_bindings_refusals(be):
    from oxinfer_amd import hip
    w = Shared([64, 50], [0, 2], [40], 2, 64, seed=3)
    cache, batch, shared = handles(w, hip)
    q = torch.randn(2, 4 * 64, device="cuda")
    for bad in (dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q[:, : 3 * 64]), dict(out=q.bfloat16()), dict(out=q), dict(cap=-1.0), dict(window=-1), dict(slopes=torch.ones(3, device="cuda")),
                dict(first=torch.ones(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            be.attend_shared(cache, batch, shared, **(dict(q=q) | bad))
    with pytest.raises(ValueError):
        hip.KvShared(shared.group_start[:2].long(), shared.common)
    with pytest.raises(ValueError):
        hip.KvShared(shared.group_start[:1], shared.common)
