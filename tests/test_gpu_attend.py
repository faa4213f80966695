"""Attention over the 8-bit cache against the same in 64 bits (kv_ref), over sizes, head layouts, masks and biases, lengths, strides and streams."""
import threading

import numpy as np
import pytest
import torch

from tests import kv_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def check(be, w, g, dtype="f32", scale=None, seed=5, strided=False, odd=False, ragged=None, loud=2.0, heads=None, **rules):
    """One call over World w against the reference; rows behind the last sequence and what lies between rows stay as they were."""
    from oxinfer_amd import hip
    rng = np.random.default_rng(seed)
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n_q, extra = w.n_kv * g, 3
    width = n_q * w.d
    cache, batch = w.tensors(hip, ragged=ragged, extra_rows=extra)
    stride = width + (8 if strided else 0) + (1 if odd else 0)
    q = torch.from_numpy(loud * rng.normal(size=(w.rows + extra, stride))).to("cuda", tt)
    flat = torch.full(((w.rows + extra) * stride + 1,), 7.5, dtype=tt, device="cuda")
    out = flat[1 if odd else 0 :][: (w.rows + extra) * stride].view(w.rows + extra, stride)
    scale = w.d**-0.5 if scale is None else scale
    up = {k: torch.from_numpy(np.ascontiguousarray(v)).to("cuda") if isinstance(v, np.ndarray) else v for k, v in rules.items()}
    if "first" in up:
        up["first"] = torch.cat([up["first"], torch.zeros(extra, dtype=torch.int32, device="cuda")])
    be.attend(cache, batch, q[:, :width], scale=scale, out=out[:, :width], **up)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want, tol = kv_ref.attend(w, q[: w.rows, :width].double().cpu().numpy().reshape(w.rows, n_q, w.d), g, scale, half=dtype == "bf16", heads=heads, **rules)
    assert (got[w.rows :] == 7.5).all() and (got[:, width:] == 7.5).all(), "what is not the call's was written"
    off = np.abs(got[: w.rows, :width].reshape(want.shape) - want)
    if heads is not None:
        off, tol = off[:, heads], tol[:, heads]
    assert (off <= tol).all(), f"{np.max(off / np.maximum(tol, 1e-300)):.2f} times the bound"
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_head_sizes(be, d, dtype):
    check(be, kv_ref.World([397, 65], 2, d, page=64, seed=d), 4, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [1, 2, 3, 5, 8, 15, 16, 17, 33])
def test_groups_of_heads(be, g, dtype):
    check(be, kv_ref.World([70, 33, 200], 3, 64, page=32, seed=g), g, dtype)
    check(be, kv_ref.World([70, 33, 200], 1, 64, page=32, seed=g, n=[2, 5, 3]), g, dtype)


@pytest.mark.parametrize("length", [0, 1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1023, 2049, 4097])
@pytest.mark.parametrize("page", [32, 256])
def test_lengths(be, length, page):
    check(be, kv_ref.World([length, 5], 2, 128, page=page, seed=length), 4)


def test_a_long_sequence(be):
    check(be, kv_ref.World([70001], 1, 64, page=128, seed=3), 2)


def test_a_sink_that_takes_most_of_the_weight(be):
    """One key with nearly all of the weight and a value of next to nothing, then 20000 alike: what is rounded away must not add up."""
    w = kv_ref.World([20001], 1, 64, page=64, seed=4)
    w.vs[w.table[0, 0], 0, 0] *= 1e-3
    from oxinfer_amd import hip
    k, v = w.sequence(0)
    q = 30 * k[0, 0] / np.linalg.norm(k[0, 0]) * 8 / np.linalg.norm(k[0, 0])
    cache, batch = w.tensors(hip)
    qt = torch.from_numpy(q[None]).to("cuda", torch.float32)
    got = be.attend(cache, batch, qt, scale=1.0).double().cpu().numpy()
    want, tol = kv_ref.attend(w, qt.double().cpu().numpy()[:, None], 1, 1.0)
    assert (np.abs(got - want[:, 0]) <= tol[:, 0]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,lens", [([1, 1], [9, 40]), ([5], [5]), ([17, 0, 3], [17, 90, 300]), ([70, 1, 33], [70, 1, 100]), ([0, 0, 4], [7, 0, 4]), ([130], [400]), ([257, 64], [300, 64])])
def test_rows_of_ragged_sequences(be, n, lens, dtype):
    for g, d in ((1, 64), (4, 128), (3, 96)):
        check(be, kv_ref.World(lens, 2, d, page=64, seed=sum(n), n=n), g, dtype, ragged=True)


def test_more_rows_than_tokens(be):
    """Rows before a sequence's first token see nothing."""
    got = check(be, kv_ref.World([3, 0, 40], 2, 64, seed=1, n=[7, 2, 40]), 2, ragged=True)
    assert (got[:4, :256] == 0).all() and (got[7:9, :256] == 0).all()


@pytest.mark.parametrize("n_seqs", [1, 63, 64, 65, 200])
def test_many_sequences(be, n_seqs):
    rng = np.random.default_rng(n_seqs)
    n = rng.integers(0, 4, n_seqs)
    n[-1] = 2
    check(be, kv_ref.World(n + rng.integers(0, 90, n_seqs), 1, 64, seed=n_seqs, n=n), 5, ragged=True)


RULES = [dict(window=1), dict(window=33), dict(window=10**6), dict(cap=5.0), dict(cap=50.0), dict(slopes=True), dict(prefix=[20, 0, 700]), dict(prefix=[-3, 64, 33]), dict(first="docs"), dict(first="none"),
         dict(window=40, cap=30.0, slopes=True, prefix=[5, 100, 0], first="docs")]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rules", RULES, ids=str)
@pytest.mark.parametrize("n", [[1, 1, 1], [3, 70, 35]], ids=["one", "many"])
def test_masks_caps_and_biases(be, rules, n, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    w = kv_ref.World([90, 150, 300], 2, 64, page=32, seed=9, n=n)
    g = 3
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-np.arange(1, 7)).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.array(rules["prefix"], np.int32)
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(3)])
    if rules.get("first") == "docs":
        rules["first"] = (pos * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    elif rules.get("first") == "none":  # every other row sees nothing at all
        rules["first"] = np.where(np.arange(w.rows) % 2, 0, np.where(np.arange(w.rows) % 4, pos + 1, 2**31 - 1)).astype(np.int32)
    got = check(be, w, g, dtype, loud=4.0, **rules)
    if isinstance(rules.get("first"), np.ndarray) and (rules["first"][0] > pos[0]):
        assert (got[0, : 2 * g * 64] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-6, 1e-30, 4.0])
def test_scales(be, scale):
    check(be, kv_ref.World([100, 37], 2, 64, seed=2), 4, scale=scale, window=30)


def test_queries_of_any_size(be):
    """Rows scaled by powers of two that f16 does not hold: the results are those of the scaled-back rows, and a zero row is the keys' mean."""
    from oxinfer_amd import hip
    w = kv_ref.World([77], 1, 64, seed=6, n=[5])
    q = np.random.default_rng(1).normal(size=(5, 64)).astype(np.float32)
    up = np.array([1e-30, 1e-7, 1.0, 1e9, 0.0], np.float32)[:, None]
    cache, batch = w.tensors(hip, ragged=True)
    for i in range(5):
        scale = float(1 / max(up[i, 0], 1e-20) / 8)
        if scale > 1e20:
            scale = 1.0
        got = be.attend(cache, batch, torch.from_numpy(q * up[i]).cuda(), scale=scale).double().cpu().numpy()
        want, tol = kv_ref.attend(w, (q * up[i]).astype(np.float64)[:, None], 1, float(np.float32(scale)))
        assert (np.abs(got - want[:, 0]) <= tol[:, 0]).all()


def test_infinite_and_nan_queries_stay_in_their_rows(be):
    from oxinfer_amd import hip
    w = kv_ref.World([77, 50], 2, 64, seed=6, n=[4, 1])
    q = torch.randn(5, 2 * 2 * 64, device="cuda")
    cache, batch = w.tensors(hip, ragged=True)
    want = be.attend(cache, batch, q)
    bad = q.clone()
    bad[1, 70] = float("nan")
    bad[3, 5] = float("inf")
    got = be.attend(cache, batch, bad)
    same = torch.ones(5, 4, dtype=torch.bool)
    same[1, 1] = same[3, 0] = False
    assert torch.equal(got.view(5, 4, 64)[same], want.view(5, 4, 64)[same])
    assert got.view(5, 4, 64)[1, 1].isnan().all() and got.view(5, 4, 64)[3, 0].isnan().all()


def test_value_scales_far_apart(be):
    """Blocks whose value scales lie at either end of what a scale may be."""
    w = kv_ref.World([200], 1, 64, seed=6)
    for b, s in enumerate([2.0**-60, 1.0, 2.0**60, 2.0**-60, 2.0**30, 2.0**-30, 1.0]):
        w.vs[w.table[0, b], 0, 0] = s
    check(be, w, 4)
    for b in range(7):
        w.vs[w.table[0, b], 0, 0] = 2.0**-60
    check(be, w, 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_addresses(be, dtype):
    for n in ([1, 1], [20, 3]):
        w = kv_ref.World([45, 100], 2, 96, seed=3, n=n)
        check(be, w, 2, dtype, strided=True)
        check(be, w, 2, dtype, strided=True, odd=True)


def test_pages_outside_the_cache(be):
    """Rows that would see a token of such a page are NaN, the others what they are."""
    from oxinfer_amd import hip
    for n in ([1, 1, 1], [40, 90, 2]):
        w = kv_ref.World([100, 90, 64], 2, 64, seed=3, n=n)
        q = torch.randn(w.rows, 4 * 64, device="cuda")
        cache, batch = w.tensors(hip)
        want = be.attend(cache, batch, q, window=50)
        pages = batch.pages.clone()
        pages[1, 1] = w.n_pages  # tokens 32 .. 63 of the second sequence
        got = be.attend(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), q, window=50)
        pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(3)])
        sees = (np.repeat(np.arange(3), w.n) == 1) & (pos >= 32) & (pos - 49 <= 63)
        assert got[torch.from_numpy(sees).cuda()].isnan().all() and sees.any()
        assert torch.equal(got[torch.from_numpy(~sees).cuda()], want[torch.from_numpy(~sees).cuda()])


def test_unsound_lengths_stay_inside_the_arrays(be):
    """Lengths that the table cannot hold, and rows that the batch does not have, are cut off: the tensors' guards stay as they were."""
    from oxinfer_amd import hip
    w = kv_ref.World([64, 64], 1, 64, seed=3, wild=False)
    cache, batch = w.tensors(hip, ragged=True)
    out = torch.full((12, 64), 7.0, device="cuda")
    for lens, start in (([2**31 - 1, 64], [0, 1, 2]), ([-5, -2**31], [0, 1, 2]), ([64, 64], [0, 1, 9000]), ([64, 64], [-7, 1, 2]), ([64, 64], [2, 1, 0]), ([64, 64], [0, 0, 0])):
        b = hip.KvBatch(torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.zeros_like(batch.pages), rows=2, row_start=torch.tensor(start, dtype=torch.int32, device="cuda"))
        be.attend(cache, b, torch.randn(4, 64, device="cuda"), out=out[4:8])
        be.kv_read(cache, b, 40)
        torch.cuda.synchronize()
        assert (out[:4] == 7).all() and (out[6:] == 7).all()


def test_a_cache_of_more_than_4_gib(be):
    """Pages whose codes lie past 2^32 bytes, and whose tokens' products of index and size pass 2^31."""
    from oxinfer_amd import hip
    n_kv, d, page = 8, 128, 256
    n_pages = 2**32 // (n_kv * d * page) + 40
    k, v = (torch.empty((n_pages, n_kv, page // 32, 32 * d), dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = [torch.empty((n_pages, n_kv, page // 32), device="cuda") for _ in range(2)]
    cache = hip.KvCache(k, v, *scales, page, d)
    small = kv_ref.World([300, 256], n_kv, d, page=page, seed=1, spare=0, wild=False)
    far = torch.tensor([n_pages - 1 - 7 * i for i in range(small.n_pages)], device="cuda")
    small_cache, small_batch = small.tensors(hip)
    for big, own in zip((k, v, *scales), (small_cache.k, small_cache.v, small_cache.k_scale, small_cache.v_scale)):
        big[far] = own
    q = torch.randn(2, 32 * d, device="cuda")
    batch = hip.KvBatch(small_batch.kv_len, far[small_batch.pages.long()].to(torch.int32))
    assert torch.equal(be.attend(cache, batch, q), be.attend(small_cache, small_batch, q))
    for a, b in zip(be.kv_read(cache, batch, 260), be.kv_read(small_cache, small_batch, 260)):
        assert torch.equal(a, b)


# ---- batches of many rows, which the matrix-core-bound kernel takes: rows x heads of 256 tiles of 128 entries and more (a few heads are checked) ----


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_prompts_of_every_head_size(be, d, dtype):
    """Both widths of workgroup, the second from 1024 tiles on; last rows that fill a tile in part, keys that end inside a block."""
    for rows, n_kv, g in ((max(130, 32768 * 128 // d // 64 + 3) if d < 128 else 513, 8, 8), (1029, 16, 8)):
        if d < 128 and rows == 1029:
            rows = 2053
        w = kv_ref.World([rows + 77], n_kv, d, page=64, seed=d, n=[rows])
        assert rows * g * n_kv // 128 >= 256 and rows * g * n_kv // 128 * d >= 256 * 128
        check(be, w, g, dtype, heads=[0, n_kv * g - 1], ragged=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rules", RULES, ids=str)
def test_prompts_with_masks_caps_and_biases(be, rules, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    n = [3, 211, 0, 130, 16, 1]
    w = kv_ref.World([90, 350, 40, 130, 200, 333], 16, 128, page=32, seed=9, n=n)
    g = 8
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-8 * np.arange(1, 129) / 128).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.array((rules["prefix"] * 2)[:6], np.int32)
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(6)])
    if rules.get("first") == "docs":
        rules["first"] = (pos * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    elif rules.get("first") == "none":
        rules["first"] = np.where(np.arange(w.rows) % 2, 0, np.where(np.arange(w.rows) % 4, pos + 1, 2**31 - 1)).astype(np.int32)
    check(be, w, g, dtype, loud=4.0, heads=[0, 60, 127], **rules)


@pytest.mark.parametrize("n,lens", [([128, 1, 128], [128, 4000, 300]), ([15, 17, 400], [15, 17, 400]), ([300, 90], [70, 33]), ([1] * 70 + [290], [33] * 70 + [290])])
@pytest.mark.parametrize("g", [3, 8, 16, 40])
def test_prompts_beside_single_tokens(be, n, lens, g):
    """Sequences on either side of the border between the kernels in one call, groups that tiles do not divide into, rows before the first token."""
    n_kv = -(-256 * 128 // (sum(n) * g)) + 1
    w = kv_ref.World(lens, n_kv, 128, page=64, seed=g, n=n)
    for dtype in ("f32", "bf16"):
        check(be, w, g, dtype, heads=[0, n_kv * g // 2, n_kv * g - 1], ragged=True)


def test_a_prompt_in_a_buffer_for_more(be):
    """The batch has room for many rows, the one sequence hardly any: the other rows stay as they are."""
    from oxinfer_amd import hip
    w = kv_ref.World([50], 8, 128, seed=2, n=[3])
    cache, batch = w.tensors(hip, ragged=True)
    big = hip.KvBatch(batch.kv_len, batch.pages, rows=1000, row_start=batch.row_start)
    q = torch.randn(1000, 64 * 128, device="cuda")
    out = torch.full_like(q, 3.0)
    be.attend(cache, big, q, out=out)
    want, tol = kv_ref.attend(w, q[:3].double().cpu().numpy().reshape(3, 64, 128), 8, 128**-0.5)
    assert (np.abs(out[:3].double().cpu().numpy().reshape(want.shape) - want) <= tol).all() and (out[3:] == 3).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_prompts_of_other_scales_strides_and_addresses(be, scale, dtype):
    w = kv_ref.World([300, 64], 16, 128, page=64, seed=3, n=[260, 5])
    check(be, w, 8, dtype, scale=scale, heads=[1, 77], strided=True)
    check(be, w, 8, dtype, scale=0.1, heads=[1, 77], strided=True, odd=True)


def test_prompts_pages_outside_the_cache_and_queries_that_are_not_numbers(be):
    from oxinfer_amd import hip
    w = kv_ref.World([400, 64], 16, 128, page=32, seed=3, n=[300, 5])
    q = torch.randn(w.rows, 128 * 128, device="cuda")
    cache, batch = w.tensors(hip)
    want = be.attend(cache, batch, q, window=100)
    pages = batch.pages.clone()
    pages[0, 5] = w.n_pages  # tokens 160 .. 191 of the first sequence
    got = be.attend(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), q, window=100)
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(2)])
    sees = torch.from_numpy((np.repeat(np.arange(2), w.n) == 0) & (pos >= 160) & (pos - 99 <= 191)).cuda()
    assert got[sees].isnan().all() and sees.any() and torch.equal(got[~sees], want[~sees])
    bad = q.clone()
    bad[7, 130] = float("nan")
    bad[200, 5] = float("inf")
    got = be.attend(cache, batch, bad, window=100).view(w.rows, 128, 128)
    same = torch.ones(w.rows, 128, dtype=torch.bool)
    same[7, 1] = same[200, 0] = False
    assert torch.equal(got[same], want.view(w.rows, 128, 128)[same]) and got[7, 1].isnan().all() and got[200, 0].isnan().all()


@pytest.mark.parametrize("seqs", [3, 70])
def test_row_numbers_that_do_not_ascend_leave_nothing_behind(be, seqs):
    """Sequences that claim each other's rows: nothing is written, and the next call of the same stream is right (parts that wait for others
    meet by counters)."""
    from oxinfer_amd import hip
    w = kv_ref.World([3000] * seqs, 2, 64, page=64, seed=4, n=[2] * seqs)
    cache, batch = w.tensors(hip, ragged=True)
    q = torch.randn(w.rows, 8 * 64, device="cuda")
    want = be.attend(cache, batch, q)
    for at, value in ((seqs - 1, 0), (1, 2 * seqs), (0, 2**31 - 1), (seqs, -(2**31))):
        start = batch.row_start.clone()
        start[at] = value
        out = torch.full_like(q, 7.5)
        be.attend(cache, hip.KvBatch(batch.kv_len, batch.pages, rows=w.rows, row_start=start), q, out=out)
        assert (out == 7.5).all()
        assert torch.equal(be.attend(cache, batch, q), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [[5, 3], [300, 5]])
def test_a_rows_bits_do_not_depend_on_the_rows_beside_it(be, n, dtype):
    from oxinfer_amd import hip
    w = kv_ref.World([900, 64], 2, 128, page=32, seed=3, n=n)
    cache, batch = w.tensors(hip)
    q = torch.randn(w.rows, 8 * 128, device="cuda").to(dtype)
    want = be.attend(cache, batch, q)
    for part in (slice(0, None, 3), slice(1, None, 2)):
        other = q.clone()
        other[part] *= 64
        kept = torch.ones(w.rows, dtype=torch.bool)
        kept[part] = False
        got = be.attend(cache, batch, other)
        assert torch.equal(got[kept], want[kept]) and not torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_by_a_recorded_plan_and_the_same_bits_every_time(be, dtype):
    from oxinfer_amd import hip
    w = kv_ref.World([1000, 500, 700], 16, 128, page=64, seed=3, n=[300, 2, 150])
    cache, batch = w.tensors(hip)
    q = torch.randn(w.rows, 128 * 128, device="cuda").to(dtype)
    out = torch.empty_like(q)
    want = {}
    lengths = [[1000, 500, 700], [300, 2, 150], [777, 499, 151], [1000, 500, 700]]
    for lens in lengths:
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        want[tuple(lens)] = be.attend(cache, batch, q)
        for _ in range(5):
            assert torch.equal(want[tuple(lens)], be.attend(cache, batch, q))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be.attend(cache, batch, q, out=out)
        stream.synchronize()
        plan = be.plan_record(lambda: be.attend(cache, batch, q, out=out))
        for lens in lengths:
            batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            out.fill_(9)
            plan.replay()
            stream.synchronize()
            assert torch.equal(out, want[tuple(lens)]), lens
    del plan


def test_nothing_to_do(be):
    from oxinfer_amd import hip
    w = kv_ref.World([64], 1, 64, seed=3, n=[0])
    cache, batch = w.tensors(hip, ragged=True)
    assert be.attend(cache, batch, torch.empty(0, 64, device="cuda")).shape == (0, 64)


def test_the_same_bits_every_time(be):
    """Splits and waves meet in a fixed order."""
    from oxinfer_amd import hip
    for n, g, dt in (([1], 8, torch.float32), ([1], 8, torch.bfloat16), ([300], 2, torch.bfloat16), ([300], 2, torch.float32)):
        w = kv_ref.World([9000], 1, 128, page=64, seed=3, n=n)
        cache, batch = w.tensors(hip)
        q = torch.randn(w.rows, g * 128, device="cuda").to(dt)
        a = be.attend(cache, batch, q)
        for _ in range(20):
            assert torch.equal(a, be.attend(cache, batch, q))


def test_a_recorded_plan_follows_the_lengths(be):
    """Recorded once, replayed for sequences of other lengths, with eager calls on another stream between: every replay is the eager result."""
    from oxinfer_amd import hip
    w = kv_ref.World([3000, 700, 64], 2, 128, page=64, seed=3)
    cache, batch = w.tensors(hip)
    q, out = torch.randn(3, 8 * 128, device="cuda"), torch.empty(3, 8 * 128, device="cuda")
    lengths = [[3000, 700, 64], [1, 2, 3], [2999, 0, 33], [64, 699, 64], [3000, 700, 64]]
    want = []
    for lens in lengths:
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        want.append(be.attend(cache, batch, q))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be.attend(cache, batch, q, out=out)
        stream.synchronize()
        plan = be.plan_record(lambda: be.attend(cache, batch, q, out=out))
        for lens, expect in zip(lengths, want):
            batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            out.fill_(9)
            plan.replay()
            stream.synchronize()
            assert torch.equal(out, expect), lens
    del plan


def test_recording_without_scratch_is_refused(be):
    from oxinfer_amd import hip
    w = kv_ref.World([300], 1, 64, seed=3)
    cache, batch = w.tensors(hip)
    q, out = torch.randn(1, 64, device="cuda"), torch.empty(1, 64, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), pytest.raises(RuntimeError, match="plan"):
        be.plan_record(lambda: be.attend(cache, batch, q, out=out))


def test_streams_and_threads(be):
    """Calls of four threads, each on a stream of its own, at once."""
    from oxinfer_amd import hip
    worlds = [kv_ref.World([4000 + 900 * i, 77], 2, 128, page=64, seed=i) for i in range(4)]
    made = [(w.tensors(hip), torch.randn(2, 8 * 128, device="cuda")) for w in worlds]
    want = [be.attend(*c, q) for c, q in made]
    torch.cuda.synchronize()
    wrong = []

    def go(i):
        (cache, batch), q = made[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                out = be.attend(cache, batch, q)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_the_bindings_refusals(be):
    from oxinfer_amd import hip
    w = kv_ref.World([64, 9], 2, 64, seed=3)
    cache, batch = w.tensors(hip)
    q = torch.randn(2, 4 * 64, device="cuda")
    for bad in (dict(q=q.half()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q[:, :-1]), dict(q=q[:, : 3 * 64]), dict(out=q.bfloat16()), dict(out=q.t().contiguous().t()), dict(cap=-1.0), dict(window=-1),
                dict(slopes=torch.ones(3, device="cuda")), dict(slopes=torch.ones(4)), dict(prefix=torch.ones(2, device="cuda")), dict(first=torch.ones(1, dtype=torch.int32, device="cuda"))):
        args = dict(q=q) | bad
        with pytest.raises((ValueError, RuntimeError)):
            be.attend(cache, batch, **args)
    with pytest.raises(ValueError):
        hip.KvBatch(batch.kv_len, batch.pages[:1])
    with pytest.raises(ValueError):
        hip.KvCache(cache.k, cache.v[:1], cache.k_scale, cache.v_scale, 32, 64)
