"""The mean keys of a cache's spans, the choice among them, and the attention over what was chosen, against the same in 64 bits (lists_ref)."""
import numpy as np
import pytest
import torch

from tests import kv_ref, lists_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def positions(w):
    return np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(len(w.lens))])


def summary(be, w, hip, cache, span, rng):
    """A summary of World w: (KvSummary, codes, scales), what no span needs being as wild as the cache."""
    code = rng.integers(-127, 128, (w.n_pages, w.n_kv, w.page // span, w.d)).astype(np.int8)
    scale = (0.01 * np.exp(rng.normal(size=code.shape[:3]))).astype(np.float32)
    return hip.KvSummary(torch.from_numpy(code.copy()).cuda(), torch.from_numpy(scale.copy()).cuda(), span), code, scale


# ---- mean keys ------------------------------------------------------------------------------------------------------------------------------


def check_means(be, w, span, ragged=None):
    from oxinfer_amd import hip
    cache, batch = w.tensors(hip, ragged=ragged)
    held, code, scale = summary(be, w, hip, cache, span, np.random.default_rng(1))
    be.kv_summarize(cache, batch, held)
    lists_ref.summarize(w, span, code, scale)
    assert np.array_equal(held.scale.cpu().numpy(), scale, equal_nan=True)
    assert np.array_equal(held.code.cpu().numpy(), code)
    for count in (1, 3):
        got = be.kv_summary_read(cache, batch, held, count).cpu().numpy()
        for s in range(len(w.lens)):
            last = (int(w.lens[s]) - 1) // span if w.lens[s] else -1
            for i in range(count):
                x = last - count + 1 + i
                if x < 0:
                    assert (got[s, i] == 0).all()
                    continue
                p, at = w.table[s, x * span // w.page], x * span % w.page // span
                want = code[p, :, at].astype(np.float32) * scale[p, :, at][:, None] if 0 <= p < w.n_pages else np.full(got[s, i].shape, np.nan)
                assert np.array_equal(got[s, i], want, equal_nan=True)


@pytest.mark.parametrize("d", range(32, 257, 32))
def test_means_of_every_head_size(be, d):
    check_means(be, kv_ref.World([397, 65, 1], 2, d, page=128, seed=d), 64)
    check_means(be, kv_ref.World([397, 65], 3, d, page=64, seed=d, n=[290, 3]), 32)


@pytest.mark.parametrize("page,span", [(32, 32), (64, 64), (256, 32), (256, 128), (1024, 1024)])
@pytest.mark.parametrize("n,lens", [([1, 1, 1], [1, 32, 33]), ([1, 1, 1], [64, 65, 1025]), ([40, 0, 2, 7], [40, 90, 300, 5]), ([700, 64, 128], [2000, 64, 130]), ([0, 3], [0, 0])])
def test_means_where_rows_begin_and_end(be, n, lens, page, span):
    check_means(be, kv_ref.World(lens, 2, 64, page=page, seed=sum(lens), n=n), span, ragged=True)


def test_means_of_scales_at_their_ends(be):
    w = kv_ref.World([300], 2, 64, page=64, seed=4, n=[300])
    for page, value in ((0, 0.0), (1, 2.0**60), (2, 2.0**-60), (3, 2.0**-61)):
        w.ks[w.table[0, page]] = value
    w.k[w.table[0, 4]] = 128  # (all keys zero)
    from oxinfer_amd import hip
    cache, batch = w.tensors(hip, ragged=True)
    held, code, scale = summary(be, w, hip, cache, 64, np.random.default_rng(1))
    be.kv_summarize(cache, batch, held)
    w.ks[w.table[0, 3]] = 0  # (a scale under 2^-60 counts as 0)
    lists_ref.summarize(w, 64, code, scale)
    assert np.array_equal(held.scale.cpu().numpy(), scale) and np.array_equal(held.code.cpu().numpy(), code)
    assert (scale[w.table[0, [0, 3, 4]]] == 0).all()


def test_means_of_pages_outside_the_cache_are_not_written(be):
    from oxinfer_amd import hip
    w = kv_ref.World([100, 90], 1, 64, page=32, seed=4, n=[100, 90])
    w.table[0, 1], w.table[1, 0] = -1, -w.n_pages
    cache, batch = w.tensors(hip)
    held, code, scale = summary(be, w, hip, cache, 32, np.random.default_rng(1))
    was = code.copy()
    be.kv_summarize(cache, batch, held)
    lists_ref.summarize(w, 32, code, scale)
    assert np.array_equal(held.code.cpu().numpy(), code) and np.array_equal(held.scale.cpu().numpy(), scale) and not np.array_equal(code, was)
    assert be.kv_summary_read(cache, batch, held, 3)[1, 0].isnan().all()


# ---- the choice -----------------------------------------------------------------------------------------------------------------------------


def check_choice(be, w, g, span, count, first=1, last=1, dtype="f32", ragged=None, change=None, q=None, strided=False):
    from oxinfer_amd import hip
    rng = np.random.default_rng(3)
    cache, batch = w.tensors(hip, ragged=ragged)
    held, code, scale = summary(be, w, hip, cache, span, rng)
    if change:
        change(code, scale)
        held = hip.KvSummary(torch.from_numpy(code.copy()).cuda(), torch.from_numpy(scale.copy()).cuda(), span)
    width = w.n_kv * g * w.d
    x = torch.from_numpy(rng.normal(size=(w.rows, width + (5 if strided else 0))) if q is None else q).to("cuda", torch.bfloat16 if dtype == "bf16" else torch.float32)
    out = torch.full((w.rows + 2, w.n_kv, count), 77, dtype=torch.int32, device="cuda")
    be.kv_select(cache, batch, held, x[:, :width], count, first=first, last=last, out=out)
    with np.errstate(all="ignore"):
        want = lists_ref.select(w, x[:, :width].float().cpu().numpy().reshape(w.rows, w.n_kv * g, w.d), g, span, code, scale, count, first, last)
    assert np.array_equal(out[: w.rows].cpu().numpy(), want)
    assert (out[w.rows :] == 77).all()
    return want


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_choice_of_every_head_size(be, d, dtype):
    check_choice(be, kv_ref.World([3000, 700, 40], 2, d, page=64, seed=d), 4, 32, 9, dtype=dtype)


@pytest.mark.parametrize("g", [1, 2, 3, 8, 15, 16, 17, 40])
def test_choice_of_groups_of_heads(be, g):
    check_choice(be, kv_ref.World([3000, 1700], 2, 64, page=128, seed=g), g, 64, 8, strided=True)


@pytest.mark.parametrize("count,first,last", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (5, 0, 5), (5, 5, 0), (5, 2, 3), (30, 1, 2), (31, 1, 2), (32, 0, 0), (33, 1, 1), (200, 3, 4)])
def test_how_many_are_taken(be, count, first, last):
    """Around the 32 spans that the longest sequence has."""
    check_choice(be, kv_ref.World([1024, 1023, 993, 992, 33, 1, 0], 2, 64, page=32, seed=count), 2, 32, count, first, last)


@pytest.mark.parametrize("n,lens", [([5, 2], [2000, 139]), ([17, 0, 3], [40, 90, 900]), ([70, 1, 33], [70, 1, 2000]), ([0, 0, 4], [7, 3, 1500]), ([7, 2], [3, 0])])
def test_choice_for_ragged_rows(be, n, lens):
    check_choice(be, kv_ref.World(lens, 2, 64, page=64, seed=sum(n), n=n), 3, 32, 4, ragged=True)


@pytest.mark.parametrize("span,page", [(32, 256), (64, 64), (256, 256)])
def test_choice_among_many_spans(be, span, page):
    check_choice(be, kv_ref.World([100001], 1, 64, page=page, seed=span), 2, span, 50)


def test_equal_scores_take_the_lower_number(be):
    w = kv_ref.World([2000, 1999], 2, 64, page=64, seed=2)

    def alike(code, scale):
        code[:] = code[0, 0, 0]
        scale[:] = 0.5

    want = check_choice(be, w, 2, 32, 10, first=1, last=2, change=alike)
    assert want[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 61, 62]

    def two(code, scale):  # every other span scores a little more or less, and scores of zero
        code[:] = code[0, 0, 0]
        scale[:] = np.random.default_rng(1).choice([0.25, 0.5, 0.0], scale.shape)

    check_choice(be, w, 2, 32, 30, change=two)


def test_scores_of_any_size(be):
    w = kv_ref.World([3000], 1, 64, page=32, seed=2)
    for spread in (1e-30, 60.0, 80.0):
        check_choice(be, w, 2, 32, 20, change=lambda code, scale: np.copyto(scale, np.exp(np.random.default_rng(1).normal(size=scale.shape) * spread / 2).clip(1e-38, 1e38).astype(np.float32)))
    q = np.random.default_rng(5).normal(size=(1, 2 * 64))
    for size in (1e-44, 1e-30, 1e30, 0.0):
        check_choice(be, w, 2, 32, 20, q=q * size)


def test_choice_of_infinities_and_nan(be):
    w = kv_ref.World([3000, 2900], 1, 64, page=32, seed=2)
    q = np.random.default_rng(5).normal(size=(2, 2 * 64))
    q[0, 3], q[0, 70], q[1, 5] = np.nan, np.inf, -np.inf
    check_choice(be, w, 2, 32, 20, q=q)


def test_choice_with_pages_outside_the_cache(be):
    """They come last; the first and last spans are taken all the same."""
    w = kv_ref.World([640, 640], 1, 64, page=32, seed=2)
    w.table[0, [3, 4, 5, 6, 7, 19]] = -1
    want = check_choice(be, w, 2, 32, 6, last=2)
    assert not set(want[0, 0].tolist()) & {3, 4, 5, 6, 7} and 19 in want[0, 0]
    check_choice(be, w, 2, 32, 17, last=2)


# ---- the attention over it ------------------------------------------------------------------------------------------------------------------


def lists(w, count, span, rng, full=False):
    """Random ascending lists, -1 behind; with the row's own span where `full`."""
    out = np.full((w.rows, w.n_kv, count), -1, np.int32)
    for r, pos in enumerate(positions(w)):
        spans = int(pos) // span + 1 if pos >= 0 else 0
        for h in range(w.n_kv):
            some = rng.permutation(spans)[: min(count, spans) if full else rng.integers(0, min(count, spans) + 1)]
            if full and spans:
                some = np.unique(np.append(some[: count - 1], spans - 1))
            out[r, h, : len(some)] = np.sort(some)
    return out


def check(be, w, g, span, chosen, dtype="f32", scale=None, ragged=None, strided=False, loud=2.0, **rules):
    from oxinfer_amd import hip
    rng = np.random.default_rng(5)
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    ragged = (w.n != 1).any() if ragged is None else ragged
    extra = 3 if ragged else 0
    n_q = w.n_kv * g
    width = n_q * w.d
    cache, batch = w.tensors(hip, ragged=ragged, extra_rows=extra)
    stride = width + (9 if strided else 0)
    q = torch.from_numpy(loud * rng.normal(size=(w.rows + extra, stride))).to("cuda", tt)
    out = torch.full((w.rows + extra, stride), 7.5, dtype=tt, device="cuda")
    scale = w.d**-0.5 if scale is None else scale
    up = {k: torch.from_numpy(np.ascontiguousarray(v)).to("cuda") if isinstance(v, np.ndarray) else v for k, v in rules.items()}
    if "first" in up:
        up["first"] = torch.cat([up["first"], torch.zeros(extra, dtype=torch.int32, device="cuda")])
    named = torch.from_numpy(np.concatenate([chosen, np.zeros((extra, *chosen.shape[1:]), np.int32)])).cuda()
    be.attend_selected(cache, batch, q[:, :width], named, span, scale=scale, out=out[:, :width], **up)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want, tol = lists_ref.attend_selected(w, q[: w.rows, :width].double().cpu().numpy().reshape(w.rows, n_q, w.d), g, scale, chosen, span, half=dtype == "bf16", **rules)
    assert (got[w.rows :] == 7.5).all() and (got[:, width:] == 7.5).all(), "what is not the call's was written"
    off = np.abs(got[: w.rows, :width].reshape(want.shape) - want)
    assert (off <= tol).all(), f"{np.max(off / np.maximum(tol, 1e-300)):.2f} times the bound"
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_attention_of_every_head_size(be, d, dtype):
    w = kv_ref.World([1397, 365], 2, d, page=64, seed=d)
    check(be, w, 4, 64, lists(w, 7, 64, np.random.default_rng(d), full=True), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [1, 2, 3, 8, 15, 16, 17, 33])
def test_attention_of_groups_of_heads(be, g, dtype):
    w = kv_ref.World([470, 833, 200], 2, 64, page=32, seed=g, n=[2, 5, 3])
    check(be, w, g, 32, lists(w, 9, 32, np.random.default_rng(g)), dtype, strided=True)


@pytest.mark.parametrize("span,page", [(32, 32), (32, 256), (64, 64), (128, 256), (1024, 1024)])
def test_attention_of_spans_and_pages(be, span, page):
    w = kv_ref.World([5000, 31, 32, 33, 1025, 1, 0], 1, 64, page=page, seed=span)
    for count in (1, 2, 64, 65, 200):
        check(be, w, 2, span, lists(w, count, span, np.random.default_rng(count), full=True))


def test_attention_of_long_lists(be):
    w = kv_ref.World([60001], 1, 64, page=64, seed=3)
    check(be, w, 2, 64, lists(w, 600, 64, np.random.default_rng(1), full=True))
    check(be, w, 2, 64, lists(w, 938, 64, np.random.default_rng(1), full=True))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,lens", [([5, 2], [40, 39]), ([17, 0, 3], [40, 90, 300]), ([70, 1, 33], [100, 60, 100]), ([0, 0, 4], [7, 3, 4]), ([7, 2], [3, 0])])
def test_attention_for_ragged_rows(be, n, lens, dtype):
    w = kv_ref.World(lens, 2, 96, page=64, seed=sum(n), n=n)
    check(be, w, 3, 32, lists(w, 3, 32, np.random.default_rng(1)), dtype, ragged=True)


RULES = [dict(window=1), dict(window=33), dict(window=100), dict(cap=5.0), dict(slopes=True), dict(prefix=[20, 0, 700]), dict(window=20, prefix=[10, 130, 4]), dict(first="docs"), dict(window=40, cap=30.0, slopes=True, prefix=[5, 100, 0], first="docs")]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rules", RULES, ids=str)
def test_attention_with_masks_caps_and_biases(be, rules, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    w = kv_ref.World([190, 350, 300], 2, 64, page=32, seed=9, n=[3, 20, 1])
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-np.arange(1, 7)).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.array(rules["prefix"], np.int32)
    if "first" in rules:
        rules["first"] = (positions(w) * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    check(be, w, 3, 32, lists(w, 6, 32, rng, full=True), dtype, loud=4.0, **rules)


# ---- batches of many rows of a sequence, a wave a row and key head: 32 rows of a sequence and 2048 of these waves at least ----


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_many_rows_of_every_head_size(be, d, dtype):
    w = kv_ref.World([1397, 365], 32, d, page=64, seed=d, n=[60, 7])
    check(be, w, 2, 64, lists(w, 7, 64, np.random.default_rng(d)), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [1, 3, 4, 5, 8, 9])
def test_many_rows_of_groups_of_heads(be, g, dtype):
    w = kv_ref.World([470, 833, 64], 32, 64, page=32, seed=g, n=[60, 35, 5])
    check(be, w, g, 32, lists(w, 9, 32, np.random.default_rng(g)), dtype, strided=True)


@pytest.mark.parametrize("span,page,count", [(32, 32, 1), (32, 256, 2), (32, 64, 65), (64, 64, 33), (128, 256, 16), (1024, 1024, 3), (32, 32, 130)])
def test_many_rows_of_spans_and_pages(be, span, page, count):
    """Lists that end at, before and behind each set's turn and each 64 blocks; rows before the first token, rows behind the last sequence."""
    w = kv_ref.World([5000, 31, 1025], 24, 64, page=page, seed=span, n=[60, 40, 6])
    check(be, w, 2, span, lists(w, count, span, np.random.default_rng(count), full=True), ragged=True)
    w = kv_ref.World([3000], 32, 32, page=page, seed=span, n=[64])
    check(be, w, 5, span, lists(w, count, span, np.random.default_rng(count)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("g", [3, 6])
@pytest.mark.parametrize("rules", RULES, ids=str)
def test_many_rows_with_masks_caps_and_biases(be, rules, g, dtype):
    rules = dict(rules)
    rng = np.random.default_rng(8)
    w = kv_ref.World([190, 350], 32, 64, page=32, seed=9, n=[46, 20])
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-8 * np.arange(1, 32 * g + 1) / (32 * g)).astype(np.float32)
    if "prefix" in rules:
        rules["prefix"] = np.array(rules["prefix"][:2], np.int32)
    if "first" in rules:
        rules["first"] = (positions(w) * rng.integers(0, 5, w.rows) // 4).astype(np.int32)
    check(be, w, g, 32, lists(w, 6, 32, rng, full=True), dtype, loud=4.0, **rules)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 30.0])
def test_many_rows_of_other_scales(be, scale):
    w = kv_ref.World([400, 300], 32, 64, page=64, seed=3, n=[60, 5])
    check(be, w, 3, 32, lists(w, 6, 32, np.random.default_rng(1)), scale=scale)


def test_many_rows_of_scales_at_their_ends(be):
    """Scales of zero, the least and the largest, in blocks of one set and of several."""
    w = kv_ref.World([800, 700], 32, 64, page=32, seed=6, n=[60, 9])
    for page, value in ((0, 0.0), (1, 2.0**-60), (2, 0.0), (3, 2.0**60), (4, 0.0), (9, 2.0**59), (10, 0.0)):
        w.vs[w.table[:, page]] = value
    w.ks[w.table[0, 3]] = w.ks[w.table[1, 4]] = 0.0
    check(be, w, 3, 32, lists(w, 14, 32, np.random.default_rng(2), full=True))


def test_many_rows_with_pages_outside_the_cache_and_lists_that_are_not_sound(be):
    from oxinfer_amd import hip
    w = kv_ref.World([300, 280], 32, 64, page=32, seed=3, n=[60, 30])
    chosen = np.random.default_rng(2).integers(-3, 12, (w.rows, 32, 6)).astype(np.int32)
    check(be, w, 2, 32, chosen)
    q = torch.randn(w.rows, 64 * 64, device="cuda")
    cache, batch = w.tensors(hip)
    up = torch.from_numpy(chosen).cuda()
    want = be.attend_selected(cache, batch, q, up, 32).view(w.rows, 32, 2, 64)
    seq, pos = np.repeat([0, 1], w.n), positions(w)
    for s, entry in ((0, 2), (1, 0), (1, 8)):
        pages = batch.pages.clone()
        pages[s, entry] = -1
        got = be.attend_selected(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), q, up, 32).view(w.rows, 32, 2, 64)
        sees = np.array([[seq[r] == s and lists_ref.named(chosen[r, h], int(pos[r]), 32)[entry * 32 : entry * 32 + 32].any() for h in range(32)] for r in range(w.rows)])
        sees = torch.from_numpy(sees).cuda()
        assert sees.any() and got[sees].isnan().all() and torch.equal(got[~sees], want[~sees])


def test_lists_that_are_not_sound(be):
    """Numbers that do not ascend, come twice, are negative or lie past the row's own span name nothing; a row without any gives zeros."""
    w = kv_ref.World([200, 200, 200, 200, 200], 1, 64, page=32, seed=3)
    big = 2**31 - 1
    chosen = np.array([[3, 3, 2, 5, -1], [-1, 0, -7, 2, 6], [7, 8, big, -(2**31), 1], [-1, -1, -1, -1, -1], [big, 0, 6, 7, 6]], np.int32)[:, None]
    got = check(be, w, 2, 32, chosen)
    assert (got[3] == 0).all()


def test_attention_with_pages_outside_the_cache(be):
    from oxinfer_amd import hip
    w = kv_ref.World([200, 180], 2, 64, page=32, seed=3, n=[2, 3])
    chosen = lists(w, 3, 32, np.random.default_rng(2))
    q = torch.randn(w.rows, 4 * 64, device="cuda")
    cache, batch = w.tensors(hip)
    named = torch.from_numpy(chosen).cuda()
    want = be.attend_selected(cache, batch, q, named, 32)
    hit = 0
    for s, entry in ((0, 2), (1, 0), (1, 4), (0, 6)):
        pages = batch.pages.clone()
        pages[s, entry] = -1
        got = be.attend_selected(cache, hip.KvBatch(batch.kv_len, pages, rows=w.rows, row_start=batch.row_start), q, named, 32).view(w.rows, 2, 2, 64)
        sees = torch.from_numpy((np.repeat([0, 1], w.n) == s)[:, None] & (chosen == entry).any(2)).cuda()
        assert got[sees].isnan().all() and torch.equal(got[~sees], want.view(w.rows, 2, 2, 64)[~sees])
        hit += int(sees.sum())
    assert hit


def test_unsound_numbers_stay_inside_the_arrays(be):
    from oxinfer_amd import hip
    w = kv_ref.World([64, 64], 1, 64, seed=3, wild=False)
    cache, batch = w.tensors(hip, ragged=True)
    held = be.kv_summary(cache, 32)
    out = torch.full((12, 64), 7.0, device="cuda")
    q = torch.randn(4, 64, device="cuda")
    picks = torch.full((12, 1, 1), 77, dtype=torch.int32, device="cuda")
    for lens, start in (([2**31 - 1, 64], [0, 1, 2]), ([-5, -2**31], [0, 1, 2]), ([64, 64], [0, 1, 9000]), ([64, 64], [-7, 1, 2]), ([64, 64], [2, 1, 0]), ([64, 64], [0, 0, 0])):
        b = hip.KvBatch(torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.zeros_like(batch.pages), rows=2, row_start=torch.tensor(start, dtype=torch.int32, device="cuda"))
        be.kv_summarize(cache, b, held)
        be.kv_summary_read(cache, b, held, 2)
        be.kv_select(cache, b, held, q, 1, first=0, last=0, out=picks[4:8])
        be.attend_selected(cache, b, q, picks[4:8], 32, out=out[4:8])
        torch.cuda.synchronize()
        assert (out[:4] == 7).all() and (out[6:] == 7).all() and (picks[:4] == 77).all() and (picks[6:] == 77).all()


def test_all_spans_are_attention_over_everything(be):
    """Where there are no more spans than are taken, the pair is `attend`."""
    from oxinfer_amd import hip
    w = kv_ref.World([300, 100, 40], 2, 64, page=64, seed=6, n=[3, 1, 2])
    cache, batch = w.tensors(hip)
    held = be.kv_summary(cache, 32)
    q = torch.randn(w.rows, 4 * 64, device="cuda")
    chosen = be.kv_select(cache, batch, held, q, 10)
    got = be.attend_selected(cache, batch, q, chosen, 32)
    want, tol = kv_ref.attend(w, q.double().cpu().numpy().reshape(w.rows, 4, 64), 2, 64**-0.5)
    assert (np.abs(got.double().cpu().numpy().reshape(want.shape) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_by_a_recorded_plan(be, dtype):
    """Append, summarize, select and attend as a layer's step runs them, recorded once and replayed token by token with eager work between; every replay's
    cache, choice and result are held to the definitions."""
    from oxinfer_amd import hip
    rng = np.random.default_rng(0)
    n_kv, g, d, page, span, count = 2, 3, 64, 64, 32, 5
    lens = [500, 33, 255]
    w = kv_ref.World([x + 40 for x in lens], n_kv, d, page=page, seed=1)
    w.lens = np.array(lens)
    cache, batch = w.tensors(hip)
    batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    held = be.kv_summary(cache, span)
    code, scale = np.zeros(held.shape, np.int8), np.zeros(held.shape[:3], np.float32)
    start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    be.kv_summarize(cache, hip.KvBatch(batch.kv_len, batch.pages, rows=sum(lens), row_start=start), held)  # (the prompts')
    w.n = np.array(lens)
    lists_ref.summarize(w, span, code, scale)
    w.n = np.ones(3, int)
    k, v, q = (torch.randn(3, x * d, device="cuda").to(dtype) for x in (n_kv, n_kv, n_kv * g))
    out, chosen = torch.empty_like(q), torch.empty((3, n_kv, count), dtype=torch.int32, device="cuda")

    def step():
        be.kv_append(cache, batch, k, v)
        be.kv_summarize(cache, batch, held)
        be.kv_select(cache, batch, held, q, count, out=chosen)
        be.attend_selected(cache, batch, q, chosen, span, out=out)

    torch.cuda.synchronize()
    stream, plan = torch.cuda.Stream(), None
    with torch.cuda.stream(stream):
        for i in range(38):
            batch.kv_len += 1
            w.lens = w.lens + 1
            for t in (k, v, q):
                t.copy_(torch.from_numpy(rng.normal(size=t.shape)))
            if plan is None:
                step()
                stream.synchronize()
            else:
                plan.replay()
            stream.synchronize()
            h = lambda t: t.double().cpu().numpy().reshape(3, -1, d)  # noqa: E731
            kv_ref.append(w, h(k), h(v))
            lists_ref.summarize(w, span, code, scale)
            assert np.array_equal(held.code.cpu().numpy(), code) and np.array_equal(held.scale.cpu().numpy(), scale)
            want = lists_ref.select(w, h(q).astype(np.float32), g, span, code, scale, count, 1, 1)
            assert np.array_equal(chosen.cpu().numpy(), want)
            want, tol = lists_ref.attend_selected(w, h(q), g, d**-0.5, want, span, half=dtype is torch.bfloat16)
            assert (np.abs(h(out) - want) <= tol).all()
            if plan is None:
                plan = be.plan_record(step)
    del plan


def test_the_same_bits_on_any_stream(be):
    from oxinfer_amd import hip
    w = kv_ref.World([20000, 9000], 2, 128, page=64, seed=3)
    cache, batch = w.tensors(hip)
    held, _, _ = summary(be, w, hip, cache, 64, np.random.default_rng(1))
    q = torch.randn(2, 8 * 128, device="cuda")
    chosen = be.kv_select(cache, batch, held, q, 100)
    want = be.attend_selected(cache, batch, q, chosen, 64)
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(torch.cuda.Stream()):
            again = be.kv_select(cache, batch, held, q, 100)
            got = be.attend_selected(cache, batch, q, again, 64)
            torch.cuda.current_stream().synchronize()
            assert torch.equal(again, chosen) and torch.equal(got, want)


def test_recording_without_scratch_is_refused(be):
    from oxinfer_amd import hip
    w = kv_ref.World([300, 310], 1, 64, seed=3)
    cache, batch = w.tensors(hip)
    chosen = torch.zeros((2, 1, 3), dtype=torch.int32, device="cuda")
    q, out = torch.randn(2, 64, device="cuda"), torch.empty(2, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()), pytest.raises(RuntimeError, match="plan"):
        be.plan_record(lambda: be.attend_selected(cache, batch, q, chosen, 32, out=out))


def test_the_bindings_refusals(be):
    from oxinfer_amd import hip
    w = kv_ref.World([200, 200], 2, 64, page=64, seed=3)
    cache, batch = w.tensors(hip)
    held = be.kv_summary(cache, 64)
    q = torch.randn(2, 4 * 64, device="cuda")
    chosen = be.kv_select(cache, batch, held, q, 2)
    for bad in (dict(q=q.half()), dict(q=q[:1]), dict(q=q[:, : 3 * 64]), dict(count=0), dict(count=1, first=1, last=1), dict(first=-1), dict(out=chosen.float()), dict(out=chosen[:1]), dict(out=chosen[:, :1]), dict(count=10**6)):
        with pytest.raises((ValueError, RuntimeError)):
            be.kv_select(cache, batch, held, **(dict(q=q, count=2) | bad))
    for bad in (dict(q=q.half()), dict(chosen=chosen[:1]), dict(chosen=chosen[:, :1]), dict(chosen=chosen.long()), dict(chosen=chosen[0]), dict(span=16), dict(span=48), dict(span=128), dict(out=q), dict(chosen=chosen[:, :, :0])):
        with pytest.raises((ValueError, RuntimeError)):
            be.attend_selected(cache, batch, **(dict(q=q, chosen=chosen, span=64) | bad))
    for span in (16, 48, 128):
        with pytest.raises(ValueError):
            be.kv_summary(cache, span)
    other = be.kv_cache(w.n_pages + 1, 2, 64, page_tokens=64)
    with pytest.raises(ValueError):
        be.kv_summarize(other, batch, held)
    with pytest.raises(ValueError):
        hip.KvSummary(held.code.float(), held.scale, 64)


# ---- the choice over tables as large as they may be (scores of more LDS than a launch has unasked), by sixteen waves and by eight ------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 300])
def test_choice_over_the_largest_table(be, n, dtype):
    """16384 spans' room, one row (sixteen waves) and as many as eight waves each take."""
    w = kv_ref.World([524027], 1, 32, page=256, seed=n, n=[n])
    assert w.table.shape[1] * 256 // 32 == 16384
    for count, last in ((100, 1), (1, 0), (16000, 7)) if n == 1 else ((64, 2),):
        check_choice(be, w, 2, 32, count, first=min(count - 1, 3), last=last, dtype=dtype, ragged=n > 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spans", [4094, 4095, 4096, 4100])
def test_choice_where_scores_outgrow_a_launchs_own_lds(be, spans, dtype):
    """4096 spans' room in a table is 32 KiB of scores. One row and drafted ones."""
    for n in ([1], [6]):
        w = kv_ref.World([32 * spans - 7], 1, 64, page=32, seed=spans, n=n)
        check_choice(be, w, 3, 32, 40, dtype=dtype, ragged=n != [1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,lens", [(64, [32700, 33000, 20]), (64, [60000, 65000, 40000]), (96, [100000, 131000, 90]), (256, [33000, 32900, 40])])
def test_choice_for_drafted_rows_over_long_caches(be, d, lens, dtype):
    """Sixteen waves over up to four rows of a sequence each, heads of any size."""
    for n, g in (([5, 3, 1], 2), ([1, 9, 2], 5), ([2, 2, 2], 16)):
        check_choice(be, kv_ref.World(lens, 1, d, page=64, seed=d, n=n), g, 32, 33, last=2, dtype=dtype, ragged=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [160, 192, 224, 256])
def test_choice_of_wide_heads_for_one_token_of_a_long_cache(be, d, dtype):
    check_choice(be, kv_ref.World([33500], 2, d, page=128, seed=d), 4, 32, 50, dtype=dtype)


def test_choice_over_the_largest_table_by_a_recorded_plan(be):
    from oxinfer_amd import hip
    w = kv_ref.World([524027], 1, 32, page=256, seed=2)
    cache, batch = w.tensors(hip)
    held, code, scale = summary(be, w, hip, cache, 32, np.random.default_rng(1))
    q, out = torch.zeros(1, 64, device="cuda"), torch.empty((1, 1, 90), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        plan = be.plan_record(lambda: be.kv_select(cache, batch, held, q, 90, out=out))
        for length in (524027, 400000, 200, 524032):
            batch.kv_len.fill_(length)
            q.normal_()
            plan.replay()
            torch.cuda.current_stream().synchronize()
            w.lens = np.array([length])
            want = lists_ref.select(w, q.cpu().numpy().reshape(1, 2, 32), 2, 32, code, scale, 90, 1, 1)
            assert np.array_equal(out.cpu().numpy(), want)
    del plan
