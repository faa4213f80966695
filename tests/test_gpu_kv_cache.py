"""Filling the 8-bit cache and reading it back, against the definition in 64 bits (kv_ref): codes and scales bit for bit."""
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


def angles(n_pos, n_rot, seed=0):
    a = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(n_rot // 2) / (n_rot / 2))
    return np.stack([np.cos(a), np.sin(a)], 2).astype(np.float32)


def same_cache(w, cache):
    """Codes of held tokens and scales of their blocks; every other byte's block is still what it was where no token came."""
    for name, codes, scales, off in (("k", w.k, w.ks, kv_ref.offsets(w.d)[0]), ("v", w.v, w.vs, kv_ref.offsets(w.d)[1])):
        got, got_s = getattr(cache, name).cpu().numpy(), getattr(cache, name + "_scale").cpu().numpy()
        for s, length in enumerate(w.lens):
            for b in range(-(-int(length) // 32)):
                p, i = w.table[s, b // w.per], b % w.per
                if not 0 <= p < w.n_pages:
                    continue
                at = off[: min(32, length - 32 * b)]
                assert np.array_equal(got_s[p, :, i], scales[p, :, i]), (name, s, b)
                assert np.array_equal(got[p, :, i][:, at], codes[p, :, i][:, at]), (name, s, b)
        used = np.zeros((w.n_pages, w.per), bool)
        for s, length in enumerate(w.lens):
            for b in range(-(-int(length) // 32)):
                if 0 <= w.table[s, b // w.per] < w.n_pages:
                    used[w.table[s, b // w.per], b % w.per] = True
        for g, c in ((got, codes), (got_s, scales)):
            assert np.array_equal(g.transpose(0, 2, 1, *range(3, g.ndim))[~used], c.transpose(0, 2, 1, *range(3, c.ndim))[~used], equal_nan=c.dtype == np.float32)


def check(be, w, g=2, dtype="f32", rot=None, interleaved=False, ragged=None, scale=1.0, strided=0, inplace=False, seed=7, n_pos=None, change=None):
    from oxinfer_amd import hip
    rng = np.random.default_rng(seed)
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    rot = w.d if rot is None else rot
    cache, batch = w.tensors(hip, ragged=ragged, extra_rows=2)
    rows, kw, qw = w.rows + 2, w.n_kv * w.d, w.n_kv * g * w.d
    x = torch.from_numpy(scale * rng.normal(size=(rows, 2 * kw + qw + strided))).to("cuda", tt)
    if change:
        change(x)
    k, v, q = x[:, :kw], x[:, kw : 2 * kw], x[:, 2 * kw : 2 * kw + qw]
    if not strided:
        k, v, q = (t.contiguous() for t in (k, v, q))
    table = angles(n_pos or int(max(w.lens.max(), 1)) + 1, rot) if rot else None
    rope = hip.Rope(torch.from_numpy(table).cuda(), interleaved) if rot else None
    hk, hv, hq = (t.double().cpu().numpy()[: w.rows] for t in (k, v, q))
    q_out = q if inplace else torch.full((rows, qw), 9.0, dtype=tt, device="cuda")
    tail = q_out[w.rows :].clone()
    be.kv_append(cache, batch, k, v, q=q, rope=rope, q_out=q_out)
    torch.cuda.synchronize()
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(len(w.lens))]).astype(int)
    hk, hv, hq = (t.reshape(w.rows, -1, w.d) for t in (hk, hv, hq))
    if rot:
        there = (pos >= 0) & (pos < len(table))
        for t in (hk, hq):
            t[there] = kv_ref.rotate(t[there], pos[there], table, interleaved)
            t[~there, :, :rot] = np.nan
    kv_ref.append(w, hk, hv)
    same_cache(w, cache)
    got = q_out.double().cpu().numpy()[: w.rows].reshape(hq.shape)
    sound = pos >= 0  # (rows before a sequence's first token are left out)
    half = torch.finfo(tt).eps / 2
    with np.errstate(invalid="ignore"):
        off = np.abs(got - hq)[sound]
        assert ((off <= half * np.abs(hq[sound]) * (1 + 2.0**-16) + 1e-45) | (np.isnan(hq[sound]) & np.isnan(got[sound]))).all()
    assert torch.equal(q_out[w.rows :], tail), "rows behind the last sequence were written"
    return cache, batch


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", range(32, 257, 32))
def test_head_sizes(be, d, dtype):
    check(be, kv_ref.World([5, 40, 32, 1], 2, d, seed=d), dtype=dtype)
    check(be, kv_ref.World([50, 90], 2, d, page=64, seed=d, n=[50, 33]), dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,lens", [([1], [1]), ([1, 1, 1], [32, 33, 64]), ([3, 0, 9], [10, 7, 40]), ([8, 9, 31], [31, 32, 33]), ([100, 65, 2, 33], [100, 70, 300, 64]), ([32, 64], [64, 64]), ([7, 2], [3, 0])])
def test_where_rows_begin_and_end(be, n, lens, dtype):
    for g, page in ((1, 32), (3, 128)):
        check(be, kv_ref.World(lens, 2, 64, page=page, seed=len(n), n=n), g, dtype, ragged=True)


@pytest.mark.parametrize("rot,interleaved", [(0, False), (64, True), (64, False), (32, False), (32, True), (6, False), (2, True)])
def test_rotations(be, rot, interleaved):
    for n in ([1, 1], [40, 3]):
        check(be, kv_ref.World([40, 70], 2, 64, seed=rot, n=n), rot=rot, interleaved=interleaved)
        check(be, kv_ref.World([40, 70], 1, 64, seed=rot, n=n), rot=rot, interleaved=interleaved, inplace=True)
    check(be, kv_ref.World([40, 70], 3, 96, seed=rot, n=[40, 3]), rot=rot, interleaved=interleaved, inplace=True, strided=8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strided", [8, 5])
def test_strides_and_addresses(be, strided, dtype):
    """Rows of a fused q / k / v buffer; with an odd stride none but the first begins at a multiple of 16 bytes."""
    for n in ([1, 1], [33, 12]):
        check(be, kv_ref.World([40, 70], 2, 64, seed=3, n=n), dtype=dtype, strided=strided)
        check(be, kv_ref.World([40, 70], 2, 64, seed=3, n=n), dtype=dtype, strided=strided, inplace=True)


def test_positions_past_the_table(be):
    for n in ([1, 1], [30, 40]):
        check(be, kv_ref.World([40, 70], 2, 64, seed=3, n=n), n_pos=35)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-18, 1e-4, 1e8, 3e20])
def test_values_of_any_size(be, scale):
    """The scale's floor and its growth from there, what is cut, all zeros."""
    for n in ([1, 1], [50, 9]):
        w = kv_ref.World([50, 75], 2, 64, seed=4, n=n)
        check(be, w, scale=scale)
        check(be, w, scale=1e3 * scale if scale < 1e9 else scale, seed=9)


def test_infinities_and_nan(be):
    def change(x):
        x[0, 3] = float("nan")
        x[1, 9] = float("inf")
        x[2, 130] = float("-inf")
        x[3, 128:192] = float("nan")
    for n in ([1, 1, 1, 1], [9, 9, 9, 9]):
        check(be, kv_ref.World([50, 75, 9, 40], 2, 64, seed=4, n=n), rot=0, change=change)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_by_token(be, dtype):
    """A block filled by 70 calls whose values grow: no code is further than a scale from its value, and the cache is the definition's."""
    from oxinfer_amd import hip
    rng = np.random.default_rng(0)
    w = kv_ref.World([70, 70], 2, 64, page=64, seed=1, wild=False)
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    cache, _ = w.tensors(hip)
    grow = np.exp(0.08 * np.arange(70))[:, None, None]
    x = torch.from_numpy(rng.normal(size=(70, 2, 4 * 64)) * grow * np.exp(rng.normal(size=(70, 2, 1)))).to("cuda", tt)
    pages = torch.from_numpy(w.table).cuda()
    kv_len = torch.zeros(2, dtype=torch.int32, device="cuda")
    batch = hip.KvBatch(kv_len, pages)
    for t in range(70):
        kv_len.fill_(t + 1)
        be.kv_append(cache, batch, x[t, :, :128], x[t, :, 128:])
        w.lens = np.array([t + 1, t + 1])
        h = x[t].double().cpu().numpy()
        kv_ref.append(w, h[:, :128].reshape(2, 2, 64), h[:, 128:].reshape(2, 2, 64))
    same_cache(w, cache)
    k, v = be.kv_read(cache, batch, 70)
    want = x.double().transpose(0, 1)
    for got, exact, scale in ((k, want[..., :128], cache.k_scale), (v, want[..., 128:], cache.v_scale)):
        off = (got.double() - exact.reshape(2, 70, 2, 64)).abs().amax(-1)
        for s in range(2):
            for b in range(3):
                at = scale[w.table[s, b // 2], :, b % 2].double()
                assert (off[s, 32 * b : 32 * b + 32] <= at * (1 + 1e-6)).all()


def test_appending_again_at_the_same_place(be):
    """A call repeated on the same lengths leaves the cache as it is (drafted tokens that are replaced)."""
    from oxinfer_amd import hip
    w = kv_ref.World([45, 70], 2, 64, seed=1, n=[3, 40])
    cache, batch = check(be, w)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.normal(size=(w.rows + 2, 8 * 64))).to("cuda", torch.float32)
    k, v = (x[:, i * 128 : (i + 1) * 128].contiguous() for i in range(2))
    rope = hip.Rope(torch.from_numpy(angles(71, 64)).cuda())
    be.kv_append(cache, batch, k, v, rope=rope)
    for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_pages_outside_the_cache_are_not_written(be):
    for n in ([1, 1], [50, 75]):
        w = kv_ref.World([50, 75], 2, 64, seed=1, n=n)
        w.table[0, 1], w.table[1, 2] = -1, w.n_pages
        check(be, w)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 64, 100, 300])
def test_reading_back(be, count, dtype):
    from oxinfer_amd import hip
    tt = torch.bfloat16 if dtype == "bf16" else torch.float32
    for d, page in ((64, 32), (96, 128), (256, 64)):
        w = kv_ref.World([64, 0, 97, 1, 200], 2, d, page=page, seed=count)
        cache, batch = w.tensors(hip)
        got = be.kv_read(cache, batch, count, dtype=tt)
        for s in range(5):
            for x, exact in zip(got, w.sequence(s)):
                m = min(count, int(w.lens[s]))
                want = np.zeros((count, 2, d))
                want[count - m :] = exact[int(w.lens[s]) - m :]
                half = torch.finfo(tt).eps / 2
                assert (np.abs(x[s].double().cpu().numpy() - want) <= half * np.abs(want)).all()
    w = kv_ref.World([64, 97], 2, 64, seed=count)
    w.table[1, 2] = -1
    cache, batch = w.tensors(hip)
    k, _ = be.kv_read(cache, batch, 97)
    assert k[1, 64:96].isnan().all() and not k[1, :64].isnan().any() and not k[0].isnan().any()


def test_the_bindings_refusals(be):
    from oxinfer_amd import hip
    w = kv_ref.World([64, 9], 2, 64, seed=3)
    cache, batch = w.tensors(hip)
    k = torch.randn(2, 128, device="cuda")
    for bad in (dict(k=k.half()), dict(v=k.bfloat16()), dict(k=k[:1]), dict(v=k[:, :64]), dict(q=k.bfloat16()), dict(q_out=k), dict(q=k, q_out=k[:, :64])):
        with pytest.raises((ValueError, RuntimeError)):
            be.kv_append(cache, batch, **(dict(k=k, v=k) | bad))
    with pytest.raises(ValueError):
        be.kv_read(cache, batch, 4, dtype=torch.float16)
    new = be.kv_cache(3, 2, 64, page_tokens=128)
    assert new.k.shape == (3, 2, 4, 2048) and be.kv_read(new, hip.KvBatch(batch.kv_len, torch.zeros((2, 1), dtype=torch.int32, device="cuda")), 9)[0].abs().max() == 0


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("n,lens", [([1, 1, 1], [0, 5, 0]), ([7, 2, 40], [3, 0, 40])])
def test_queries_before_the_first_token_are_left_as_they_are(be, n, lens, inplace):
    from oxinfer_amd import hip
    w = kv_ref.World(lens, 2, 64, seed=1, n=n)
    cache, batch = w.tensors(hip)
    k = torch.randn(w.rows, 128, device="cuda")
    q = torch.randn(w.rows, 256, device="cuda")
    out = q if inplace else torch.full_like(q, 9.0)
    was = out.clone()
    be.kv_append(cache, batch, k, k, q=q, q_out=out, rope=hip.Rope(torch.from_numpy(angles(50, 64)).cuda()))
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(3)])
    assert torch.equal(out[torch.from_numpy(pos < 0).cuda()], was[torch.from_numpy(pos < 0).cuda()]) and not (out == was)[torch.from_numpy(pos > 0).cuda()].all()
