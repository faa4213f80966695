"""Appending behind first tokens that another sequence holds, also where these end inside a block: a sequence's own tokens go into pages with whatever scales and codes their
former owners left, and cache and attention are those of the tokens that were given."""
import numpy as np
import pytest
import torch

from tests import kv_ref
from tests.lists_ref import Shared
from tests.test_gpu_kv_cache import angles

pytestmark = pytest.mark.gpu

STALE = np.array([np.nan, np.inf, 2.0**60, 30.0, 1.0, 2.0**-7, 2.0**-60, 0.0, -1.0], np.float32)


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


class World(Shared):
    """A cache of nothing but left-over codes and scales, and what its sequences' own tokens were given as: given[s] [2, length, n_kv, d]."""

    def __init__(self, room, group_start, common, n_kv, d, page, seed):
        super().__init__(room, group_start, common, n_kv, d, page=page, seed=seed)
        for a in (self.ks, self.vs):
            a[:] = self.rng.choice(STALE, a.shape)
        for a in (self.k, self.v):
            a[:] = self.rng.integers(0, 256, a.shape)
        self.given = [np.zeros((2, n, n_kv, d)) for n in room]
        self.touched = np.zeros((self.n_pages, self.per), bool)
        self.set(np.zeros(len(room), int), np.zeros(len(room), int))

    def set(self, lens, n):
        self.lens, self.n = np.asarray(lens), np.asarray(n)
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.rows = int(self.start[-1])

    def own(self, s):
        leader, common = self.shares(s)
        return 0 if leader == s else common

    def append(self, new):
        """new [2, rows, n_kv, d] f64: keys (rotated) and values."""
        for s in range(len(self.lens)):
            n, length, own = int(self.n[s]), int(self.lens[s]), self.own(s)
            before = length - n
            x = new[:, self.start[s] : self.start[s] + n]
            at = max(before, 0)
            self.given[s][:, at:length] = x[:, at - before :]
            for b in range(max(before, own, 0) // 32, -(-length // 32)):
                lo, hi = max(32 * b, before, own), min(32 * b + 32, length)
                if hi <= lo:
                    continue
                p, i = self.table[s, b // self.per], b % self.per
                self.touched[p, i] = True
                for codes, scales, off, y in zip((self.k, self.v), (self.ks, self.vs), kv_ref.offsets(self.d), x[:, lo - before : hi - before]):
                    old = off[max(own - 32 * b, 0) : lo - 32 * b]
                    for h in range(self.n_kv):
                        scale = need = max(float(np.float32(np.abs(y[:, h]).max() / 127)), kv_ref.FLOOR)
                        if len(old):
                            was = scale = float(scales[p, h, i])
                            while scale < need:
                                scale *= 2
                            codes[p, h, i][old] = np.rint((codes[p, h, i][old].astype(np.float64) - 128) * (was / scale)) + 128
                        scales[p, h, i] = scale
                        codes[p, h, i][off[lo - 32 * b : hi - 32 * b]] = np.rint(y[:, h] / scale) + 128

    def same(self, cache):
        for name, codes, scales, off in (("k", self.k, self.ks, kv_ref.offsets(self.d)[0]), ("v", self.v, self.vs, kv_ref.offsets(self.d)[1])):
            got, got_s = getattr(cache, name).cpu().numpy(), getattr(cache, name + "_scale").cpu().numpy()
            for s, length in enumerate(self.lens):
                own = self.own(s)
                for b in range(own // 32, -(-int(length) // 32)):
                    p, i = self.table[s, b // self.per], b % self.per
                    if not self.touched[p, i]:
                        continue
                    at = off[max(own - 32 * b, 0) : min(32, length - 32 * b)]
                    assert np.array_equal(got_s[p, :, i], scales[p, :, i]), (name, s, b)
                    assert np.array_equal(got[p, :, i][:, at], codes[p, :, i][:, at]), (name, s, b)
            for g, c in ((got, codes), (got_s, scales)):
                assert np.array_equal(g.transpose(0, 2, 1, *range(3, g.ndim))[~self.touched], c.transpose(0, 2, 1, *range(3, c.ndim))[~self.touched], equal_nan=c.dtype == np.float32)

    def tokens(self, s):
        leader, common = self.shares(s)
        return np.concatenate([self.given[leader][:, :common], self.given[s][:, common:]], 1)[:, : self.lens[s]] if leader != s else self.given[s][:, : self.lens[s]]

    def held_as_given(self):
        """What the cache holds is a scale from what was given at most, and no scale is twice what the block's own largest token asks for: nothing in it is of what was there before."""
        for s in range(len(self.lens)):
            for x, held, scales in zip(self.tokens(s), self.sequence(s), (self.ks, self.vs)):
                leader, common = self.shares(s)
                for b in range(-(-int(self.lens[s]) // 32)):
                    for lo, hi, whose in ((32 * b, min(32 * b + 32, common), leader), (max(32 * b, common if leader != s else 0), 32 * b + 32, s)):
                        if lo < min(hi, self.lens[s]):
                            by = scales[self.table[whose, b // self.per], :, b % self.per].astype(np.float64)
                            assert (np.abs(held[lo:hi] - x[lo:hi]) <= by[None, :, None] * (1 + 1e-12)).all()
                            first = max(self.own(whose), 32 * b)
                            most = np.abs(self.given[whose][0 if scales is self.ks else 1][first : 32 * b + 32]).max((0, 2)) / 127
                            assert (by <= 2 * most * (1 + 2.0**-23)).all()

    def attention(self, q, g, scale, half):
        """(out, bound): the attention over the tokens as they were given; the bound adds to that of kv_ref (over what is held) what a scale's error in each key and value makes of
        a score (d |q| s, twice in a weight) and of a result."""
        want, tol = kv_ref.attend(self, q, g, scale, half=half)
        out, far = np.zeros_like(want), np.zeros_like(want)
        for s in range(len(self.lens)):
            (k, v), (hk, hv) = self.tokens(s), self.sequence(s)
            for i in range(int(self.n[s])):
                r, pos = int(self.start[s]) + i, int(self.lens[s] - self.n[s]) + i
                for h in range(q.shape[1]):
                    j = slice(0, pos + 1)
                    x = scale * (k[j, h // g] @ q[r, h])
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[r, h] = p @ v[j, h // g]
                    ds = np.abs(scale) * np.abs(hk[j, h // g] - k[j, h // g]) @ np.abs(q[r, h])
                    dv = np.abs(hv[j, h // g] - v[j, h // g])
                    far[r, h] = (np.exp(2 * ds.max()) - 1) * (p @ np.abs(v[j, h // g]) + np.abs(out[r, h])) + np.exp(2 * ds.max()) * (p @ dv)
        return want, tol, out, tol + far


def step(be, w, cache, pages, shared, lens, n, rng, tt, g, ragged, rope=None, table=None, loud=1.0, look=True):
    from oxinfer_amd import hip
    w.set(lens, n)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()  # noqa: E731
    batch = hip.KvBatch(up(w.lens), pages, rows=w.rows if ragged else None, row_start=up(w.start) if ragged else None)
    kw, qw = w.n_kv * w.d, w.n_kv * g * w.d
    k, v, q = (torch.from_numpy(loud * rng.normal(size=(w.rows, c))).to("cuda", tt) for c in (kw, kw, qw))
    q_out = torch.full_like(q, 9.0)
    be.kv_append(cache, batch, k, v, q=q, q_out=q_out, rope=rope, shared=shared)
    out = be.attend_shared(cache, batch, shared, q_out)
    torch.cuda.synchronize()
    h = lambda t: t.double().cpu().numpy().reshape(w.rows, -1, w.d)  # noqa: E731
    pos = np.concatenate([w.lens[s] - w.n[s] + np.arange(w.n[s]) for s in range(len(w.lens))])
    hk, hq = (kv_ref.rotate(h(t), pos, table, False) if rope else h(t) for t in (k, q))
    assert (np.abs(h(q_out) - hq) <= torch.finfo(tt).eps / 2 * np.abs(hq) * (1 + 2.0**-16) + 1e-45).all()
    w.append(np.stack([hk, h(v)]))
    w.same(cache)
    if look:
        w.held_as_given()
        want, tol, given, far = w.attention(h(q_out), g, w.d**-0.5, tt is torch.bfloat16)
        assert (np.abs(h(out) - want) <= tol).all()
        assert (np.abs(h(out) - given) <= far).all()


def begin(be, w):
    from oxinfer_amd import hip
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    cache = hip.KvCache(up(w.k), up(w.v), up(w.ks), up(w.vs), w.page, w.d)
    return cache, up(w.table), hip.KvShared(up(w.group_start), up(w.common))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("common,page", [(1, 32), (31, 32), (32, 64), (53, 64), (63, 32), (100, 64), (127, 256)])
@pytest.mark.parametrize("ragged", [False, True])
def test_token_by_token(be, ragged, common, page, dtype):
    """Answers of three sequences behind a prompt that a first one keeps, and of one that shares nothing, whose tokens grow; the first tokens also a little smaller than those left over."""
    rng = np.random.default_rng(common)
    w = World([common + 80, common + 70, common + 75, common + 71, 80], [0, 4], [common], 2, 64, page, common)
    cache, pages, shared = begin(be, w)
    lens = np.array([common, common, common, common, 0])
    step(be, w, cache, pages, shared, lens, [common, 0, 0, 0, 0], rng, dtype, 2, True, look=False)
    for i in range(70):
        if ragged:
            n = np.array([0, 1, i % 3 != 1, i % 2, 1]) if i else np.array([0, 1, 2, 1, 1])
        else:  # (the first sequence has a row too, its own behind the shared ones)
            n = np.ones(5, int)
        lens = lens + n
        step(be, w, cache, pages, shared, lens, n, rng, dtype, 2, ragged, loud=np.exp(0.05 * i), look=i % 9 == 0 or lens[1] % 32 < 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
def test_chunks(be, d, dtype):
    """Rows of several blocks, of a block in part, before the own tokens and across their first one (of the first kind only the queries are rotated), several groups, the first sequence's
    own tokens in the block that the shared ones end in."""
    rng = np.random.default_rng(d)
    room = [300, 260, 280, 200, 150, 170, 90]
    w = World(room, [0, 3, 5], [75, 45], 2, d, 64, d)
    cache, pages, shared = begin(be, w)
    table = angles(400, 32)
    from oxinfer_amd import hip
    rope = hip.Rope(torch.from_numpy(table).cuda())
    go = lambda lens, n, **more: step(be, w, cache, pages, shared, lens, n, rng, dtype, 3, True, rope, table, **more)  # noqa: E731
    go([75, 0, 0, 45, 0, 10, 0], [75, 0, 0, 45, 0, 10, 0], look=False)
    go([75, 70, 60, 45, 12, 10, 3], [0, 20, 60, 0, 12, 0, 3])  # (nothing of sequences 1, 2 and 4 is stored)
    go([90, 100, 76, 45, 54, 10, 3], [15, 30, 16, 0, 42, 0, 0])
    go([91, 200, 80, 120, 55, 100, 40], [1, 100, 4, 75, 1, 90, 37], loud=3.0)
    go([300, 260, 280, 200, 150, 170, 90], [209, 60, 200, 80, 95, 70, 50], loud=0.5)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("groups", [1, 63, 64, 65, 300])
def test_many_groups(be, groups, ragged):
    """Groups of two, some that share nothing, some without sequences; sequences behind all groups."""
    rng = np.random.default_rng(groups)
    n_seqs = 2 * groups + 3
    start = np.sort(np.concatenate([2 * np.arange(groups + 1), rng.integers(0, 2 * groups, groups // 10)]))
    common = rng.integers(0, 40, len(start) - 1)
    w = World([64] * n_seqs, start, common, 1, 32, 32, groups)
    cache, pages, shared = begin(be, w)
    lens = np.array([max(w.shares(s)[1], 1) for s in range(n_seqs)])
    step(be, w, cache, pages, shared, lens, np.where([w.own(s) for s in range(n_seqs)], 0, lens), rng, torch.float32, 2, True, look=False)
    for i in range(3):
        lens = lens + 1
        step(be, w, cache, pages, shared, lens, np.ones(n_seqs, int), rng, torch.float32, 2, ragged, look=i == 2)


def test_single_tokens_before_the_own_ones(be):
    w = World([64, 64], [0, 2], [40], 2, 64, 32, 1)
    cache, pages, shared = begin(be, w)
    rng = np.random.default_rng(0)
    step(be, w, cache, pages, shared, [40, 0], [40, 0], rng, torch.float32, 1, True, look=False)
    for length in (1, 20, 40, 41, 42):
        step(be, w, cache, pages, shared, [40 + (length > 40), length], [1, 1], rng, torch.float32, 1, False, look=length > 40)


def test_recorded(be):
    """One plan for all steps: the lengths, and with them which block begins anew, are read on the device."""
    from oxinfer_amd import hip
    common, n = 45, 4
    w = World([common + 60] * n, [0, n], [common], 2, 64, 32, 5)
    cache, pages, shared = begin(be, w)
    rng = np.random.default_rng(3)
    step(be, w, cache, pages, shared, [common] * n, [common] + [0] * (n - 1), rng, torch.bfloat16, 2, True, look=False)
    kv_len = torch.full((n,), common, dtype=torch.int32, device="cuda")
    batch = hip.KvBatch(kv_len, pages)
    k, v, q = (torch.zeros(n, c, device="cuda", dtype=torch.bfloat16) for c in (128, 128, 256))
    out = torch.empty_like(q)

    def layer():
        be.kv_append(cache, batch, k, v, shared=shared)
        be.attend_shared(cache, batch, shared, q, out=out)

    plan = None
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for i in range(40):
            kv_len += 1
            for t in (k, v, q):
                t.normal_(0, 1 + 0.1 * i)
            layer() if plan is None else plan.replay()
            torch.cuda.current_stream().synchronize()
            w.set([common + 1 + i] * n, [1] * n)
            h = lambda t: t.double().cpu().numpy().reshape(n, -1, 64)  # noqa: E731
            w.append(np.stack([h(k), h(v)]))
            w.same(cache)
            if i % 8 == 0:
                w.held_as_given()
            want, tol = kv_ref.attend(w, h(q), 2, 0.125, half=True)
            assert (np.abs(h(out) - want) <= tol).all()
            if plan is None:
                plan = be.plan_record(layer)
    del plan


def test_the_bindings_refusals(be):
    from oxinfer_amd import hip
    w = World([64, 64], [0, 2], [40], 2, 64, 32, 1)
    cache, pages, shared = begin(be, w)
    batch = hip.KvBatch(torch.tensor([41, 41], dtype=torch.int32, device="cuda"), pages)
    k = torch.zeros(2, 128, device="cuda")
    for bad in (dict(shared=hip.KvShared(torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")), k=k[:1]), dict(k=k.half()), dict(q_out=k)):
        with pytest.raises(ValueError):
            be.kv_append(**(dict(cache=cache, batch=batch, k=k, v=k, shared=shared) | bad))
    with pytest.raises(ValueError):
        hip.KvShared(torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
