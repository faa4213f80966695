"""The draw of next tokens against the same in 64 bits (lists_ref.sample): the token is the same, its log-probability within the roundings of f32."""
import numpy as np
import pytest
import torch

from tests.lists_ref import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def rules_of(t, rng, names):
    made = dict(temperature=rng.uniform(0.3, 1.5, t).astype(np.float32), top_k=rng.integers(0, 60, t).astype(np.int32), top_p=rng.uniform(0.2, 1.05, t).astype(np.float32), min_p=rng.uniform(-0.05, 0.3, t).astype(np.float32))
    return {k: made[k] for k in names}


def check(be, x, u, strided=False, **rules):
    """x: a torch tensor of logits on the device. logp: a weight is a whole number of 2^-unit of the largest (unit = 62 - log2 vocab, 46 at most), made of a series that is
    off by 2^-42 of it; so a share is off by 2^-41 of itself and, for itself and for the sum, by vocab such units, which are more of a small share; then
    one rounding to f32."""
    t, vocab = x.shape
    up = {k: torch.from_numpy(v).cuda() for k, v in rules.items()}
    got, logp = be.sample(x, torch.from_numpy(u).cuda(), **up)
    want, logs = sample(x.double().cpu().numpy(), u, **rules)
    assert got.tolist() == want.tolist()
    logp = logp.double().cpu().numpy()
    live = want >= 0
    assert (logp[~live] == -np.inf).all()
    unit = min(46, 62 - (vocab - 1).bit_length())
    with np.errstate(over="ignore"):
        share = 2.0**-unit * (1 + np.exp(-logs[live]))
    assert (np.abs(logp[live] - logs[live]) <= 2.0**-24 * np.abs(logs[live]) + vocab * share + 2.0**-41).all()
    return got


NAMES = ("temperature", "top_k", "top_p", "min_p")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4095, 4096, 4097, 32003, 128256])
@pytest.mark.parametrize("rows", [1, 5])
def test_sizes(be, rows, vocab, dtype):
    rng = np.random.default_rng(vocab + rows)
    x = torch.from_numpy(3 * rng.normal(size=(rows, vocab))).cuda().to(dtype)
    check(be, x, rng.random(rows).astype(np.float32), **rules_of(rows, rng, NAMES))


@pytest.mark.parametrize("names", [(), ("temperature",), ("top_k",), ("top_p",), ("min_p",), ("top_k", "top_p"), ("top_k", "min_p"), ("top_p", "min_p"), NAMES], ids=str)
@pytest.mark.parametrize("spread", [0.01, 1.0, 5.0, 100.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rules(be, names, spread, dtype):
    """Logits that hardly differ, ordinary ones, and ones of which one is all."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(spread * rng.normal(size=(40, 20011))).cuda().to(dtype)
    check(be, x, rng.random(40).astype(np.float32), **rules_of(40, rng, names))


def test_many_rows_and_shares(be):
    """The same row with random numbers from 0 to 1: each token comes as often as its weight says."""
    rng = np.random.default_rng(1)
    row = 2 * rng.normal(size=3001)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    x = torch.from_numpy(np.repeat(row[None], n, 0)).cuda().float()
    got = check(be, x, u, top_k=np.full(n, 50, np.int32), top_p=np.full(n, 0.8, np.float32)).cpu().numpy()
    assert (np.diff(got) >= 0).all()  # (in the order of the ids)
    w = np.exp(x[0].double().cpu().numpy())
    order = np.argsort(-w, kind="stable")[:50]
    kept = order[: 1 + int((np.cumsum(w[order])[:-1] < 0.8 * w[order].sum()).sum())]
    count = np.bincount(got, minlength=3001)
    share = np.zeros(3001)
    share[kept] = w[kept] / w[kept].sum()
    assert (np.abs(count - n * share) <= 1.001).all() and set(np.flatnonzero(count)) <= set(kept.tolist())


def test_equal_logits_go_by_their_ids(be):
    """Whole rows alike, and few different values, so that the limits fall among equal ones."""
    rng = np.random.default_rng(2)
    x = np.zeros((12, 9000))
    x[4:8] = rng.integers(-3, 3, (4, 9000))
    x[8:] = rng.integers(0, 2, (4, 9000)) * 1e-30
    u = np.linspace(0, 0.999, 12).astype(np.float32)
    for rules in (dict(), dict(top_k=np.full(12, 7, np.int32)), dict(top_k=np.full(12, 5000, np.int32)), dict(top_p=np.full(12, 0.3, np.float32)), dict(top_k=np.full(12, 100, np.int32), top_p=np.full(12, 0.255, np.float32)),
                  dict(min_p=np.full(12, 1.0, np.float32)), dict(min_p=np.full(12, 0.3, np.float32), top_k=np.full(12, 4000, np.int32))):
        for dtype in (torch.float32, torch.bfloat16):
            check(be, torch.from_numpy(x).cuda().to(dtype), u, **rules)


def test_values_a_hairs_breadth_apart(be):
    """f32 values next to each other, around zero and around a large one, that the limits tell apart."""
    rng = np.random.default_rng(2)
    near = np.float32(1000.0) + np.arange(-300, 300).astype(np.float32) * np.float32(2.0**-14)
    tiny = rng.integers(-300, 300, 600).astype(np.float32) * np.float32(1e-45)
    mixed = np.concatenate([tiny[:300], np.float32(8.0) + np.arange(300).astype(np.float32) * np.float32(2.0**-20)])
    x = torch.from_numpy(np.stack([rng.permutation(v) for v in (near, tiny, mixed)])).cuda()
    for k in (1, 2, 299, 300, 301, 450, 599):
        check(be, x, np.array([0.999, 0.5, 0.9999], np.float32), top_k=np.full(3, k, np.int32))
        check(be, x, np.array([0.1, 0.7, 0.99], np.float32), top_k=np.full(3, k, np.int32), temperature=np.array([1e-3, 1e30, 0.01], np.float32), top_p=np.full(3, 0.9, np.float32))


def test_temperatures_at_their_ends(be):
    rng = np.random.default_rng(4)
    heats = np.array([0.0, -1.0, np.nan, 1e-45, 1e-38, 1e-3, 1e3, 1e30, 3e38, np.inf, -0.0, -np.inf], np.float32)
    x = torch.from_numpy(3 * rng.normal(size=(12, 5000))).cuda().float()
    x[:, 77] = x.amax(1)  # (two best ones)
    for rules in (dict(), dict(top_k=np.full(12, 20, np.int32)), dict(top_p=np.full(12, 0.5, np.float32))):
        check(be, x, rng.random(12).astype(np.float32), temperature=heats, **rules)


def test_limits_at_their_ends(be):
    rng = np.random.default_rng(4)
    x = torch.from_numpy(3 * rng.normal(size=(10, 5000))).cuda().float()
    u = rng.random(10).astype(np.float32)
    check(be, x, u, top_p=np.array([0.0, -1.0, 1.0, 2.0, np.nan, 1e-30, 1 - 2.0**-24, np.inf, -np.inf, 0.5], np.float32))
    check(be, x, u, min_p=np.array([0.0, -1.0, 1.0, 2.0, np.nan, 1e-30, 1 - 2.0**-24, np.inf, -np.inf, 0.5], np.float32))
    check(be, x, u, top_k=np.array([0, -1, 1, 2, 4999, 5000, 5001, 2**31 - 1, -(2**31), 3], np.int32))
    for at in (0.0, 1e-45, 1 - 2.0**-24, 1.0, 2.0, -1.0, np.nan, np.inf):
        check(be, x, np.full(10, at, np.float32), top_k=np.full(10, 30, np.int32))
        check(be, x, np.full(10, at, np.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_and_nan(be, dtype):
    rng = np.random.default_rng(6)
    x = 3 * rng.normal(size=(9, 6000))
    x[0] = -np.inf
    x[1] = np.nan
    x[2, rng.permutation(6000)[:5990]] = -np.inf
    x[3, rng.permutation(6000)[:3000]] = np.nan
    x[4, [5, 900, 5999]] = np.inf
    x[5, :] = -np.inf
    x[5, 4321] = -3e38
    x[6, 10] = 3e38
    x[7] = rng.choice([-3e38, 3e38, 0.0], 6000)
    x[8, 0] = np.inf
    x[8, 1] = np.nan
    up = torch.from_numpy(x).cuda().to(dtype)
    for u in (0.0, 0.4, 0.9999):
        for rules in ({}, dict(top_k=np.full(9, 2, np.int32)), dict(top_p=np.full(9, 0.6, np.float32)), dict(min_p=np.full(9, 0.1, np.float32)), rules_of(9, rng, NAMES), dict(temperature=np.zeros(9, np.float32))):
            check(be, up, np.full(9, u, np.float32), **rules)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_addresses(be, dtype):
    rng = np.random.default_rng(7)
    flat = torch.from_numpy(3 * rng.normal(size=1 + 5 * 5017)).cuda().to(dtype)
    check(be, flat[: 5 * 5016].view(5, 5016)[:, :5000], rng.random(5).astype(np.float32), **rules_of(5, rng, NAMES))
    check(be, flat[1:].view(5, 5017)[:, :5003], rng.random(5).astype(np.float32), **rules_of(5, rng, NAMES))


def test_behind_the_logits_rules_by_a_recorded_plan(be):
    """Rules, then the draw, recorded once; replays over other logits and random numbers are the eager results, and tokens that a mask takes away never come."""
    rng = np.random.default_rng(8)
    t, vocab = 6, 40000
    x, out, u = torch.randn(t, vocab, device="cuda") * 3, torch.empty(t, vocab, device="cuda"), torch.rand(t, device="cuda")
    allowed = torch.from_numpy(rng.integers(-2**31, 2**31, (t, vocab // 32)).astype(np.int32)).cuda()
    rules = {k: torch.from_numpy(v).cuda() for k, v in rules_of(t, rng, NAMES).items()}
    kept = []

    def step():
        be.adjust_logits(x, out=out, want_next=False, allowed=allowed)
        kept.append(be.sample(out, u, **rules))

    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        plan = be.plan_record(step)
        held = kept[-1]
        for i in range(8):
            x.normal_(0, 3)
            u.uniform_()
            for a in held:
                a.fill_(0)
            plan.replay()
            stream.synchronize()
            got, logp = (a.clone() for a in held)
            step()
            stream.synchronize()
            assert torch.equal(got, kept[-1][0]) and torch.equal(logp, kept[-1][1])
            want, _ = sample(out.double().cpu().numpy(), u.cpu().numpy(), **{k: v.cpu().numpy() for k, v in rules.items()})
            assert got.tolist() == want.tolist()
            assert all(int(allowed[r, v // 32]) >> (v % 32) & 1 for r, v in enumerate(got.tolist()))
    del plan


def test_the_same_token_every_time(be):
    rng = np.random.default_rng(9)
    x = torch.from_numpy(2 * rng.normal(size=(16, 50000))).cuda().float()
    u = torch.rand(16, device="cuda")
    rules = {k: torch.from_numpy(v).cuda() for k, v in rules_of(16, rng, NAMES).items()}
    a, la = be.sample(x, u, **rules)
    for _ in range(20):
        with torch.cuda.stream(torch.cuda.Stream()):
            b, lb = be.sample(x, u, **rules)
            torch.cuda.current_stream().synchronize()
        assert torch.equal(a, b) and torch.equal(la, lb)
    assert be.sample(x, u, want_logp=False, **rules)[1] is None


def test_a_vocabulary_past_a_million(be):
    """More slices than sums are kept of."""
    rng = np.random.default_rng(12)
    x = torch.from_numpy(3 * rng.normal(size=(3, 1_100_003))).cuda().float()
    for names in ((), ("top_k",), ("top_p",), NAMES):
        check(be, x, rng.random(3).astype(np.float32), **rules_of(3, rng, names))
    check(be, x.bfloat16(), rng.random(3).astype(np.float32), top_k=np.array([1_000_000, 5, 0], np.int32), top_p=np.array([0.999, 1.0, 0.5], np.float32))


def test_more_rows_than_the_workspace_holds(be):
    """What a row draws is no matter of the rows beside it, nor of how many of them a launch takes."""
    rng = np.random.default_rng(13)
    x = 3 * torch.randn(900, 151936, device="cuda").bfloat16()
    u = torch.rand(900, device="cuda")
    rules = {k: torch.from_numpy(v).cuda() for k, v in rules_of(900, rng, NAMES).items()}
    got, logp = be.sample(x, u, **rules)
    for lo, hi in ((0, 1), (1, 40), (40, 170), (500, 570), (895, 900)):
        a, b = be.sample(x[lo:hi], u[lo:hi].contiguous(), **{k: v[lo:hi].contiguous() for k, v in rules.items()})
        assert torch.equal(a, got[lo:hi]) and torch.equal(b, logp[lo:hi])
    some = [0, 133, 450, 899]
    want, _ = sample(x[some].double().cpu().numpy(), u[some].cpu().numpy(), **{k: v[some].cpu().numpy() for k, v in rules.items()})
    assert got[some].tolist() == want.tolist()


def test_recording_without_scratch_is_refused(be):
    x, u = torch.randn(2, 300, device="cuda"), torch.rand(2, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()), pytest.raises(RuntimeError, match="plan"):
        be.plan_record(lambda: be.sample(x, u))


def test_threads_on_streams_of_their_own(be):
    import threading
    rng = np.random.default_rng(14)
    made = []
    for i in range(4):
        x, u = 3 * torch.randn(3 + 5 * i, 30000 + 7000 * i, device="cuda"), torch.rand(3 + 5 * i, device="cuda")
        rules = {k: torch.from_numpy(v).cuda() for k, v in rules_of(len(u), rng, NAMES).items()}
        made.append((x, u, rules, be.sample(x, u, **rules)))
    torch.cuda.synchronize()
    wrong = []

    def go(i):
        x, u, rules, want = made[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = be.sample(x, u, **rules)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])):
                    wrong.append(i)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_bindings_refusals(be):
    x, u = torch.randn(3, 100, device="cuda"), torch.rand(3, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (dict(logits=x.half()), dict(logits=x.cpu()), dict(u=u[:2]), dict(u=u.double()), dict(u=u.cpu()), dict(temperature=i), dict(top_k=u), dict(top_k=i[:2]), dict(top_p=u.double()), dict(min_p=u[:1]), dict(logits=x.t().contiguous().t())):
        with pytest.raises((ValueError, RuntimeError)):
            be.sample(**(dict(logits=x, u=u) | bad))
    assert be.sample(x[:0], u[:0])[0].shape == (0,)


def below(top, ulps):
    """The f32 value so many steps of f32 below `top`."""
    for _ in range(ulps):
        top = np.nextafter(np.float32(top), np.float32(-np.inf))
    return top


def test_small_temperatures_pass_no_limit_over(be):
    """Best logits over the temperature of 2^23 and more, where neighbouring f32 logits weigh what the limits tell apart."""
    x = np.full((2, 5000), -1e4, np.float32)
    top = np.float32(15.160547)
    x[:, 40] = top
    x[:, [10, 20, 30]] = below(top, 2)  # 0.148 of the best: top-p keeps one of them, and so does top-k
    up = torch.from_numpy(x).cuda()
    u, heat, least = np.full(2, 0.2, np.float32), np.full(2, 1e-6, np.float32), np.full(2, 0.1388, np.float32)
    assert check(be, up, u, temperature=heat, min_p=least, top_p=np.full(2, 0.75, np.float32)).tolist() == [40, 40]
    assert check(be, up, u, temperature=heat, min_p=least, top_k=np.full(2, 2, np.int32)).tolist() == [40, 40]
    # 2^-37 of the best: with top-k 2 one of them is left, and the random number lies between it and the next
    x[:] = -1e4
    top = np.float32(14.092963218688965)
    x[:, 3] = top
    x[:, :3] = below(top, 4)
    up = torch.from_numpy(x).cuda()
    heat = np.full(2, 1.4791656610668724e-07, np.float32)
    assert check(be, up, np.full(2, 600 * 2.0**-46, np.float32), temperature=heat, top_k=np.full(2, 2, np.int32)).tolist() == [3, 3]


def test_neighbouring_logits_at_any_temperature(be):
    rng = np.random.default_rng(21)
    t, vocab = 400, 6000
    heat = (10 ** rng.uniform(-8, -4, t)).astype(np.float32)
    x = np.full((t, vocab), -1e4, np.float32)
    least = np.zeros(t, np.float32)
    for r in range(t):
        top = np.float32(rng.uniform(1, 40) * rng.choice([1, 1, -1]))
        ids = rng.permutation(vocab)
        at = 0
        for ulps in (0, 1, 2, 3):
            n = int(rng.integers(1, 7)) if ulps else int(rng.integers(1, 3))
            x[r, ids[at : at + n]] = below(top, ulps)
            at += n
        w = np.exp((float(below(top, int(rng.integers(0, 4)))) - float(top)) / float(heat[r]))
        least[r] = w * rng.uniform(0.3, 0.98)
    up = torch.from_numpy(x).cuda()
    u, p, k = rng.uniform(0.001, 0.999, t).astype(np.float32), rng.uniform(0.2, 0.999, t).astype(np.float32), rng.integers(1, 12, t).astype(np.int32)
    for rules in (dict(top_p=p), dict(top_k=k), dict(min_p=least), dict(top_p=p, min_p=least), dict(top_k=k, min_p=least), dict(top_p=p, top_k=k), dict(top_p=p, top_k=k, min_p=least)):
        check(be, up, u, temperature=heat, **rules)


def test_top_k_behind_the_last_weight(be):
    """More tokens are asked for than weigh anything, and the last ones that do share a step of weight with some that do not: none is left out of the sum."""
    x = np.full((1, 9000), -1e4, np.float32)
    best = 0.5 / (4 / np.log(2))  # (in the middle of a step, as is then the weight of half a unit, 2^-47)
    at = lambda octaves: np.float32(best - octaves * np.log(2))  # noqa: E731
    x[0, :3000] = at(46.95)  # one unit
    x[0, 5100:8100] = at(47.05)  # none
    x[0, [5000, 8500]] = best
    # the middle of the whole lies between the two best ones, 1500 units before the end of the first
    assert check(be, torch.from_numpy(x).cuda(), np.array([0.5], np.float32), top_k=np.array([4000], np.int32)).tolist() == [5000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_top_k_of_the_whole_vocabulary_is_none(be, dtype):
    """Bit for bit what no top-k gives, beside rows that have one; of one token less the last of equal ones is left out."""
    rng = np.random.default_rng(16)
    x = (3 * torch.randn(12, 40003, device="cuda")).to(dtype)
    u = torch.rand(12, device="cuda")
    for names in ((), ("top_p",), ("min_p",), ("temperature", "top_p", "min_p")):
        rules = {k: torch.from_numpy(v).cuda() for k, v in rules_of(12, rng, names).items()}
        none = be.sample(x, u, **rules)
        for k in (40003, 40004, 2**31 - 1):
            got = be.sample(x, u, top_k=torch.full((12,), k, dtype=torch.int32, device="cuda"), **rules)
            assert all(torch.equal(a, b) for a, b in zip(got, none))
        some = torch.tensor([k for _ in range(4) for k in (40003, 7, 0)], dtype=torch.int32, device="cuda")
        got = be.sample(x, u, top_k=some, **rules)
        assert all(torch.equal(a[some != 7], b[some != 7]) for a, b in zip(got, none))
    flat = torch.zeros(2, 5000, device="cuda", dtype=dtype)
    assert check(be, flat, np.full(2, 0.99999, np.float32), top_k=np.array([4999, 5000], np.int32)).tolist() == [4998, 4999]
    assert check(be, flat[:, :1], np.zeros(2, np.float32), top_k=np.array([1, 5], np.int32)).tolist() == [0, 0]


@pytest.mark.parametrize("rows", [1, 64, 170, 256])
def test_tokens_set_apart_and_the_room_for_them(be, rows):
    """Slices of 4096 with 180 to 250 tokens above the limit's step and 10 to 300 in it, in launches of few rows and of as many as leave a slice room for about 256."""
    rng = np.random.default_rng(rows)
    vocab = 100_000
    v = np.arange(vocab) % 4096
    x = (0.02 * rng.normal(size=(rows, vocab))).astype(np.float32)
    above, at = rng.integers(180, 251, rows), rng.integers(10, 301, rows)
    x += np.where(v < above[:, None], 8, np.where(v < (above + at)[:, None], 7, 0)).astype(np.float32)
    up, u = torch.from_numpy(x).cuda(), rng.random(rows).astype(np.float32)
    w = np.exp(np.array([8.0, 7.0]))
    p = ((above * w[0] + at * w[1] * rng.uniform(0.1, 0.9, rows)) / (above * w[0] + at * w[1] + (4096 - above - at))).astype(np.float32)  # (falls among those of 7)
    k = ((above + (at * rng.uniform(0.1, 0.9, rows)).astype(int)) * (vocab // 4096)).astype(np.int32)
    least = np.exp(rng.uniform(-1.1, -0.9, rows)).astype(np.float32)
    for rules in (dict(top_p=p), dict(top_k=k), dict(top_p=p, min_p=least), dict(top_k=k, min_p=least), dict(top_k=k, top_p=p)):
        some = np.unique(rng.integers(0, rows, 12))
        got, logp = be.sample(up, torch.from_numpy(u).cuda(), **{n: torch.from_numpy(a).cuda() for n, a in rules.items()})
        few = check(be, up[torch.from_numpy(some).cuda()], u[some], **{n: a[some] for n, a in rules.items()})
        assert few.tolist() == got[torch.from_numpy(some).cuda()].tolist()
