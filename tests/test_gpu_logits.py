"""Penalties, biases and grammar masks on logits, and the best token, against the same in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def make(t, vocab, most=60, seed=0, biases=7, masks=True):
    """Arguments on the host: histories with ids outside the vocabulary, biases that name an id twice and one that is infinite."""
    r = np.random.default_rng(seed)
    a = dict(history=r.integers(-3, vocab + 3, (t, most)).astype(np.int32))
    a["history"][:, ::3] = r.integers(0, min(vocab, 5), a["history"][:, ::3].shape)
    a["history_len"] = r.integers(0, most + 1, t).astype(np.int32)
    a["history_len"][0] = most
    a["prompt_len"] = r.integers(0, most // 2 + 1, t).astype(np.int32)
    for n, lo, hi in (("repetition", 0.8, 1.4), ("presence", -0.5, 1), ("frequency", 0, 0.5)):
        a[n] = r.uniform(lo, hi, t).astype(np.float32)
    if biases:
        count = r.integers(0, biases + 1, t)
        count[0] = biases
        a["bias_start"] = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
        n = int(count.sum())
        a["bias_id"] = r.integers(-1, vocab + 1, n).astype(np.int32)
        a["bias_id"][: biases : 2] = a["bias_id"][0]
        a["bias"] = (4 * r.normal(size=n)).astype(np.float32)
        a["bias"][n // 2] = -np.inf
    if masks:
        a["allowed"] = r.integers(-2**31, 2**31, (3, (vocab + 31) // 32 + 1)).astype(np.int32)
        a["allowed_row"] = r.integers(-1, 3, t).astype(np.int32)
    return a


def plain(x, a):
    """(values in f64, how far each may be off before its rounding to the output's type): one rounding (u = 2^-24) of what each step forms."""
    x = x.astype(np.float64).copy()
    tol = np.zeros_like(x)
    t, vocab = x.shape
    u = 2.0**-24
    for r in range(t):
        if any(k in a for k in ("repetition", "presence", "frequency")):
            said = a["history"][r, : max(0, min(int(a["history_len"][r]), a["history"].shape[1]))]
            new = said[int(a["prompt_len"][r]) if "prompt_len" in a else 0 :]
            ok = lambda v: v[(v >= 0) & (v < vocab)]  # noqa: E731
            for i in np.unique(ok(said)):
                p = float(a["repetition"][r]) if "repetition" in a else 1.0
                x[r, i] = x[r, i] / p if x[r, i] > 0 else x[r, i] * p
                tol[r, i] += u * abs(x[r, i])
            ids, n = np.unique(ok(new), return_counts=True)
            f, p = (float(a[k][r]) if k in a else 0.0 for k in ("frequency", "presence"))
            tol[r, ids] += u * (f * n) + u * (np.abs(x[r, ids]) + 2 * f * n) + u * (np.abs(x[r, ids]) + f * n + abs(p)) * 2
            x[r, ids] -= f * n + p
        if "bias_start" in a:
            last = {}
            for e in range(int(a["bias_start"][r]), int(a["bias_start"][r + 1])):
                last[int(a["bias_id"][e])] = float(a["bias"][e])
            for i, b in last.items():
                if 0 <= i < vocab:
                    x[r, i] += b
                    tol[r, i] += 2 * u * (abs(x[r, i]) if np.isfinite(x[r, i]) else 0)
        if "allowed" in a:
            m = int(a["allowed_row"][r]) if "allowed_row" in a else r
            if m >= 0:
                bits = np.unpackbits(a["allowed"][m].view(np.uint8), bitorder="little")[:vocab] if m < len(a["allowed"]) else np.zeros(vocab)
                x[r, bits == 0] = -np.inf
    return x, tol


def check(be, logits, a, strided=0, inplace=False, **how):
    up = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    t, vocab = logits.shape
    wide = torch.full((t, vocab + strided), 3.25, dtype=logits.dtype, device="cuda")
    wide[:, :vocab] = logits
    x = wide[:, :vocab]
    want, tol = plain(logits.double().cpu().numpy(), a)
    out, best = be.adjust_logits(x, out=x if inplace else None, **up, **how)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    half = torch.finfo(logits.dtype).eps / 2 if logits.dtype == torch.bfloat16 else 0.0
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    f = np.isfinite(want)
    assert (np.abs(got[f] - want[f]) <= tol[f] * (1 + half) + half * np.abs(want[f])).all()
    assert (wide[:, vocab:] == 3.25).all()
    for r in range(t):  # the best of the values that came out: the lowest id of equal ones, none of nothing
        row = got[r]
        live = row > -np.inf
        assert int(best[r]) == (int(np.flatnonzero(row == row[live].max())[0]) if live.any() else -1)
    return got, best


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,vocab", [(1, 1), (1, 7), (3, 33), (2, 1000), (5, 4095), (5, 4096), (5, 4097), (4, 32003), (1, 151936), (70, 300)])
def test_sizes(be, t, vocab, dtype):
    x = (3 * torch.randn(t, vocab, generator=torch.Generator().manual_seed(t))).cuda().to(dtype)
    check(be, x, make(t, vocab, seed=vocab))
    check(be, x, make(t, vocab, seed=vocab + 1), inplace=True)


@pytest.mark.parametrize("names", [("repetition",), ("presence",), ("frequency",), (), ("repetition", "prompt_len"), ("frequency", "prompt_len")], ids=str)
@pytest.mark.parametrize("biases,masks", [(0, False), (5, False), (0, True)])
def test_single_rules(be, names, biases, masks):
    a = make(6, 500, biases=biases, masks=masks)
    for k in ("repetition", "presence", "frequency", "prompt_len"):
        if k not in names:
            del a[k]
    if not names:
        del a["history"], a["history_len"]
    check(be, torch.randn(6, 500, device="cuda"), a)


@pytest.mark.parametrize("most", [1, 255, 256, 257, 5000, 20000])
def test_long_histories(be, most):
    check(be, torch.randn(3, 5000, device="cuda"), make(3, 5000, most=most, biases=300, seed=most))


@pytest.mark.parametrize("split", [(0, 0), (4096, 512), (4200, 600), (5000, 700)])
def test_slices_that_only_some_rules_reach(be, split):
    """Histories and biases that lie in one slice of the vocabulary at first, and in others behind their first entries."""
    r = np.random.default_rng(7)
    hist, bias = np.empty((2, 5000), np.int32), np.empty(1400, np.int32)
    hist[:, : split[0]], hist[:, split[0] :] = r.integers(0, 4096, (2, split[0])), r.integers(4096, 8192, (2, 5000 - split[0]))
    ids = r.integers(12288, 16384, (2, 700))
    ids[:, : split[1]] = r.integers(0, 4096, (2, split[1]))
    bias[:] = ids.reshape(-1)
    a = dict(history=hist, history_len=np.array([5000, 4500], np.int32), prompt_len=np.array([10, 4400], np.int32), repetition=np.array([1.3, 0.9], np.float32),
             presence=np.array([0.5, -0.25], np.float32), frequency=np.array([0.01, 0.25], np.float32), bias_start=np.array([0, 700, 1400], np.int32), bias_id=bias,
             bias=r.normal(size=1400).astype(np.float32))
    check(be, torch.from_numpy(r.normal(size=(2, 17000)).astype(np.float32)).cuda(), a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("strided", [1, 8])
def test_strides(be, strided, dtype):
    x = torch.randn(4, 4100, device="cuda").to(dtype)
    check(be, x, make(4, 4100), strided=strided)
    check(be, x, make(4, 4100), strided=strided, inplace=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_nan_and_equal_values(be, dtype):
    x = torch.randint(-2, 3, (6, 9000), device="cuda").to(dtype)
    x[0, 5] = float("nan")
    x[1, 8999] = float("inf")
    x[2, :] = float("-inf")
    x[3, :] = float("nan")
    x[4, :] = -0.0
    x[4, 7000:] = 0.0
    x[5, :] = torch.finfo(dtype).min
    check(be, x, dict())
    check(be, x, {k: v for k, v in make(6, 9000).items() if not k.startswith("bias")})


def test_masks_that_allow_nothing_and_masks_that_are_not_there(be):
    a = make(5, 700, biases=0)
    a["allowed"][0] = 0
    a["allowed_row"] = np.array([0, 1, -1, 3, 2**31 - 1], np.int32)
    _, best = check(be, torch.randn(5, 700, device="cuda"), a)
    assert best.tolist()[0] == -1 and best.tolist()[3:] == [-1, -1]
    a = make(3, 700, biases=0)
    del a["allowed_row"]
    check(be, torch.randn(3, 700, device="cuda"), a)


def test_unsound_lengths_and_offsets(be):
    """Lengths past the history's room and offsets past the biases are cut off."""
    a = make(4, 300)
    a["history_len"] = np.array([10**9, -5, 60, 61], np.int32)
    x = torch.randn(4, 300, device="cuda")
    check(be, x, a)
    up = {k: torch.from_numpy(v).cuda() for k, v in a.items()}
    want, _ = be.adjust_logits(x, **up)
    up["bias_start"] = up["bias_start"].clone()
    n = int(up["bias_start"][-1])
    up["bias_start"][-1] = 2**31 - 1
    got, _ = be.adjust_logits(x, **up)
    assert torch.equal(got, want) and n == up["bias"].numel()


def test_only_one_of_the_results(be):
    x = torch.randn(3, 5000, device="cuda")
    up = {k: torch.from_numpy(v).cuda() for k, v in make(3, 5000).items()}
    out, best = be.adjust_logits(x, **up)
    assert be.adjust_logits(x, want_next=False, **up)[1] is None and torch.equal(be.adjust_logits(x, want_next=False, **up)[0], out)
    none, again = be.adjust_logits(x, want_out=False, **up)
    assert none is None and torch.equal(again, best)
    assert be.adjust_logits(x[:0])[0].shape == (0, 5000)


def test_a_recorded_plan_and_eager_calls(be):
    """Replays over changed logits and histories, with eager calls on other streams between, are the eager results."""
    a = {k: torch.from_numpy(v).cuda() for k, v in make(8, 40000).items()}
    x, out = torch.randn(8, 40000, device="cuda"), torch.empty(8, 40000, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be.adjust_logits(x, out=out, **a)
        stream.synchronize()
        kept = []
        plan = be.plan_record(lambda: kept.append(be.adjust_logits(x, out=out, **a)[1]))
        for i in range(5):
            x.normal_()
            a["history_len"].fill_(10 * i)
            plan.replay()
            stream.synchronize()
            got, best = out.clone(), kept[0].clone()
            eager, again = be.adjust_logits(x, **a)
            stream.synchronize()
            assert torch.equal(got, eager) and torch.equal(best, again)
    del plan


def test_the_bindings_refusals(be):
    x = torch.randn(3, 100, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (dict(history=i[:, None]), dict(repetition=x[:, 0].contiguous()), dict(history=i[:, None], history_len=i[:2]), dict(history=i[:, None], history_len=i, repetition=i), dict(bias_start=i), dict(bias=x[0]),
                dict(allowed=i[:, None]), dict(allowed_row=i), dict(out=x.bfloat16()), dict(want_out=False, want_next=False), dict(logits=x.half()), dict(logits=x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            be.adjust_logits(**(dict(logits=x) | bad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("others", [False, True])
def test_a_history_without_room(be, others, dtype):
    """A sampler's first step without a prompt: no token has come, so no penalty touches a logit; the other rules hold."""
    x = torch.randn(3, 5000, device="cuda").to(dtype)
    a = {k: torch.from_numpy(v).cuda() for k, v in make(3, 5000).items()}
    names = ("history", "history_len", "prompt_len", "repetition", "presence", "frequency")
    rest = {k: v for k, v in a.items() if k not in names} if others else {}
    none = dict(history=a["history"][:, :0], **{k: a[k] for k in names[1:]})
    want, best = be.adjust_logits(x, **rest)
    got, again = be.adjust_logits(x, **none, **rest)
    assert torch.equal(got, want) and torch.equal(best, again)
    for bad in (dict(history_len=None), dict(history_len=a["history_len"][:2]), dict(repetition=a["prompt_len"]), dict(history=a["history"][:2, :0]), dict(history=a["history"][:, :0].long())):
        with pytest.raises(ValueError):
            be.adjust_logits(x, **(none | bad))
