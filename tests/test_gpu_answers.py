"""Several answers to one prompt, token by token, as a server draws them: the layer's step over the shared prompt (append, attention, the mean keys, the choice among them and the
attention over it) and the draw of the next tokens, recorded once each and replayed. Every stage is held to its definition in 64 bits on what the stages before gave it."""
import numpy as np
import pytest
import torch

from tests import kv_ref, lists_ref

pytestmark = pytest.mark.gpu

N_KV, G, D, PAGE, SPAN, COUNT, VOCAB = 2, 2, 64, 64, 32, 6, 700


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("answers", [5, 40])
def test_answers_to_a_prompt(be, answers, dtype):
    from oxinfer_amd import hip
    rng = np.random.default_rng(answers)
    half, width, prompt = dtype is torch.bfloat16, N_KV * G * D, 192 + 21
    # all tables begin with the prompt's whole pages; the page that it ends in is each answer's own
    w = kv_ref.World([prompt + 40] * answers, N_KV, D, page=PAGE, seed=1)
    w.table[1:, : prompt // PAGE] = w.table[0, : prompt // PAGE]
    w.lens = np.full(answers, prompt)
    cache, batch = w.tensors(hip)
    held = be.kv_summary(cache, SPAN)
    code, scale = np.zeros(held.shape, np.int8), np.zeros(held.shape[:3], np.float32)
    shared = hip.KvShared(torch.tensor([0, answers], dtype=torch.int32, device="cuda"), torch.tensor([prompt // PAGE * PAGE], dtype=torch.int32, device="cuda"))
    embed, head = torch.randn(VOCAB, (G + 2) * N_KV * D, device="cuda"), torch.randn(2 * width, VOCAB, device="cuda") / 12
    numpy = lambda t: t.double().cpu().numpy()  # noqa: E731

    def rows(ids):  # keys, values and queries of tokens
        return [x.contiguous().to(dtype) for x in embed[ids].split([N_KV * D, N_KV * D, width], 1)]

    # the prompt, for the first answer; then the rest of its last page for each other one
    ids = torch.from_numpy(rng.integers(0, VOCAB, prompt)).cuda()
    for s in range(answers):
        lo = 0 if s == 0 else prompt // PAGE * PAGE
        n = np.zeros(answers, int)
        n[s] = prompt - lo
        start = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")
        b = hip.KvBatch(batch.kv_len, batch.pages, rows=prompt - lo, row_start=start)
        k, v, _ = rows(ids[lo:])
        be.kv_append(cache, b, k, v)
        be.kv_summarize(cache, b, held)
        w.n, w.start, w.rows = n, np.concatenate([[0], np.cumsum(n)]), prompt - lo
        kv_ref.append(w, numpy(k).reshape(-1, N_KV, D), numpy(v).reshape(-1, N_KV, D))
        lists_ref.summarize(w, SPAN, code, scale)
    w.n, w.start, w.rows = np.ones(answers, int), np.arange(answers + 1), answers

    k, v, q = rows(torch.zeros(answers, dtype=torch.int64, device="cuda"))
    whole, some, chosen = torch.empty_like(q), torch.empty_like(q), torch.empty((answers, N_KV, COUNT), dtype=torch.int32, device="cuda")
    logits, ruled, u = torch.empty(answers, VOCAB, device="cuda"), torch.empty(answers, VOCAB, device="cuda"), torch.rand(answers, device="cuda")
    history, history_len = torch.zeros((answers, 64), dtype=torch.int32, device="cuda"), torch.zeros(answers, dtype=torch.int32, device="cuda")
    rules = dict(temperature=torch.linspace(0, 1.4, answers, device="cuda"), top_k=torch.arange(answers, dtype=torch.int32, device="cuda") * 7 % 60, top_p=torch.linspace(0.5, 1.1, answers, device="cuda"),
                 min_p=torch.linspace(-0.05, 0.2, answers, device="cuda"))
    penalty = torch.full((answers,), 1.3, device="cuda")
    drawn = []

    def layer():
        be.kv_append(cache, batch, k, v)
        be.attend_shared(cache, batch, shared, q, out=whole)
        be.kv_summarize(cache, batch, held)
        be.kv_select(cache, batch, held, q, COUNT, out=chosen)
        be.attend_selected(cache, batch, q, chosen, SPAN, out=some)

    def draw():
        be.adjust_logits(logits, out=ruled, want_next=False, history=history, history_len=history_len, repetition=penalty)
        drawn.append(be.sample(ruled, u, **rules))

    tokens, seen = ids[-1].repeat(answers), []
    torch.cuda.synchronize()
    plans = None
    with torch.cuda.stream(torch.cuda.Stream()):
        wait = torch.cuda.current_stream().synchronize
        for step in range(37):
            batch.kv_len += 1
            w.lens = w.lens + 1
            for to, x in zip((k, v, q), rows(tokens)):
                to.copy_(x)
            u.copy_(torch.from_numpy(rng.random(answers).astype(np.float32)))
            layer() if plans is None else plans[0].replay()
            torch.mm(torch.cat([whole, some], 1).float(), head, out=logits)
            draw() if plans is None else plans[1].replay()
            wait()
            h = lambda t: numpy(t).reshape(answers, -1, D)  # noqa: E731
            kv_ref.append(w, h(k), h(v))
            lists_ref.summarize(w, SPAN, code, scale)
            assert np.array_equal(held.code.cpu().numpy(), code) and np.array_equal(held.scale.cpu().numpy(), scale)
            want, tol = kv_ref.attend(w, h(q), G, D**-0.5, half=half)
            assert (np.abs(h(whole) - want) <= tol).all()
            want = lists_ref.select(w, h(q).astype(np.float32), G, SPAN, code, scale, COUNT, 1, 1)
            assert np.array_equal(chosen.cpu().numpy(), want)
            want, tol = lists_ref.attend_selected(w, h(q), G, D**-0.5, want, SPAN, half=half)
            assert (np.abs(h(some) - want) <= tol).all()
            want, _ = lists_ref.sample(numpy(ruled), u.cpu().numpy(), **{n: t.cpu().numpy() for n, t in rules.items()})
            got = (drawn[-1] if plans is None else kept)[0]
            assert got.tolist() == want.tolist()
            tokens = got.long().clone()
            seen.append(tokens.tolist())
            history.scatter_(1, history_len.long()[:, None], got[:, None])
            history_len += 1
            if plans is None:
                wait()
                plans = [be.plan_record(layer), be.plan_record(draw)]
                kept = drawn[-1]
    assert len({tuple(t) for t in zip(*seen)}) == answers  # (the answers differ)
    del plans
