"""Prompts and a decode loop through the library alone: matmuls, rotation and append, attention over the 8-bit cache, logits' rules. Every
stage between the matmuls is held to its definition in 64 bits on what the matmuls gave it, token by token."""
import numpy as np
import pytest
import torch

from tests import kv_ref
from tests.test_gpu_logits import plain

pytestmark = pytest.mark.gpu

H, N_Q, N_KV, D, INTER, VOCAB, LAYERS, PAGE = 256, 4, 2, 64, 512, 999, 2, 64
SEQS, MOST = 3, 192


@pytest.fixture(scope="module")
def be():
    from oxinfer_amd import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


class Model:
    """Two small dense layers in Q8_0, a head, and the buffers of a batch."""

    def __init__(self, be):
        from oxinfer_amd import hip, synth
        self.be, self.hip = be, hip
        spec = dict(q=(N_Q * D, H), k=(N_KV * D, H), v=(N_KV * D, H), o=(H, N_Q * D), gate=(INTER, H), up=(INTER, H), down=(H, INTER))
        up = lambda n, k, seed: be.upload_gguf(hip.GGML_Q8_0, synth.gguf_q8_0(n, k, seed), n, k)  # noqa: E731
        self.layers = [{n: up(*s, 10 * i + j) for j, (n, s) in enumerate(spec.items())} for i in range(LAYERS)]
        self.head = up(VOCAB, H, 99)
        g = torch.Generator(device="cuda").manual_seed(1)
        self.embed = torch.randn(VOCAB, H, generator=g, device="cuda")
        self.unit = [{n: torch.full((w.n_in,), float(1 / (w.n_in**0.5 * be.dequantize(w).std())), device="cuda") for n, w in layer.items()} for layer in self.layers]
        self.head_unit = torch.full((H,), float(3 / (H**0.5 * be.dequantize(self.head).std())), device="cuda")
        a = np.arange(MOST)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D / 2))
        self.table = np.stack([np.cos(a), np.sin(a)], 2).astype(np.float32)
        self.rope = hip.Rope(torch.from_numpy(self.table).cuda())
        per = MOST // PAGE
        self.caches = [be.kv_cache(SEQS * per + 2, N_KV, D, page_tokens=PAGE) for _ in range(LAYERS)]
        self.pages = torch.randperm(SEQS * per + 2, device="cuda")[: SEQS * per].reshape(SEQS, per).to(torch.int32).contiguous()
        self.kv_len = torch.zeros(SEQS, dtype=torch.int32, device="cuda")
        self.step = hip.KvBatch(self.kv_len, self.pages)
        f = dict(dtype=torch.float32, device="cuda")
        self.x, self.act = torch.zeros(SEQS, H, **f), torch.zeros(SEQS, INTER, **f)
        self.qkv = [torch.zeros(SEQS, (N_Q + 2 * N_KV) * D, **f) for _ in range(LAYERS)]
        self.rot = [torch.zeros(SEQS, N_Q * D, **f) for _ in range(LAYERS)]
        self.att = [torch.zeros(SEQS, N_Q * D, **f) for _ in range(LAYERS)]
        self.logits, self.out = torch.zeros(SEQS, VOCAB, **f), torch.zeros(SEQS, VOCAB, **f)
        self.history = torch.zeros(SEQS, MOST, dtype=torch.int32, device="cuda")
        self.history_len, self.prompt_len = (torch.zeros(SEQS, dtype=torch.int32, device="cuda") for _ in range(2))
        self.allowed = torch.from_numpy(np.random.default_rng(4).integers(-2**31, 2**31, (1, 32)).astype(np.int32)).cuda()
        self.rules = dict(history=self.history, history_len=self.history_len, prompt_len=self.prompt_len, repetition=torch.full((SEQS,), 1.2, **f), presence=torch.full((SEQS,), 0.3, **f),
                          frequency=torch.full((SEQS,), 0.2, **f), bias_start=torch.tensor([0, 2, 2, 3], dtype=torch.int32, device="cuda"), bias_id=torch.tensor([5, 7, 9], dtype=torch.int32, device="cuda"),
                          bias=torch.tensor([1.5, -50.0, 2.0], **f), allowed=self.allowed, allowed_row=torch.tensor([-1, 0, -1], dtype=torch.int32, device="cuda"))

    def mirror(self):
        """The caches' definition: a World per layer that shares the page table."""
        worlds = []
        for _ in range(LAYERS):
            w = kv_ref.World([0] * SEQS, N_KV, D, page=PAGE, n=[0] * SEQS, spare=SEQS * MOST // PAGE + 2, wild=False)
            w.table = self.pages.cpu().numpy()
            worlds.append(w)
        return worlds

    def decode(self):
        """One token of every sequence: embeddings in self.x, logits and tokens out."""
        be, hip = self.be, self.hip
        for i, w in enumerate(self.layers):
            _, qa = be.rmsnorm_quantize(self.x, self.unit[i]["q"], want_out=False)
            for n, at, width in (("q", 0, N_Q), ("k", N_Q, N_KV), ("v", N_Q + N_KV, N_KV)):
                y = be.decode(w[n], xa=qa)
                self.qkv[i][:, at * D : (at + width) * D].copy_(y)
                self.keep.append(y)  # (what a plan writes must stay its own)
            q, k, v = self.qkv[i].split([N_Q * D, N_KV * D, N_KV * D], 1)
            be.kv_append(self.caches[i], self.step, k, v, q=q, rope=self.rope, q_out=self.rot[i])
            be.attend(self.caches[i], self.step, self.rot[i], out=self.att[i])
            qo = be.quantize_act(self.att[i])
            assert be.linear(w["o"], self.x, xa=qo, mode=hip.LIN_ADD)
            _, qa = be.rmsnorm_quantize(self.x, self.unit[i]["gate"], want_out=False)
            assert be.linear(w["gate"], self.act, xa=qa, mode=hip.LIN_SILU_PAIR, w2=w["up"])
            qd = be.quantize_act(self.act)
            assert be.linear(w["down"], self.x, xa=qd, mode=hip.LIN_ADD)
            self.keep.append((qa, qo, qd))
        _, qa = be.rmsnorm_quantize(self.x, self.head_unit, want_out=False)
        be.decode(self.head, xa=qa, y=self.logits)
        self.next = be.adjust_logits(self.logits, out=self.out, **self.rules)[1]
        self.keep.append(qa)

    def prompt(self, ids, worlds):
        """Ragged prompts by the prefill products, f32 rows; returns the embeddings' rows after the layers."""
        be, hip = self.be, self.hip
        n = np.array([len(p) for p in ids])
        start = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")
        self.kv_len += torch.tensor(n, dtype=torch.int32, device="cuda")
        batch = hip.KvBatch(self.kv_len, self.pages, rows=int(n.sum()), row_start=start)
        x = self.embed[torch.tensor(np.concatenate(ids), device="cuda")]
        norm = lambda x, u: x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6) * u  # noqa: E731
        for i, w in enumerate(self.layers):
            xn = norm(x, self.unit[i]["q"])
            q, k, v = (be.gemm(w[m], xn) for m in "qkv")
            rq = be.kv_append(self.caches[i], batch, k, v, q=q, rope=self.rope)
            out = be.attend(self.caches[i], batch, rq)
            self.hold(worlds[i], n, i, q, k, v, rq, out)
            x = x + be.gemm(w["o"], out)
            xn = norm(x, self.unit[i]["gate"])
            x = x + be.gemm(w["down"], be.glu(be.gemm(w["gate"], xn), be.gemm(w["up"], xn)))
        return x[start[1:].long() - 1]

    def hold(self, world, n, i, q, k, v, rotated, out):
        """What the stages made of q, k and v, against their definitions."""
        world.n, world.start = n, np.concatenate([[0], np.cumsum(n)])
        world.rows = int(n.sum())
        world.lens = self.kv_len.cpu().numpy()
        pos = np.concatenate([world.lens[s] - n[s] + np.arange(n[s]) for s in range(SEQS)])
        h = lambda t: t.double().cpu().numpy().reshape(world.rows, -1, D)  # noqa: E731
        kv_ref.append(world, kv_ref.rotate(h(k), pos, self.table, False), h(v))
        want = kv_ref.rotate(h(q), pos, self.table, False)
        assert (np.abs(h(rotated) - want) <= 2.0**-24 * np.abs(want) * 1.001).all()
        want, tol = kv_ref.attend(world, h(rotated), N_Q // N_KV, D**-0.5)
        assert (np.abs(h(out) - want) <= tol).all()
        cache = self.caches[i]
        for s in range(SEQS):
            for b in range(-(-int(world.lens[s]) // 32)):
                p, j = world.table[s, b // world.per], b % world.per
                assert np.array_equal(cache.k_scale[p, :, j].cpu().numpy(), world.ks[p, :, j]) and np.array_equal(cache.v_scale[p, :, j].cpu().numpy(), world.vs[p, :, j])


def test_prompts_then_tokens_by_a_recorded_plan(be):
    m = Model(be)
    worlds = m.mirror()
    rng = np.random.default_rng(0)
    prompts = [list(rng.integers(0, VOCAB, n)) for n in (50, 1, 71)]
    last = m.prompt(prompts, worlds)
    m.keep = []
    for s, p in enumerate(prompts):
        m.history[s, : len(p)] = torch.tensor(p, dtype=torch.int32)
        m.history_len[s] = m.prompt_len[s] = len(p)
    _, first = be.adjust_logits(be.gemm(m.head, last * torch.rsqrt((last * last).mean(1, keepdim=True) + 1e-6) * m.head_unit), **m.rules)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        def advance(tokens):  # the step's inputs: embeddings, lengths, histories
            m.x.copy_(m.embed[tokens.long()])
            m.kv_len += 1
            m.history.scatter_(1, m.history_len.long()[:, None], tokens[:, None])
            m.history_len.add_(1)

        tokens = first
        advance(tokens)
        m.decode()  # once by single calls: the stream's scratch comes into being
        stream.synchronize()
        plan, seen = None, []
        for step in range(40):
            if step:
                advance(tokens)
                plan.replay()
                stream.synchronize()
            for i in range(LAYERS):
                m.hold(worlds[i], np.ones(SEQS, int), i, *m.qkv[i].split([N_Q * D, N_KV * D, N_KV * D], 1), m.rot[i], m.att[i])
            want, tol = plain(m.logits.double().cpu().numpy(), {k: v.cpu().numpy() for k, v in m.rules.items()})
            got = m.out.double().cpu().numpy()
            f = np.isfinite(want)
            assert np.array_equal(f, np.isfinite(got)) and (np.abs(got[f] - want[f]) <= tol[f] + 1e-30).all()
            assert m.next.tolist() == [int(r.argmax()) for r in got]
            tokens = m.next.clone()
            seen.append(tokens.tolist())
            if plan is None:
                kept = m.next
                plan = be.plan_record(m.decode)
                assert kept is not m.next
    assert len({t[0] for t in seen}) > 5 and all(t[0] != 7 for t in seen)
    assert int(m.kv_len[2]) == 71 + 40
    del plan
