"""Attention over shared prefixes and chosen spans, the choice itself and the draw of tokens in plain 64-bit numpy, for the tests."""
import numpy as np

from tests import kv_ref


class Shared(kv_ref.World):
    """A World whose sequences lo .. hi - 1 of each group (group_start) begin with `common` tokens of the group's first one. Their own tables name other pages with
    other tokens there, which nobody is to read."""

    def __init__(self, lens, group_start, common, *args, **kwargs):
        super().__init__(lens, *args, **kwargs)
        self.group_start, self.common = np.asarray(group_start, np.int32), np.asarray(common, np.int32)

    def shares(self, s):
        """(the group's first sequence, the tokens that s shares)."""
        i = int(np.searchsorted(self.group_start, s, side="right")) - 1
        return (int(self.group_start[i]), int(self.common[i])) if 0 <= i < len(self.common) else (s, 0)

    def sequence(self, s):
        leader, common = self.shares(s)
        own = super().sequence(s)
        if leader == s or not common:
            return own
        return [np.concatenate([a[:common], b[common:]])[: self.lens[s]] for a, b in zip(super().sequence(leader), own)]


def named(chosen, pos, span, length=None):
    """How often a list of spans names each token (of `length`) for a row at `pos`."""
    sees, before = np.zeros(pos + 1 if length is None else length, int), -1
    for c in chosen.tolist():
        if before < c and 0 <= c <= pos // span:
            sees[c * span : (c + 1) * span] += 1
        before = c
    return sees


def attend_selected(w, q, g, scale, chosen, span, half=False, **rules):
    """As kv_ref.attend, over the spans alone that `chosen` [rows, n_kv, count] names."""
    out, tol = np.zeros((w.rows, w.n_kv * g, w.d)), np.zeros((w.rows, w.n_kv * g, w.d))
    u = 2.0**-24
    for s in range(len(w.lens)):
        k, v = w.sequence(s)
        for i in range(int(w.n[s])):
            r, pos = int(w.start[s]) + i, int(w.lens[s] - w.n[s]) + i
            if pos < 0:
                continue
            for h in range(w.n_kv * g):
                sees = named(chosen[r, h // g], pos, span, len(k))
                j = np.arange(len(k))
                rule = j <= pos
                if rules.get("window"):
                    rule &= j > pos - rules["window"]
                if rules.get("first") is not None:
                    rule &= j >= rules["first"][r]
                if rules.get("prefix") is not None:
                    rule |= j < rules["prefix"][s]
                often = sees[sees * rule > 0]
                sees = sees * rule > 0
                if not sees.any():
                    continue
                x, kh, vh = q[r, h], k[:, h // g][sees], v[:, h // g][sees]
                score = scale * (kh @ x)
                # (the terms of kv_ref.attend's bound)
                ds = (w.d + 8) * u * abs(scale) * (np.abs(kh) @ np.abs(x))
                if not half:
                    ds = ds + 2.0**-22 * abs(scale) * np.abs(x).max() * np.abs(kh).sum(1)
                if rules.get("cap"):
                    score = rules["cap"] * np.tanh(score / rules["cap"])
                    ds = ds + 8 * u * rules["cap"]
                if rules.get("slopes") is not None:
                    bias = rules["slopes"][h] * np.abs(pos - j[sees])
                    score = score - bias
                    ds = ds + 4 * u * np.abs(bias)
                ds = ds + 8 * u * (np.abs(score) + 84)
                p = often * np.exp(score - score.max())
                o = p @ vh / p.sum()
                rel = 2 * ds + (2.0**-11 if half else 2.0**-21) + (64 + len(p) / 128) * 2 * u
                e = (p * rel) @ np.abs(vh) / p.sum() + (p * rel).sum() / p.sum() * np.abs(o) + 2.0**-36 * len(p) * np.abs(vh).max() / p.sum()
                out[r, h], tol[r, h] = o, e + (2.0**-8 * np.abs(o) if half else 0)
    return out, tol


def summarize(w, span, code, scale):
    """The mean keys of the spans that the rows of World w touch, into code [n_pages, n_kv, page / span, d] and scale."""
    for s in range(len(w.lens)):
        n, length = int(w.n[s]), int(w.lens[s])
        if not n or not length:
            continue
        k, _ = w.sequence(s)
        for x in range(max(length - n, 0) // span, (length - 1) // span + 1):
            p, i = w.table[s, x * span // w.page], x * span % w.page // span
            if not 0 <= p < w.n_pages:
                continue
            mean = k[x * span : (x + 1) * span].mean(0)
            scale[p, :, i] = (np.abs(mean).max(1) / 127).astype(np.float32)
            by = scale[p, :, i].astype(np.float64)[:, None]
            code[p, :, i] = np.where(by > 0, np.rint(mean / np.where(by > 0, by, 1)), 0)


def select(w, q, g, span, code, scale, count, first, last):
    """The spans of each row [rows, n_kv, count]: q [rows, n_kv * g, d] f32."""
    out = np.full((w.rows, w.n_kv, count), -1, np.int32)
    q = np.clip(np.where(np.isnan(q), 0, q), -np.finfo(np.float32).max, np.finfo(np.float32).max).astype(np.float32)
    q_scale = np.abs(q).max(2) * (np.float32(1) / np.float32(127))
    by = q_scale.astype(np.float64)[..., None]
    q_code = np.where(by > 0, np.clip(np.rint(q.astype(np.float64) / np.where(by > 0, by, 1)), -127, 127), 0).astype(np.int64)
    for s in range(len(w.lens)):
        for i in range(int(w.n[s])):
            r, pos = int(w.start[s]) + i, int(w.lens[s] - w.n[s]) + i
            spans = pos // span + 1 if pos >= 0 else 0
            if spans <= count:
                out[r, :, :spans] = np.arange(spans)
                continue
            x = np.arange(spans)
            page, at = w.table[s, x * span // w.page], x * span % w.page // span
            there = (page >= 0) & (page < w.n_pages)
            page = np.where(there, page, 0)
            for h in range(w.n_kv):
                dot = code[page, h, at].astype(np.int64) @ q_code[r, h * g : (h + 1) * g].T
                score = (dot.astype(np.float64) * scale[page, h, at].astype(np.float64)[:, None] * q_scale[r, h * g : (h + 1) * g].astype(np.float64)).max(1)
                score[~there] = -np.inf
                score[(x < first) | (x >= spans - last)] = np.inf
                out[r, h] = np.sort(np.argsort(-score, kind="stable")[:count])
    return out


def sample(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(next, logp) of rows of logits x f64 [rows, vocab]."""
    tokens, logs = [], []
    for r, row in enumerate(x):
        row = np.where(np.isnan(row), -np.inf, row)
        order = np.argsort(-row, kind="stable")
        top = row[order[0]]
        heat = 1.0 if temperature is None else float(temperature[r])
        if top == -np.inf:
            tokens.append(-1)
            logs.append(-np.inf)
            continue
        if not heat > 0:
            tokens.append(int(order[0]))
            logs.append(0.0)
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(row[order] == top, 1.0, np.exp((row[order] - top) / heat) if np.isfinite(top) and np.isfinite(heat) else (row[order] > -np.inf) * float(np.isfinite(top)))
        w = w[w > 0]
        if top_k is not None and top_k[r] > 0:
            w = w[: top_k[r]]
        if top_p is not None and top_p[r] < 1:
            w = w[: 1 + int((np.cumsum(w)[:-1] < float(top_p[r]) * w.sum()).sum())]
        if min_p is not None and min_p[r] > 0:
            w = w[w >= min(float(min_p[r]), 1.0)]
        ids = order[: len(w)]
        by = np.argsort(ids)
        upto = np.cumsum(w[by])
        share = float(u[r]) if u[r] > 0 else 0.0
        at = min(int(np.searchsorted(upto, share * upto[-1], side="right")), len(w) - 1)
        tokens.append(int(ids[by][at]))
        logs.append(float(np.log(w[by][at] / upto[-1])))
    return np.array(tokens), np.array(logs)
