"""The 8-bit key / value cache in plain 64-bit numpy: its layout, its quantization and the attention over it, for the tests."""
import numpy as np
import torch

BLOCK = 32
FLOOR, CEIL = 2.0**-60, 2.0**60


def offsets(d):
    """Byte of (token, channel) in a block of keys and of values."""
    t, c = np.meshgrid(np.arange(BLOCK), np.arange(d), indexing="ij")
    k = c // 32 * 1024 + c % 32 // 8 * 256 + t % 16 * 16 + t // 16 * 8 + c % 8
    v = c // 32 * 1024 + t % 16 // 4 * 256 + c % 16 * 16 + c % 32 // 16 * 8 + t // 16 * 4 + t % 4
    return k, v


class World:
    """A cache with random codes and scales, sequences with random pages, and whatever no token needs set to the worst it may hold."""

    def __init__(self, lens, n_kv, d, page=32, seed=0, n=None, spare=2, wild=True, device="cuda", loud=0.5):
        r = self.rng = np.random.default_rng(seed)
        self.lens, self.n_kv, self.d, self.page = np.asarray(lens), n_kv, d, page
        self.n = np.ones(len(lens), int) if n is None else np.asarray(n)
        self.per = page // BLOCK
        need = -(-self.lens // page)
        self.n_pages = int(need.sum()) + spare
        width = int(max(need.max(), 1)) + 1
        ids = r.permutation(self.n_pages)
        bad = np.array([-1, -2**31, 2**31 - 1, self.n_pages], np.int64)
        self.table = bad[r.integers(0, 4, (len(lens), width))].astype(np.int32) if wild else np.zeros((len(lens), width), np.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = ids[at : at + k]
            at += k
        shape = (self.n_pages, n_kv, self.per)
        self.k, self.v = (r.integers(0, 256, (*shape, BLOCK * d)).astype(np.uint8) if wild else np.full((*shape, BLOCK * d), 128, np.uint8) for _ in range(2))
        self.ks, self.vs = (np.full(shape, np.nan, np.float32) for _ in range(2))
        held = np.clip(np.rint(r.normal(0, 40, (2, int(self.lens.sum()), n_kv, d))), -127, 127) + 128
        ko, vo = offsets(d)
        at = 0
        for s, length in enumerate(self.lens):
            for b in range(-(-length // BLOCK)):
                p, i = self.table[s, b // self.per], b % self.per
                m = min(BLOCK, length - b * BLOCK)
                for codes, off, x in ((self.k, ko, held[0]), (self.v, vo, held[1])):
                    codes[p, :, i][:, off[:m].reshape(-1)] = x[at : at + m].transpose(1, 0, 2).reshape(n_kv, -1)
                self.ks[p, :, i] = 0.02 * np.exp(0.3 * r.normal(size=n_kv))
                self.vs[p, :, i] = 0.02 * np.exp(loud * r.normal(size=n_kv))
                at += m
        self.device = device
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.rows = int(self.start[-1])

    def tensors(self, hip, ragged=None, extra_rows=0):
        """(KvCache, KvBatch) on the device."""
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.device)  # noqa: E731
        cache = hip.KvCache(up(self.k), up(self.v), up(self.ks), up(self.vs), self.page, self.d)
        ragged = (self.n != 1).any() if ragged is None else ragged
        batch = hip.KvBatch(up(self.lens.astype(np.int32)), up(self.table), rows=self.rows + extra_rows if ragged else None, row_start=up(self.start) if ragged else None)
        return cache, batch

    def sequence(self, s):
        """The f64 keys and values [length, n_kv, d] of sequence s."""
        out = []
        for codes, scales, off in zip((self.k, self.v), (self.ks, self.vs), offsets(self.d)):
            x = np.zeros((-(-self.lens[s] // BLOCK) * BLOCK, self.n_kv, self.d))
            for b in range(len(x) // BLOCK):
                p, i = self.table[s, b // self.per], b % self.per
                x[b * BLOCK : (b + 1) * BLOCK] = ((codes[p, :, i][:, off].astype(np.float64) - 128) * scales[p, :, i].astype(np.float64)[:, None, None]).transpose(1, 0, 2)
            out.append(x[: self.lens[s]])
        return out


def attend(w, q, g, scale, cap=0.0, slopes=None, window=0, prefix=None, first=None, half=False, heads=None):
    """(out, bound) f64 [rows, n_kv * g, d]: the attention of q [rows, n_kv * g, d] over World w, and how far a result may be from it (of `heads`
    alone, if given).

    The bound counts roundings, u = 2^-24 being half a step of f32, of the quantities that the kernel forms:
      a score's error: the product's d terms and the two halves' sum, (d + 8) u of sum |q k| scale, and 2^-22 of the row's largest |q| in each
      channel (f32 rows as two f16 values of 11 bits; bf16 rows are exact); the factors' and the exponent's roundings, 8 u of (|score| + 24 + 60);
      with a cap 8 u cap more, with a slope 4 u of slope * distance; a weight's relative error is twice that, and its own rounding 2^-21 (two f16
      values) or 2^-11 (`half`: one); what f16 cannot resolve, 2^-36 of the largest weight; the sums' 64 + length / 128 additions."""
    n_q, d = w.n_kv * g, w.d
    out, tol = np.zeros((w.rows, n_q, d)), np.zeros((w.rows, n_q, d))
    u = 2.0**-24
    for s in range(len(w.lens)):
        length, n, r0 = int(w.lens[s]), int(w.n[s]), int(w.start[s])
        if not n or not length:
            continue
        k, v = w.sequence(s)
        j = np.arange(length)
        pos = length - n + np.arange(n)
        sees = j[None] <= pos[:, None]
        if window:
            sees &= j[None] > pos[:, None] - window
        if first is not None:
            sees &= j[None] >= np.asarray(first)[r0 : r0 + n, None]
        if prefix is not None:
            sees |= j[None] < prefix[s]
        for h in range(n_q) if heads is None else heads:
            x, kh, vh = q[r0 : r0 + n, h], k[:, h // g], v[:, h // g]
            score = scale * (x @ kh.T)
            mass = abs(scale) * (np.abs(x) @ np.abs(kh).T)
            ds = (d + 8) * u * mass
            if not half:
                ds += 2.0**-22 * abs(scale) * np.abs(x).max(1, keepdims=True) * np.abs(kh).sum(1)[None]
            if cap:
                score = cap * np.tanh(score / cap)
                ds += 8 * u * cap
            if slopes is not None:
                bias = slopes[h] * np.abs(pos[:, None] - j[None])
                score = score - bias
                ds += 4 * u * np.abs(bias)
            ds += 8 * u * (np.abs(score) + 84)
            score = np.where(sees, score, -np.inf)
            top = score.max(1, keepdims=True)
            p = np.exp(score - np.where(np.isfinite(top), top, 0))
            total = p.sum(1, keepdims=True)
            live = total[:, 0] > 0
            o = p @ vh / np.where(total > 0, total, 1)
            out[r0 : r0 + n, h] = np.where(live[:, None], o, 0)
            ds = np.where(sees, ds, 0)
            rel = 2 * ds + (2.0**-11 if half else 2.0**-21) + (64 + length / 128) * 2 * u
            e = (p * rel) @ np.abs(vh) / np.where(total > 0, total, 1)
            e += (p * rel).sum(1, keepdims=True) / np.where(total > 0, total, 1) * np.abs(o)
            e += 2.0**-36 * length * np.abs(vh).max() / np.where(total > 0, total, 1)
            if half:
                e += 2.0**-8 * np.abs(o)
            tol[r0 : r0 + n, h] = np.where(live[:, None], e, 0)
    return out, tol


def rotate(x, pos, table, interleaved):
    """x [rows, heads, d] f64 by the table's angles of positions pos."""
    x = np.array(x, np.float64)
    half = table.shape[1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = (table[pos][:, None, :, k].astype(np.float64) for k in (0, 1))
    xa, xb = x[..., a], x[..., b]
    x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


def append(w, new_k, new_v):
    """Puts the rows' keys and values [rows, n_kv, d] f64 (already rotated) into World w as the cache's definition has it."""
    ko, vo = offsets(w.d)
    for s in range(len(w.lens)):
        n, length = int(w.n[s]), int(w.lens[s])
        before = length - n
        for codes, scales, off, new in ((w.k, w.ks, ko, new_k), (w.v, w.vs, vo, new_v)):
            x = np.clip(np.nan_to_num(new[w.start[s] : w.start[s] + n], nan=0.0, posinf=np.inf, neginf=-np.inf), -127 * CEIL, 127 * CEIL)
            for b in range(max(before, 0) // BLOCK, -(-length // BLOCK)):
                lo, hi = max(b * BLOCK, before, 0), min((b + 1) * BLOCK, length)
                if hi <= lo:
                    continue
                p, i = w.table[s, b // w.per], b % w.per
                if not 0 <= p < w.n_pages:
                    continue
                y = x[lo - before : hi - before]
                old = off[: lo - b * BLOCK]
                for h in range(w.n_kv):
                    need = max(float(np.float32(np.abs(y[:, h]).max() / 127)), FLOOR)
                    scale = need
                    if len(old):
                        was = float(scales[p, h, i])
                        if was > FLOOR:
                            scale = was
                            while scale < need:
                                scale *= 2
                        held = codes[p, h, i][old].astype(np.float64) - 128
                        codes[p, h, i][old] = np.rint(held * (was / scale)) + 128
                    scales[p, h, i] = scale
                    codes[p, h, i][off[lo - b * BLOCK : hi - b * BLOCK]] = np.clip(np.rint(y[:, h] / scale), -127, 127) + 128
