"""The operators of a serving step restated with numpy in 64 bits (TEST
INFRASTRUCTURE): the paged 8-bit cache, attention over it and the verification
of drafts, straight from their definitions in include/squirrel_hip.h."""
import numpy as np

PAGE = 64


def inv_freq(half, base=500000.0):
    return (base ** (-np.arange(half, dtype=np.float64) / max(half, 1))).astype(np.float32)


def rotate(x, pos, inv):
    """x [rows, heads, dim] f64; the first 2 * len(inv) dimensions rotated."""
    x = np.array(x, np.float64)
    half = len(inv)
    if half:
        angle = np.asarray(pos, np.float64)[:, None] * inv.astype(np.float64)[None, :]
        c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
        a, b = x[..., 0:2 * half:2].copy(), x[..., 1:2 * half:2].copy()
        x[..., 0:2 * half:2] = a * c - b * s
        x[..., 1:2 * half:2] = a * s + b * c
    return x


class Cache:
    """One layer's pages: int8 values and f32 scales, keys ([0]) and values ([1])."""

    def __init__(self, n_pages, kv_heads, dim, inv=()):
        self.q = np.zeros((2, n_pages, kv_heads, PAGE, dim), np.int64)
        self.s = np.zeros((2, n_pages, kv_heads), np.float32)
        self.kv_heads, self.dim, self.inv = kv_heads, dim, np.asarray(inv, np.float32)

    def append(self, past, new, tables, k, v, rotated=False):
        row = 0
        for i in range(len(past)):
            a, n = int(past[i]), int(new[i])
            pos = np.arange(a, a + n)
            kk = k[row:row + n].reshape(n, self.kv_heads, self.dim).astype(np.float64)
            vv = v[row:row + n].reshape(n, self.kv_heads, self.dim).astype(np.float64)
            if not rotated:
                kk = rotate(kk, pos, self.inv)
            for which, x in ((0, kk), (1, vv)):
                for page in sorted(set(pos // PAGE)):
                    rows = pos // PAGE == page
                    self._append_page(which, int(tables[i][page]), pos[rows] % PAGE, x[rows])
            row += n

    def _append_page(self, which, page, slots, x):
        tok0 = int(slots[0])
        for h in range(self.kv_heads):
            old = self.s[which, page, h] if tok0 else np.float32(0)
            s = max(old, np.float32(np.abs(x[:, h]).max() / 127.0))
            q = self.q[which, page, h]
            if tok0 and s > old:
                q[:tok0] = np.rint(q[:tok0] * np.float64(old) / np.float64(s))
            new = np.rint(x[:, h] / np.float64(s)) if s > 0 else np.zeros_like(x[:, h])
            q[slots] = np.clip(new, -127, 127)
            self.s[which, page, h] = s

    def values(self, table, length, which, first=0):
        """[length - first, kv_heads, dim]: the f32 values q * s."""
        pos = np.arange(first, length)
        pages = np.asarray(table)[pos // PAGE]
        q = self.q[which][pages, :, pos % PAGE].astype(np.float32)
        return q * self.s[which][pages][:, :, None]


def sdpa(cache, past, new, tables, q, heads, window=0, sinks=0, rotated=False):
    """[rows, heads * dim] in 64 bits, and for each (row, head) the largest sum
    |q_d k_d| / sqrt(d) over its keys and the largest |v|."""
    D, G = cache.dim, heads // cache.kv_heads
    out, amp, vmax = [], [], []
    row = 0
    for i in range(len(past)):
        a, n = int(past[i]), int(new[i])
        if n == 0:
            continue
        k = cache.values(tables[i], a + n, 0).astype(np.float64)
        v = cache.values(tables[i], a + n, 1).astype(np.float64)
        x = q[row:row + n].reshape(n, heads, D).astype(np.float64)
        if not rotated:
            x = rotate(x, np.arange(a, a + n), cache.inv)
        for r in range(n):
            p = a + r
            at = np.arange(a + n)
            seen = at <= p
            if window:
                seen &= (at > p - window) | (at < sinks)
            kk, vv = k[seen], v[seen]
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk[:, h // G] @ x[r, h] / np.sqrt(D)
                    e = np.exp(s - s.max())
                    out.append((e / e.sum()) @ vv[:, h // G])
                    amp.append((np.abs(kk[:, h // G]) @ np.abs(x[r, h])).max() / np.sqrt(D))
                vmax.append(np.abs(vv[:, h // G]).max())
        row += n
    return (np.array(out).reshape(row, heads * D), np.array(amp).reshape(row, heads, 1),
            np.array(vmax).reshape(row, heads, 1))


def verify(target, draft, tokens, u, n_draft, temperature):
    accepted, token = [], []
    t0 = d0 = 0

    def prob(row):
        z = row.astype(np.float64) / temperature
        z = np.exp(z - z.max())
        return z / z.sum()

    def greedy(row):  # the last of equal maxima, as sq_greedy
        return len(row) - 1 - int(np.argmax(row[::-1]))

    for n in map(int, n_draft):
        got, w = 0, None
        for j in range(n):
            x = int(tokens[d0 + j])
            if temperature == 0:
                if x != greedy(target[t0 + j]):
                    break
            else:
                p = prob(target[t0 + j])
                q = prob(draft[d0 + j]) if draft is not None else (np.arange(len(p)) == x).astype(np.float64)
                if not np.float64(u[t0 + j]) * q[x] < p[x]:
                    w = np.maximum(p - q, 0)
                    if not w.sum() > 0:
                        w = p
                    break
            got += 1
        accepted.append(got)
        if temperature == 0:
            token.append(greedy(target[t0 + got]))
        else:
            if w is None:
                w = prob(target[t0 + n])
            cum = np.cumsum(w)
            t = int(np.searchsorted(cum, np.float64(u[t0 + n]) * cum[-1], side="right"))
            token.append(min(t, int(np.nonzero(w)[0][-1])))
        t0, d0 = t0 + n + 1, d0 + n
    return np.array(accepted, np.uint32), np.array(token, np.uint32)
