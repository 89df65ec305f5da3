"""Oracle of the paged 4-bit key/value cache: the format in numpy (fp32 arithmetic step by step, as the definition has it), attention in
float64, the page operations as plain loops over Python lists.  Nothing here is imported by the product."""
import numpy as np


def formats():
    return [(d, g) for d in (64, 128) for g in (32, 64, 128) if g <= d]


def tile_bytes(D, G):
    return 16 * D + 128 * D // G


def quantize(x, G):
    """x fp16 [..., D] -> codes uint8 [..., D], s fp16 and m fp16 [..., D/G]."""
    y = x.astype(np.float32).reshape(*x.shape[:-1], -1, G)
    lo, hi = y.min(-1), y.max(-1)
    with np.errstate(all="ignore"):
        s = ((hi - lo) / np.float32(15)).astype(np.float16)
        odd = ~np.isfinite(y).all(-1)
        s = np.where(odd, np.float16(np.nan), s)
        n = np.minimum(np.rint((y - lo[..., None]) / s.astype(np.float32)[..., None]), np.float32(15))
        n = np.where((s > 0)[..., None], n, 0).astype(np.uint8)
    return n.reshape(x.shape), s, lo.astype(np.float16)


def value(n, s, m, G):
    """What codes stand for, float64."""
    y = n.astype(np.float64).reshape(*n.shape[:-1], -1, G)
    return (m.astype(np.float64)[..., None] + y * s.astype(np.float64)[..., None]).reshape(n.shape)


def held(x, G):
    return value(*quantize(x, G), G)


def rotate(x, cos, sin):
    """fp16 [..., D] with fp16 tables [..., D]: fp32 products and sum, each rounded, then fp16."""
    x = x.astype(np.float32)
    d = x.shape[-1] // 2
    y = np.concatenate((-x[..., d:], x[..., :d]), -1)
    return (x * cos.astype(np.float32) + y * sin.astype(np.float32)).astype(np.float16)


class Pages:
    """One layer's pool as numpy bytes [pages, kv, P/16, T] with its table [B, width]."""

    def __init__(self, pool, table, D, G):
        self.pool, self.table, self.D, self.G = pool, table, D, G
        self.P = pool.shape[2] * 16

    def _tile(self, b, head, t):
        return self.pool[self.table[b, t // self.P], head, t % self.P // 16]

    def _places(self, r):
        """Byte and shift of every dim's code, and byte of every group's (s, m), for the key and the value row r of a tile."""
        D, G = self.D, self.G
        J, half, par = D // 32, 8 * D, 64 * D // G
        kb, vb, sh = [], [], []
        for d in range(D):
            w, h = d // 8, d // 4
            kb.append(r * (D // 2) + 4 * ((w % 4) * J + w // 4) + d % 8 // 2)
            v = 2 * ((h % 8) * J + h // 8) + d % 4 // 2
            if D == 128 and (r >> 1) & 1:
                v ^= 32
            vb.append(half + par + r * (D // 2) + v)
            sh.append(4 * (d % 2))
        kp = [half + (r * (D // G) + g) * 4 for g in range(D // G)]
        vp = [2 * half + par + (r * (D // G) + g) * 4 for g in range(D // G)]
        return np.array(kb), np.array(vb), np.array(sh), kp, vp

    def store(self, b, head, t, k, v):
        """k, v fp16 [D] -> position t of row b."""
        tile, (kb, vb, sh, kp, vp) = self._tile(b, head, t), self._places(t % 16)
        for x, at, par in ((k, kb, kp), (v, vb, vp)):
            n, s, m = quantize(x, self.G)
            tile[at] = 0
            np.bitwise_or.at(tile, at, (n << sh).astype(np.uint8))
            for g, p in enumerate(par):
                tile[p:p + 4] = np.array([s[g], m[g]], dtype=np.float16).view(np.uint8)

    def load(self, b, head, t):
        """-> k, v float64 [D]."""
        tile, (kb, vb, sh, kp, vp) = self._tile(b, head, t), self._places(t % 16)
        out = []
        for at, par in ((kb, kp), (vb, vp)):
            sm = np.stack([tile[p:p + 4].copy().view(np.float16) for p in par])
            out.append(value((tile[at] >> sh) & 15, sm[:, 0], sm[:, 1], self.G))
        return out

    def rows(self, b, head, n):
        """K, V float64 [n, D] of positions 0 .. n-1; positions whose page is outside the pool are left out."""
        ts = [t for t in range(n) if 0 <= self.table[b, t // self.P] < self.pool.shape[0]]
        kv = [self.load(b, head, t) for t in ts]
        return np.array([x[0] for x in kv]).reshape(-1, self.D), np.array([x[1] for x in kv]).reshape(-1, self.D)


def attend(q, K, V, scale):
    """One query [D] over K, V [n, D], float64; zeros over nothing."""
    if not len(K):
        return np.zeros(len(q))
    x = K @ q * scale
    p = np.exp(x - x.max())
    return p @ V / p.sum()


# ---- pages: table and lens are lists (of lists), refs a list; all changed in place ----

def _deal(refs, n):
    return [p for p, r in enumerate(refs) if r == 0][:n]


def reserve(table, lens, refs, counts, P):
    pos, failed, free = [], False, sum(r == 0 for r in refs)
    for r, c in enumerate(counts):
        if c <= 0 or lens[r] < 0 or lens[r] + c > len(table[r]) * P:
            pos.append(-1)
            continue
        have = -(-lens[r] // P)
        need = -(-(lens[r] + c) // P) - have
        if need and (failed or need > free):
            failed = True
            pos.append(-1)
            continue
        free -= need
        for i, p in enumerate(_deal(refs, need)):
            table[r][have + i] = p
            refs[p] = 1
        pos.append(lens[r])
        lens[r] += c
    return pos


def free(table, lens, refs, rows):
    for r in rows:
        if 0 <= r < len(table):
            for p in table[r]:
                if p >= 0:
                    refs[p] -= 1
            table[r][:] = [-1] * len(table[r])
            lens[r] = 0


def fork(pool, table, lens, refs, src, dst, P):
    """pool [layers, pages, kv, P/16, T]."""
    was, failed, taken = list(lens), False, set()
    for s, d in zip(src, dst):
        first = d not in taken
        taken.add(d)
        if not (first and 0 <= s < len(table) and 0 <= d < len(table)) or was[d] != 0 or any(p >= 0 for p in table[d]):
            continue
        n = was[s]
        if n == 0:
            continue
        full, part = n // P, n % P
        page = None
        if part:
            page = _deal(refs, 1)
            if failed or not page:
                failed = True
                continue
            page = page[0]
            refs[page] = 1
            tiles = -(-part // 16)
            pool[:, page, :, :tiles] = pool[:, table[s][full], :, :tiles]
        for c in range(full):
            table[d][c] = table[s][c]
            refs[table[s][c]] += 1
        if part:
            table[d][full] = page
        lens[d] = n


def compact(pool, table, refs):
    used = sum(r != 0 for r in refs)
    src = [p for p in range(used, len(refs)) if refs[p]]
    dst = [p for p in range(used) if not refs[p]]
    to = dict(zip(src, dst))
    for a, b in to.items():
        pool[:, b] = pool[:, a]
        refs[b], refs[a] = refs[a], 0
    for row in table:
        row[:] = [to.get(p, p) for p in row]
