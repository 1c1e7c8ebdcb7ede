"""A 4-bit cache in pages as numpy has it: its groups, its bytes, and its table's steps entry by entry."""
import numpy as np

SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]  # of a word's eight codes


def half(x):
    """float64 rounded to f16 (numpy rounds once), as float64."""
    with np.errstate(over="ignore"):
        return x.astype(np.float16).astype(np.float64)


def groups(x):
    """Rows [..., D] (float64): codes [..., D/32, 32], steps and lows [..., D/32]; NaN lows where a group is not held."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(g).max(-1) <= 65504)
        g = np.where(bad[..., None], 0.0, g)
        low = half(g.min(-1))
        room = np.maximum((g.max(-1) - low) / 15.0, 0.0)
        step = room.astype(np.float16)
        step = np.where(step.astype(np.float64) > room, np.nextafter(step, np.float16(-1)), step).astype(np.float64)
        y = np.rint((g - low[..., None]) / np.where(step > 0, step, np.inf)[..., None])
    return np.clip(y, 0, 15).astype(np.int64), step, np.where(bad, np.nan, low)


def values(code, step, low):
    """[..., D] as float64."""
    return half(low[..., None] + step[..., None] * code).reshape(*code.shape[:-2], -1)


def row_bytes(x):
    """Rows [..., D] as their codes [..., D/2] and words [..., D/8], uint8."""
    code, step, low = groups(x)
    c = code.reshape(*code.shape[:-2], -1, 8).astype(np.uint64)
    words = sum(c[..., i] << np.uint64(SHIFTS[i]) for i in range(8)).astype(np.uint32)
    bits = [np.where(np.isnan(a), np.uint16(0x7E00), (a + 0.0).astype(np.float16).view(np.uint16)).astype(np.uint32)
            for a in (step, low)]
    meta = (bits[1] << np.uint32(16)) | bits[0]
    return tuple(np.ascontiguousarray(a.astype(np.uint32)).view(np.uint8) for a in (words, meta))


class Pool:
    """The bytes of a pool, its table and counts."""

    def __init__(self, rng, n_layer, n_page, page, nk, D, n_seq, n_table):
        self.n_layer, self.n_page, self.page, self.nk, self.D = n_layer, n_page, page, nk, D
        self.n_seq, self.n_table = n_seq, n_table
        self.data = rng.integers(0, 256, (n_layer, n_page, nk, page * D * 5 // 4), dtype=np.uint8)
        self.table = np.full((n_seq, n_table), -1, np.int32)
        self.refs = np.zeros(n_page, np.int32)

    def blocks(self):
        """Views [layer][page][kv head][slot][bytes]: key codes, value codes, key words, value words."""
        at, out = 0, []
        for w in (self.D // 2, self.D // 2, self.D // 8, self.D // 8):
            out.append(self.data[..., at:at + self.page * w].reshape(*self.data.shape[:3], self.page, w))
            assert out[-1].base is not None
            at += self.page * w
        return out

    def where(self, s, slot):
        """(page, row) of a slot, None without a page."""
        if not 0 <= slot < self.n_table * self.page:
            return None
        p = int(self.table[s, slot // self.page])
        return (p, slot % self.page) if 0 <= p < self.n_page else None

    def put(self, layer, s, slot, k, v):
        """Rows k, v [nk][D] into a slot."""
        at = self.where(s, slot)
        if at:
            for i, x in enumerate((k, v)):
                c, m = row_bytes(x)
                b = self.blocks()
                b[i][layer, at[0], :, at[1]], b[2 + i][layer, at[0], :, at[1]] = c, m

    def get(self, layer, pages):
        """Keys and values of whole pages [n][nk][page][D] as float64."""
        out = []
        b = self.blocks()
        for i in range(2):
            c = np.ascontiguousarray(b[i][layer, pages]).view(np.uint32)
            m = np.ascontiguousarray(b[2 + i][layer, pages]).view(np.uint16).reshape(*c.shape[:-1], -1, 2)
            f = m.view(np.float16).astype(np.float64)
            code = np.stack([(c >> np.uint32(s)) & np.uint32(15) for s in SHIFTS], -1).reshape(*c.shape[:-1], -1, 32)
            with np.errstate(invalid="ignore"):
                out.append(values(code.astype(np.float64), f[..., 0], f[..., 1]))
        return out

    def rows(self, layer, s, n):
        """Keys and values of a sequence's first n slots [nk][n][D]; NaN without a page."""
        e = -(-n // self.page)
        t = self.table[s, :e].astype(np.int64)
        ok = (t >= 0) & (t < self.n_page)
        out = []
        for x in self.get(layer, np.where(ok, t, 0)):
            x = np.where(ok[:, None, None, None], x, np.nan)
            out.append(x.transpose(1, 0, 2, 3).reshape(self.nk, e * self.page, self.D)[:, :n])
        return out

    def valid(self, p):
        return 0 <= p < self.n_page

    def reserve(self, start, length, want):
        """Returns how many pages were short."""
        asked = [(s, e) for s in range(self.n_seq)
                 for e in range(max(int(start[s]), 0) // self.page, self.n_table)
                 if want[s] > max(int(start[s]), 0) and e * self.page < want[s]]
        holders = {}
        for s, e in asked:
            p = int(self.table[s, e])
            if self.valid(p) and self.refs[p] > 1:
                holders.setdefault(p, []).append((s, e))
        stays = {v[-1] for p, v in holders.items() if len(v) == self.refs[p]}
        fresh = [(s, e) for s, e in asked if not self.valid(int(self.table[s, e]))
                 or (self.refs[self.table[s, e]] > 1 and (s, e) not in stays)]
        free = np.flatnonzero(self.refs <= 0)
        if len(fresh) > len(free):
            return len(fresh) - len(free)
        for (s, e), new in zip(fresh, free):
            p = int(self.table[s, e])
            if self.valid(p):
                self.refs[p] -= 1
                n = min(max(int(length[s]) - e * self.page, 0), self.page)
                for b in self.blocks():
                    b[:, new, :, :n] = b[:, p, :, :n]
            self.table[s, e], self.refs[new] = new, 1
        return 0

    def fork(self, parent, keep=None):
        old = self.table.copy()
        for s in range(self.n_seq):
            n = self.n_table if keep is None else -(-max(int(keep[s]), 0) // self.page)
            for e in range(self.n_table):
                if self.valid(int(old[s, e])):
                    self.refs[old[s, e]] -= 1
                p = int(old[parent[s], e]) if 0 <= parent[s] < self.n_seq and e < n else -1
                self.table[s, e] = p if self.valid(p) else -1
                if self.valid(p):
                    self.refs[p] += 1

    def free(self, keep):
        for s in range(self.n_seq):
            if keep[s] < 0:
                continue
            for e in range(-(-int(keep[s]) // self.page), self.n_table):
                if self.valid(int(self.table[s, e])):
                    self.refs[self.table[s, e]] -= 1
                self.table[s, e] = -1

    def compact(self, start, rows, counts):
        """All rows are read before any is written."""
        for s in range(self.n_seq):
            moves = []
            for i in range(int(counts[s])):
                a, b = self.where(s, int(rows[s][i])), self.where(s, int(start[s]) + i)
                if a and b:
                    moves.append((b, [x[:, a[0], :, a[1]].copy() for x in self.blocks()]))
            for b, old in moves:
                for x, y in zip(self.blocks(), old):
                    x[:, b[0], :, b[1]] = y
