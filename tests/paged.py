"""A paged cache and the attention over it, restated in numpy: one operation after the other, one sequence after the other."""
import numpy as np

EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 30: 2.0 ** -8}  # half a step, relative: f32, f16, bf16


class PoolModel:
    """The state of a pool and what each call does to it. `rows` is [n_stores][n_pages * page][width] (any dtype)."""

    def __init__(self, page, n_pages, n_slots, max_pages, rows):
        self.page, self.n_pages, self.n_slots, self.max_pages = page, n_pages, n_slots, max_pages
        self.table = np.full((n_slots, max_pages), -1, np.int32)
        self.lens = np.zeros(n_slots, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.rows = rows
        self.no_pages = self.bad = False

    def pages(self, n):
        return -(-int(n) // self.page)

    def row(self, slot, pos):
        return int(self.table[slot, pos // self.page]) * self.page + pos % self.page

    def _copy(self, src, dst, n):
        self.rows[:, dst * self.page:dst * self.page + n] = self.rows[:, src * self.page:src * self.page + n]

    def _grant(self, needs):
        """Pages for a list of needs (None: an entry that is skipped), in order, from the lowest free ones."""
        free, at, out = list(np.flatnonzero(self.refs == 0)), 0, []
        for n in needs:
            if n is None:
                out.append(None)
                continue
            if n and at + n > len(free):
                self.no_pages = True
                out.append(None)
            else:
                out.append([int(p) for p in free[at:at + n]])
            at += n
        return out

    def fork(self, src, dst):
        lens, refs, table, seen, needs = self.lens.copy(), self.refs.copy(), self.table.copy(), set(), []
        for s, d in zip(src, dst):
            ok = d < self.n_slots and d not in seen
            seen.add(d)
            ok = ok and s < self.n_slots and s != d and lens[d] == 0
            self.bad |= not ok
            needs.append(int(lens[s] % self.page != 0) if ok else None)
        for s, d, got in zip(src, dst, self._grant(needs)):
            if got is None:
                continue
            full = lens[s] // self.page
            self.table[d] = -1
            self.table[d, :full] = table[s, :full]
            for p in table[s, :full]:
                self.refs[p] += 1
            if got:
                self._copy(table[s, full], got[0], lens[s] % self.page)
                self.table[d, full] = got[0]
                self.refs[got[0]] = 1
            self.lens[d] = lens[s]

    def reserve(self, slots, new):
        lens, refs, table, seen, needs, cows = self.lens.copy(), self.refs.copy(), self.table.copy(), set(), [], []
        for s, n in zip(slots, new):
            ok = s < self.n_slots and s not in seen and 0 <= n <= self.max_pages * self.page
            seen.add(s)
            self.bad |= not ok
            cow = -1
            if ok and n > lens[s] and lens[s] % self.page and refs[table[s, lens[s] // self.page]] > 1:
                cow = int(table[s, lens[s] // self.page])
            needs.append(None if not ok else 0 if n <= lens[s] else self.pages(n) - self.pages(lens[s]) + (cow >= 0))
            cows.append(cow)
        for s, n, cow, got in zip(slots, new, cows, self._grant(needs)):
            if got is None or n <= lens[s]:
                continue
            for p in got:
                self.refs[p] = 1
            if cow >= 0:
                self._copy(cow, got[0], lens[s] % self.page)
                self.refs[cow] -= 1
                self.table[s, self.pages(lens[s]) - 1] = got[0]
                got = got[1:]
            for i, p in enumerate(got):
                self.table[s, self.pages(lens[s]) + i] = p
            self.lens[s] = n

    def truncate(self, slots, new=None):
        for s, n in zip(slots, [0] * len(slots) if new is None else new):
            if s >= self.n_slots or n < 0:
                self.bad = True
                continue
            self.lens[s] = min(self.lens[s], n)
            for p in range(self.pages(n), self.max_pages):
                if self.table[s, p] >= 0:
                    self.refs[self.table[s, p]] -= 1
                    self.table[s, p] = -1

    def compact(self):
        used = int((self.refs > 0).sum())
        holes = [p for p in range(used) if self.refs[p] == 0]
        for to, source in zip(holes, [p for p in range(used, self.n_pages) if self.refs[p] > 0]):
            self._copy(source, to, self.page)
            self.table[self.table == source] = to
            self.refs[to], self.refs[source] = self.refs[source], 0
        return used

    def accept(self, slots, n_rows, accepted, counts):
        seen = set()
        for s, n, acc, k in zip(slots, n_rows, accepted, counts):
            acc = list(acc[:max(0, k)])
            ok = s < self.n_slots and s not in seen and 0 <= k <= n and len(acc) == k and all(0 <= a < n for a in acc) and \
                all(a < b for a, b in zip(acc, acc[1:])) and self.lens[s] >= n
            seen.add(s)
            if not ok:
                self.bad = True
                continue
            base = int(self.lens[s]) - n
            moved = [self.rows[:, self.row(s, base + a)].copy() for a in acc]
            for j, r in enumerate(moved):
                self.rows[:, self.row(s, base + j)] = r
            self.truncate([s], [base + k])


def visible(n, ctx, mask_words):
    """[n][ctx + n] truth values from mask words ([n][words] uint64), or a chain for None."""
    see = np.zeros((n, ctx + n), bool)
    see[:, :ctx] = True
    for j in range(n):
        for u in range(n):
            if mask_words is None:
                see[j, ctx + u] = u <= j
            elif u // 64 < mask_words.shape[1]:
                see[j, ctx + u] = bool((int(mask_words[j, u // 64]) >> (u % 64)) & 1)
    return see


def attention(q, k, v, see, scale):
    """One head in f64: (out, the same sum with |v|, the largest sum of |q||k| * scale over the visible keys)."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    out, size, terms = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros(len(q))
    for j in range(len(q)):
        at = np.flatnonzero(see[j])
        if not len(at):
            continue
        z = k[at] @ q[j] * scale
        w = np.exp(z - z.max())
        w /= w.sum()
        out[j], size[j] = w @ v[at], w @ np.abs(v[at])
        terms[j] = (np.abs(k[at]) @ np.abs(q[j])).max() * abs(scale)
    return out, size, terms


def tolerance(out, size, terms, keys, head_dim, dtype, rounded_weights):
    """What rounding can do to a result, element for element.

    A score is a sum of head_dim products in f32: off by at most head_dim + 4 half steps of the sum of their sizes (`terms`), and a
    weight by that factor, up and down, against the sum of all weights (2x). Sums over the keys: one half step per key of the sum
    of sizes, in numerator and denominator. exp2 is within 2 steps (4 half steps). Weights rounded to the row type: one half step
    of that type each. The result is rounded once to the row type."""
    f32 = EPS[0]
    rel = 2 * ((head_dim + 4) * f32 * terms[:, None] + keys * f32 + 8 * f32) + (EPS[dtype] if rounded_weights else 0)
    tiny = 2.0 ** -24 if dtype == 1 else 2.0 ** -126  # below the smallest normal value steps stop shrinking
    return rel * size * (1 + EPS[dtype]) + EPS[dtype] * np.abs(out) + tiny
