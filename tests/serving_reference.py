"""Plain implementations of the serving operators for their tests: attention in 64 bits, the pages' books in Python."""
import math

import torch

EPS = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def gather(pages, row, length, head):
    """The first `length` rows of one sequence and key head, in 64 bits."""
    size = pages.shape[2]
    at = row[: -(-length // size)].long()
    return pages[at, head].flatten(0, 1)[:length].double()


def decode(q, k_pages, v_pages, table, lens, scale=None, attend_current=False):
    """(o, rem, bound of |error| of o, of rem): 64 bits, and what a kernel that computes in 32 bits may be off by.

    Bounds.  A score is a sum of d products, each rounding at most 2^-24 of what has been added up: off by at most
    dz = (d + 2) 2^-24 s sum|q k|.  log a_j = log beta_j + sum over later keys of log(1 - beta); a score's error enters the first
    with a factor of at most 1 and the others with beta <= -log(1 - beta), so log a_j is off by dz (1 + S), S = -log of the stick
    that is left (104 at most: behind that a weight is 0 in 32 bits).  The functions (exp, log1p and their fast forms) and the
    sums over keys: within 2^-20 of 1 + S.  Weights as the sum of two 16-bit numbers: 2^-17 of each.  o is then off by that share
    of sum a_j |v_j|, rem by that share of itself, both by half a step of their type and its smallest number."""
    batch, heads, new, d = q.shape
    group = heads // k_pages.shape[1]
    scale = d ** -0.5 if scale is None else scale
    o, rem = torch.zeros(q.shape, dtype=torch.float64), torch.ones(q.shape[:3], dtype=torch.float64)
    o_err, rem_err = torch.zeros_like(o), torch.zeros_like(rem)
    half = EPS[q.dtype] / 2
    q, k_pages, v_pages, table, lens = (t.cpu() for t in (q, k_pages, v_pages, table, lens))
    for b, n in enumerate(lens.tolist()):
        for h in range(heads):
            k, v = gather(k_pages, table[b], n, h // group), gather(v_pages, table[b], n, h // group)
            for t in range(new):
                last = max(n - new + t + int(attend_current), 0)
                if last == 0:
                    continue
                row = q[b, h, t].double()
                z = k[:last] @ row * scale
                broken = torch.nn.functional.softplus(z)
                incl = broken.flip(0).cumsum(0).flip(0)
                a = torch.exp(z - incl)
                o[b, h, t] = a @ v[:last]
                rem[b, h, t] = torch.exp(-incl[0])
                dz = (d + 2) * 2.0 ** -24 * abs(scale) * float((k[:last].abs() @ row.abs()).max())
                used = 1 + min(float(incl[0]), 104.0)
                share = (dz + 2.0 ** -20) * used + (2.0 ** -17 if q.dtype != torch.float32 else 0)
                o_err[b, h, t] = share * (a @ v[:last].abs()) + half * o[b, h, t].abs()
                rem_err[b, h, t] = (share + half) * rem[b, h, t]
    small = SMALLEST[q.dtype]
    return o, rem, o_err + small, rem_err + small


def check_decode(got, want):
    o, rem, o_err, rem_err = want
    for name, a, b, err in (("o", got[0], o, o_err), ("rem", got[1], rem, rem_err)):
        a = a.detach().cpu().double()
        assert torch.isfinite(a).all(), f"{name} has values that are not finite"
        off = (a - b).abs() / err
        i = int(off.argmax())
        assert float(off.max()) <= 1.0, (f"{name}: {float(a.flatten()[i]):.8g} for {float(b.flatten()[i]):.8g}, "
                                         f"{float(off.max()):.3g} times what rounding explains")


def make_cache(gen, lens, kv_heads, page, d, dtype, spare=3, shift=0.0, width=None, poison=True):
    """Pools whose rows behind the sequences' ends, and whose spare pages, hold NaN; a table of scattered pages, -1 behind."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lens), width or max(max(counts), 1) + 1), -1, dtype=torch.int32)
    k = torch.full((pages, kv_heads, page, d), float("nan") if poison else 0.0).to(dtype)
    v = k.clone()
    at = 0
    for b, (n, count) in enumerate(zip(lens, counts)):
        table[b, :count] = order[at:at + count].int()
        at += count
        for i in range(count):
            rows = min(page, n - i * page)
            k[table[b, i], :, :rows] = (torch.randn(kv_heads, rows, d, generator=gen) - shift).to(dtype)
            v[table[b, i], :, :rows] = torch.randn(kv_heads, rows, d, generator=gen).to(dtype)
    return k, v, table, torch.tensor(lens, dtype=torch.int32)


class Books:
    """The keeping of the pages, one token and page at a time.  `data` maps (page, slot) to a number that stands for the token."""

    def __init__(self, max_seqs, max_pages, num_pages, page):
        self.page, self.max_pages = page, max_pages
        self.rows = [[] for _ in range(max_seqs)]
        self.lens, self.refs, self.data = [0] * max_seqs, [0] * num_pages, {}

    def _take(self, count):
        free = [i for i, n in enumerate(self.refs) if n == 0][:count]
        return free if len(free) == count else None

    def extend(self, counts):
        if not torch.is_tensor(counts):
            counts = [counts if n else 0 for n in self.lens]
        counts = [int(c) for c in counts]
        after = [n + c for n, c in zip(self.lens, counts)]
        if min(counts) < 0 or max(after) > self.max_pages * self.page:
            return False
        need = [-(-n // self.page) - len(row) for n, row in zip(after, self.rows)]
        free = self._take(sum(need))
        if free is None:
            return False
        for row, n in zip(self.rows, need):
            for _ in range(n):
                row.append(free.pop(0))
                self.refs[row[-1]] = 1
        self.lens = after
        return True

    def fork(self, src, dst):
        src, dst = [int(x) for x in src], [int(x) for x in dst]
        seqs = range(len(self.rows))
        if any(s not in seqs for s in src) or any(d not in seqs or self.lens[d] for d in dst) or len(set(dst)) < len(dst) or set(src) & set(dst):
            return False
        free = self._take(sum(self.lens[s] % self.page > 0 for s in src))
        if free is None:
            return False
        for s, d in zip(src, dst):
            full, rest = divmod(self.lens[s], self.page)
            self.rows[d] = self.rows[s][:full]
            for page in self.rows[d]:
                self.refs[page] += 1
            if rest:
                page = free.pop(0)
                self.refs[page] = 1
                for slot in range(rest):
                    self.data[page, slot] = self.data[self.rows[s][full], slot]
                self.rows[d].append(page)
            self.lens[d] = self.lens[s]
        return True

    def free(self, seqs):
        if any(int(s) not in range(len(self.rows)) for s in seqs):
            return False
        for s in set(int(x) for x in seqs):
            for page in self.rows[s]:
                self.refs[page] -= 1
            self.rows[s], self.lens[s] = [], 0
        return True

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        moved = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        place = dict(zip(moved, holes))
        for old, new in place.items():
            self.refs[new], self.refs[old] = self.refs[old], 0
            for slot in range(self.page):
                if (old, slot) in self.data:
                    self.data[new, slot] = self.data[old, slot]
        self.rows = [[place.get(page, page) for page in row] for row in self.rows]

    def write(self, seq, pos, value):
        self.data[self.rows[seq][pos // self.page], pos % self.page] = value

    def tokens(self, seq):
        return [self.data[self.rows[seq][i // self.page], i % self.page] for i in range(self.lens[seq])]

    def table(self):
        t = torch.full((len(self.rows), self.max_pages), -1, dtype=torch.int32)
        for row, pages in zip(t, self.rows):
            row[: len(pages)] = torch.tensor(pages, dtype=torch.int32)
        return t
