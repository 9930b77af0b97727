"""Plain forms of the paged key-value cache for the tests: float64 attention and writes, and the
page bookkeeping one entry after the other on the host."""
import torch

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}


def table_for(lens, page, width, pages, gen=None, rows=None):
    """int32 [rows, width] on the host: each sequence's pages in shuffled order, -1 behind."""
    rows = len(lens) if rows is None else rows
    order = torch.randperm(pages, generator=gen).tolist()
    t = torch.full((rows, width), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range(min(width, -(-max(n, 0) // page))):
            t[i, j] = order.pop()
    return t


def attention64(q, k_pages, v_pages, table, lens, scale, k_scale=None, v_scale=None):
    """(out, lse, sum p |v|) in float64 on the host."""
    q = q.detach().cpu().double()
    kp, vp, table = k_pages.cpu(), v_pages.cpu(), table.cpu()
    b, heads, dim = q.shape
    pages, hkv, page, _ = kp.shape
    out = torch.zeros(b, heads, dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((b, heads), float("-inf"), dtype=torch.float64)
    for i, n in enumerate(lens.tolist()):
        n = max(0, min(n, table.shape[1] * page))
        at = [(int(table[i, p // page]), p % page) for p in range(n)]
        at = [(x, y) for x, y in at if 0 <= x < pages]
        if not at:
            continue
        px, py = (torch.tensor(z) for z in zip(*at))
        for h in range(hkv):
            k = kp[px, h, py].double() * (1 if k_scale is None else float(k_scale[h]))
            v = vp[px, h, py].double() * (1 if v_scale is None else float(v_scale[h]))
            g = slice(h * (heads // hkv), (h + 1) * (heads // hkv))
            s = q[i, g] @ k.T * scale
            lse[i, g] = torch.logsumexp(s, -1)
            w = torch.softmax(s, -1)
            out[i, g], mag[i, g] = w @ v, w @ v.abs()
    return out, lse, mag


def write64(qkv, heads, hkv, dim, positions, q_norm, k_norm, cos, sin, eps):
    """(q, k, v, size of the terms of q, k) in float64 on the host, before any store."""
    x = qkv.detach().cpu().double().reshape(qkv.shape[0], -1, dim)
    y = x.clone()
    mag = x.abs()
    half = dim // 2
    for h in range(heads + hkv):
        w = q_norm if h < heads else k_norm
        if w is not None:
            y[:, h] = x[:, h] / (x[:, h].square().mean(-1, keepdim=True) + eps).sqrt() * \
                w.cpu().double()
        mag[:, h] = y[:, h].abs()
        if cos is not None:
            p = positions.cpu().clamp(0, cos.shape[0] - 1)
            c, s = cos.cpu().double()[p], sin.cpu().double()[p]
            r = torch.cat([-y[:, h, half:], y[:, h, :half]], -1)
            mag[:, h] = (y[:, h] * c).abs() + (r * s).abs()
            y[:, h] = y[:, h] * c + r * s
    return y[:, :heads], y[:, heads:heads + hkv], y[:, heads + hkv:], mag


class Pages:
    """The bookkeeping, one entry after the other."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens, self.refs = table.tolist(), lens.tolist(), refs.tolist()
        self.page, self.width = page, table.shape[1]

    def _held(self, n):
        return -(-n // self.page)

    def _free(self):
        return self.refs.index(0) if 0 in self.refs else None

    def _bad(self, seqs):
        return any(not 0 <= s < len(self.lens) for s in seqs) or len(set(seqs)) < len(seqs)

    def extend(self, seqs, counts):
        """(status, copies); nothing changes unless the status is 0."""
        if self._bad(seqs) or any(
                c < 0 or self.lens[s] + c > self.width * self.page for s, c in zip(seqs, counts)):
            return 2, []
        kept = [r[:] for r in self.table], self.lens[:], self.refs[:]
        copies = []
        for s, c in zip(seqs, counts):
            n = self.lens[s]
            fresh = list(range(self._held(n), self._held(n + c)))
            if c > 0 and n % self.page and self.refs[self.table[s][n // self.page]] > 1:
                fresh.insert(0, n // self.page)
            for j in fresh:
                p = self._free()
                if p is None:
                    self.table, self.lens, self.refs = kept
                    return 1, []
                if j < self._held(n):
                    copies.append((self.table[s][j], p))
                    self.refs[self.table[s][j]] -= 1
                self.refs[p], self.table[s][j] = 1, p
            self.lens[s] = n + c
        return 0, copies

    def fork(self, parents, children):
        if self._bad(children) or any(not 0 <= p < len(self.lens) for p in parents) or \
                any(self.lens[c] for c in children) or set(parents) & set(children):
            return 2
        for p, c in zip(parents, children):
            n = self._held(self.lens[p])
            self.table[c][:n], self.lens[c] = self.table[p][:n], self.lens[p]
            for x in self.table[p][:n]:
                self.refs[x] += 1
        return 0

    def truncate(self, seqs, new):
        if self._bad(seqs) or any(not 0 <= n <= self.lens[s] for s, n in zip(seqs, new)):
            return 2
        for s, n in zip(seqs, new):
            for j in range(self._held(n), self._held(self.lens[s])):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = n
        return 0

    def compact(self):
        """(live, moves); the tables are rewritten."""
        live, goes = sum(r > 0 for r in self.refs), {}
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                goes[p] = self.refs.index(0)
                self.refs[goes[p]], self.refs[p] = self.refs[p], 0
        self.table = [[goes.get(x, x) for x in r] for r in self.table]
        return live, list(goes.items())
