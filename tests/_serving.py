"""Plain 64-bit restatements of the serving operators, for their tests."""

from __future__ import annotations

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative error of one rounding


def attend(q, k, v, allowed, scale):
    """One head's rows in 64 bits over the allowed keys only: output, logarithm
    of the sum, and the mean of |v| under the weights (the error scale).
    Disallowed keys and values are never touched, so anything may stand there."""
    q, k, v = q.double(), k.double(), v.double()
    out, lse, size = torch.zeros(q.shape, dtype=torch.float64), torch.full((q.shape[0],), -torch.inf, dtype=torch.float64), None
    size = torch.zeros(q.shape, dtype=torch.float64)
    for r in range(q.shape[0]):
        at = allowed[r].nonzero()[:, 0]
        if len(at) == 0:
            continue
        s = (k[at] @ q[r]) * scale
        lse[r] = torch.logsumexp(s, 0)
        w = torch.exp(s - lse[r])[:, None]
        out[r], size[r] = (w * v[at]).sum(0), (w * v[at].abs()).sum(0)
    return out, lse, size


def check(out, lse, want, want_lse, size, dtype, scores=8.0):
    """Bounds of the arithmetic: the output's own rounding u |o|; the
    probabilities' rounding, u sum w |v|; scores in FP32, whose error of about
    2^-20 of their size (a few units) moves every weight by less than 1e-4;
    fp16's smallest steps, 2^-24, for outputs and (against the largest one)
    probabilities. The sums of exponentials are FP32: 1e-4 covers lse."""
    u, out = UNIT[dtype], out.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), finite), "non-finite values in other places"
    tiny = 0.0 if dtype == torch.bfloat16 else 2.0 ** -12
    tol = u * want.abs() + (u + 1e-4) * size + tiny * 2.0 ** -12 + 1e-6
    bad = finite & ((out - want).abs() > tol)
    assert not bad.any(), f"{int(bad.sum())} outputs out of bounds, worst {float(((out - want).abs() / tol)[finite].max()):.2f}x"
    lse = lse.double().cpu()
    empty = want_lse == -torch.inf
    assert torch.equal(lse == -torch.inf, empty)
    assert torch.all((lse - want_lse)[~empty].abs() <= 1e-4)


class HostCache:
    """The paged cache's bookkeeping and data as the definitions say it, on the host."""

    def __init__(self, cache):
        self.size = cache.page_size
        self.k, self.v = cache.k.cpu().view(torch.int16).numpy().copy(), cache.v.cpu().view(torch.int16).numpy().copy()
        self.tables, self.lens, self.refs = (t.cpu().numpy().copy() for t in (cache.tables, cache.lens, cache.refs))

    def _take(self):
        page = int(np.flatnonzero(self.refs == 0)[0])
        self.refs[page] = 1
        return page

    def append(self, sequences, counts, k, v, rows):
        free, need = int((self.refs == 0).sum()), 0
        for s, n in zip(sequences, counts):
            need += -(-(self.lens[s] + n) // self.size) - -(-self.lens[s] // self.size)
            if -(-(self.lens[s] + n) // self.size) > self.tables.shape[1]:
                return False
        if need > free:
            return False
        t = 0
        for s, n in zip(sequences, counts):
            for _ in range(n):
                p, slot = divmod(int(self.lens[s]), self.size)
                if slot == 0:
                    self.tables[s, p] = self._take()
                self.k[:, self.tables[s, p], :, slot] = k[:, rows[t]]
                self.v[:, self.tables[s, p], :, slot] = v[:, rows[t]]
                self.lens[s] += 1
                t += 1
        return True

    def trim(self, sequences, lens):
        for s, n in zip(sequences, lens):
            if n < self.lens[s] and n % self.size and self.refs[self.tables[s, n // self.size]] > 1:
                return False
        for s, n in zip(sequences, lens):
            n = min(n, self.lens[s])
            for p in range(-(-n // self.size), -(-self.lens[s] // self.size)):
                self.refs[self.tables[s, p]] -= 1
                self.tables[s, p] = -1
            self.lens[s] = n
        return True

    def fork(self, parents, children):
        if sum(self.lens[p] % self.size > 0 for p in parents) > int((self.refs == 0).sum()):
            return False
        for a, b in zip(parents, children):
            full, part = divmod(int(self.lens[a]), self.size)
            self.tables[b, :full] = self.tables[a, :full]
            for p in self.tables[a, :full]:
                self.refs[p] += 1
            if part:
                new, old = self._take(), self.tables[a, full]
                self.tables[b, full] = new
                self.k[:, new, :, :part], self.v[:, new, :, :part] = self.k[:, old, :, :part], self.v[:, old, :, :part]
            self.lens[b] = self.lens[a]
        return True

    def compact(self):
        live = np.flatnonzero(self.refs > 0)
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        for old, new in zip([p for p in live if p >= len(live)], holes):
            self.k[:, new], self.v[:, new] = self.k[:, old], self.v[:, old]
            self.refs[new], self.refs[old] = self.refs[old], 0
            self.tables[self.tables == old] = new
        return True

    def same(self, cache):
        for name in ("tables", "lens", "refs"):
            assert np.array_equal(getattr(cache, name).cpu().numpy(), getattr(self, name)), name
        for name in ("k", "v"):
            assert np.array_equal(getattr(cache, name).cpu().view(torch.int16).numpy(), getattr(self, name)), name
