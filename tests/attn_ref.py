"""Plain 64-bit forms of the attention-half operators, and error bounds for their bf16
kernels.  Test infrastructure."""
from __future__ import annotations

import math

import torch

BF16 = torch.bfloat16
U = 2.0 ** -8          # half a bf16 step, relative to the value


def visible(p, n, window, sinks):
    """Mask [n] of the keys that the token at index p sees."""
    j = torch.arange(n)
    see = j <= p
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


def gather(pages, row, n):
    """Keys (or values) 0..n-1 of a sequence, [Hkv, n, D] in 64 bits; rows without a page NaN."""
    ps = pages.shape[2]
    out = torch.full((pages.shape[1], n, pages.shape[3]), math.nan, dtype=torch.float64)
    for j0 in range(0, n, ps):
        i = j0 // ps
        p = int(row[i]) if i < len(row) else -1
        if 0 <= p < pages.shape[0]:
            m = min(ps, n - j0)
            out[:, j0:j0 + m] = pages[p, :, :m].double()
    return out


def attention(q, k_pages, v_pages, table, lens, cu, scale, window=0, sinks=0):
    """(out, bound) of a packed batch, in 64 bits, row by row over visible keys only.

    bound: how far a kernel's bf16 output may be off.  The weights p_j are rounded to bf16
    for the product with v (at most U each, so U * sum p|v| / sum p), the output once (U |o|);
    a score's dot product of D terms in 32 bits is off by at most (D + 2) 2^-24 scale
    sum|q||k|, and the exponential by a few 2^-23 of its argument, which moves every weight by that
    relatively, in the numerator and the denominator; sums of n terms by n 2^-24."""
    q, k_pages, v_pages = (t.detach().cpu() for t in (q, k_pages, v_pages))
    table, lens, cu = (t.cpu().tolist() for t in (table, lens, cu))
    T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    G = Hq // Hkv
    cap = len(table[0]) * k_pages.shape[2] if table else 0
    out = torch.zeros((T, Hq, D), dtype=torch.float64)
    bound = torch.full_like(out, 1e-30)      # rows that see nothing: exactly zero
    for b, n in enumerate(lens):
        if cu[b + 1] == cu[b]:
            continue
        if n > cap:
            out[cu[b]:cu[b + 1]] = math.nan
            continue
        k, v = gather(k_pages, table[b], max(n, 0)), gather(v_pages, table[b], max(n, 0))
        for t in range(cu[b], cu[b + 1]):
            p = n - (cu[b + 1] - t)
            if p < 0:
                continue
            see = visible(p, n, window, sinks)
            kk, vv = k[:, see], v[:, see]
            qq = q[t].double().view(Hkv, G, D)
            s = torch.einsum("hgd,hnd->hgn", qq, kk) * scale
            sabs = torch.einsum("hgd,hnd->hgn", qq.abs(), kk.abs()) * abs(scale)
            w = torch.softmax(s, -1)
            o = torch.einsum("hgn,hnd->hgd", w, vv)
            a = torch.einsum("hgn,hnd->hgd", w, vv.abs())
            n_see = int(see.sum())
            ds = (D + 2) * 2.0 ** -24 * sabs.amax(-1) + 8 * 2.0 ** -23 * (s.abs().amax(-1) + 1)
            rel = U + 2 * ds + 2 * n_see * 2.0 ** -24
            out[t] = o.reshape(Hq, D)
            bound[t] = (U * o.abs() + rel[..., None] * a).reshape(Hq, D) * 1.01 + 1e-30
    return out, bound


def axis_of(i, axes, sections, interleaved):
    if interleaved:
        a = i % axes
        return a if i < axes * sections[a] else 0
    end = 0
    for a, n in enumerate(sections):
        end += n
        if i < end:
            return a
    raise AssertionError


def rope(x, positions, inv_freq, sections, interleaved, w=None, eps=1e-6, mscale=1.0):
    """(y, bound) of rows x [T, heads, D] in 64 bits.  bound: the result's rounding (U |y|)
    and the 32-bit norm, sine and products (a few 2^-23 of the pair's magnitudes)."""
    x = x.detach().cpu().double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (1 + w.cpu().double())
    half = inv_freq.numel()
    y, mag = x.clone(), x.abs()
    for i in range(half):
        pos = positions[axis_of(i, positions.shape[0], sections, interleaved)].cpu().double()
        ang = pos * float(inv_freq[i])
        c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
        a, b = x[..., i], x[..., i + half]
        y[..., i], y[..., i + half] = a * c - b * s, b * c + a * s
        mag[..., i] = mag[..., i + half] = (a.abs() + b.abs()) * abs(mscale)
    return y, U * y.abs() + 2.0 ** -19 * mag + 1e-30


def within(got, want, bound, what=""):
    got = got.detach().cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    off = ((got - want).abs() / bound)[~nan]
    if off.numel():
        assert float(off.max()) <= 1.0, f"{what}: {float(off.max()):.3f} of the bound"


class Cache:
    """The page bookkeeping as plain lists."""

    def __init__(self, n_pages, page_size, max_seqs, max_pages):
        self.ps, self.max_pages = page_size, max_pages
        self.refs = [0] * n_pages
        self.tables = [[-1] * max_pages for _ in range(max_seqs)]
        self.lens = [0] * max_seqs

    def _free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def grow(self, slots, add):
        free, ok, total, seen = self._free(), [], 0, set()
        for s, a in zip(slots, add):
            good = 0 <= s < len(self.lens) and s not in seen and a >= 0
            if 0 <= s < len(self.lens):
                seen.add(s)
            good = good and self.lens[s] + a <= self.max_pages * self.ps
            if not good:
                ok.append(0)
                continue
            have = -(-self.lens[s] // self.ps)
            need = -(-(self.lens[s] + a) // self.ps) - have
            total += need
            if total > len(free):
                ok.append(0)
                continue
            for j in range(need):
                p = free[total - need + j]
                self.refs[p] = 1
                self.tables[s][have + j] = p
            self.lens[s] += a
            ok.append(1)
        return ok

    def fork(self, src, dst, keep):
        """(ok, copies): copies = (from page, to page, used rows)."""
        free, ok, copies, total, seen = self._free(), [], [], 0, set()
        S = len(self.lens)
        old = list(self.lens)
        for s, d, k in zip(src, dst, keep):
            good = (0 <= s < S and 0 <= d < S and d not in seen and s not in dst and old[d] == 0
                    and 0 <= k <= old[s])
            if 0 <= d < S:
                seen.add(d)
            if not good:
                ok.append(0)
                continue
            full, used = divmod(k, self.ps)
            tail = used > 0 and self.tables[s][full] >= 0
            total += tail
            if total > len(free):
                ok.append(0)
                continue
            for j in range(full):
                p = self.tables[s][j]
                self.tables[d][j] = p
                if p >= 0:
                    self.refs[p] += 1
            if tail:
                p = free[total - 1]
                self.refs[p] = 1
                self.tables[d][full] = p
                copies.append((self.tables[s][full], p, used))
            self.lens[d] = k
            ok.append(1)
        return ok, copies

    def free(self, slots, window=0, sinks=0):
        for s in slots:
            if not 0 <= s < len(self.lens):
                continue
            lo, hi = 0, self.max_pages
            if window:
                lo, hi = -(-sinks // self.ps), max(0, self.lens[s] - window) // self.ps
            for j in range(lo, min(hi, self.max_pages)):
                if self.tables[s][j] >= 0:
                    self.refs[self.tables[s][j]] -= 1
                    self.tables[s][j] = -1
            if not window:
                self.lens[s] = 0

    def compact(self):
        """(live, remap)."""
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        remap = [p if r > 0 else -1 for p, r in enumerate(self.refs)]
        for h, m in zip(holes, movers):
            remap[m] = h
            self.refs[h], self.refs[m] = self.refs[m], 0
        self.tables = [[remap[p] if p >= 0 else p for p in row] for row in self.tables]
        return live, remap
