"""Plain 64-bit forms of the paged-cache operators for the tests, and the
building of caches with pages in random order."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


class Cache:
    """Sequences of the given lengths in a pool of pages in random order.
    Slots that hold no token, and pages of no sequence, hold `junk`."""

    def __init__(self, lens, nkv, hd, page, dtype, device, seed=0, junk=float("nan"), nhd=False, extra=3, wide=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        total = sum(need) + extra
        order = torch.randperm(total, generator=g).tolist()
        width = max(max(need), 1) + wide
        self.page, self.lens, self.n_pages = page, list(lens), total
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.rows = rows
        self.table = torch.tensor(rows, dtype=torch.int32, device=device)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=device)
        self.refs = torch.zeros(total, dtype=torch.int32)
        for r in rows:
            for p in r:
                if p >= 0:
                    self.refs[p] += 1
        self.refs = self.refs.to(device)
        shape = (total, page, nkv, hd) if nhd else (total, nkv, page, hd)
        pool = []
        for _ in range(2):
            t = torch.randn(shape, generator=g, dtype=torch.float32).to(dtype).to(device)
            t = t.transpose(1, 2) if nhd else t
            held = torch.zeros(total, page, dtype=torch.bool)
            for r, n in zip(rows, lens):
                for j in range(-(-n // page)):
                    held[r[j], : min(page, n - j * page)] = True
            t.masked_fill_(~held.to(device)[:, None, :, None], junk)
            pool.append(t)
        self.k, self.v = pool

    def tokens(self, s):
        """(K, V) of sequence s in order, f64 [kv_heads, tokens, hd]."""
        n = self.lens[s]
        out = []
        for pool in (self.k, self.v):
            if n == 0:
                out.append(pool.new_zeros((pool.shape[1], 0, pool.shape[3]), dtype=torch.float64))
            else:
                out.append(torch.cat([pool[p] for p in self.rows[s][: -(-n // self.page)]], 1)[:, :n].double())
        return out


def starts_of(rows, device, first=0):
    s = [first]
    for n in rows:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=device)


def attention(q, cache, rows, scale, softcap=0.0, window=0, first=0):
    """(out, bound, lse) in 64 bits; `bound` the error that the operator's
    roundings can make of each value.

    Per row: u |o| for the output's rounding; with A = sum_j p_j |v_j|: u A
    for the rounded probabilities (f32: two tf32 halves, 2^-21 A each for P
    and V), A x 2 d for scores that are off by d (each moves its own
    probability and the sum), (n + 64) 2^-23 A for sums of n + 64 terms in
    f32 (tensor cores may truncate) and the 2-ulp exponentials. d: hd + 4
    roundings of scale sum |q k|; f32 adds its split operands; a tanh in 16
    bits is off by 2^-21 of the cap (f32: 2^-22), the score's 2^-23."""
    T, H, D = q.shape
    out = torch.full((T, H, D), float("nan"), dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-30)
    lse = torch.full((T, H), float("nan"), dtype=torch.float64, device=q.device)
    at, u, f32 = first, EPS[q.dtype], q.dtype == torch.float32
    for s, n in enumerate(rows):
        t = cache.lens[s]
        k, v = cache.tokens(s)
        pos = torch.arange(t - n, t, device=q.device)[:, None]
        key = torch.arange(t, device=q.device)[None]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        for h in range(H):
            kk, vv = k[h // (H // k.shape[0])], v[h // (H // k.shape[0])]
            x = scale * (q[at:at + n, h].double() @ kk.T)
            mag = scale * (q[at:at + n, h].double().abs() @ kk.abs().T)
            d = ((D + 4) * 2.0 ** -24 + (2.0 ** -20 if f32 else 0)) * mag + 2.0 ** -22 * x.abs()
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                d = d + softcap * (2.0 ** -22 if f32 else 2.0 ** -21) * 2
            x = torch.where(seen, x, -math.inf)
            d = torch.where(seen, d, 0.0).nan_to_num(0.0).amax(1, keepdim=True) if t else torch.zeros(n, 1, dtype=torch.float64, device=q.device)
            if t == 0:
                out[at:at + n, h] = 0
                lse[at:at + n, h] = -math.inf
                continue
            top = x.amax(1, keepdim=True)
            e = torch.where(seen, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
            tot = e.sum(1, keepdim=True)
            p = e / torch.where(tot == 0, 1.0, tot)
            # A value that no row may see counts for nothing, whatever it is.
            clean = torch.where(torch.isfinite(vv), vv, 0.0)
            o = p @ clean
            for j in (~torch.isfinite(vv)).any(1).nonzero()[:, 0].tolist():
                o = o + torch.where(seen[:, j:j + 1] & ~torch.isfinite(vv[j])[None], vv[j][None], 0.0)
            A = p @ clean.abs()
            out[at:at + n, h] = o
            bound[at:at + n, h] = u * o.abs() + A * ((2.0 ** -20 if f32 else 1.01 * u) + 2 * d + (t + 64) * 2.0 ** -23) + 1e-30
            if not f32:
                bound[at:at + n, h] += 2.0 ** -24 * (q.dtype == torch.float16)  # halves below the normal range
            lse[at:at + n, h] = torch.where(tot == 0, -math.inf, torch.log(tot) + top)[:, 0]
        at += n
    return out, bound, lse


def rope(x, pos, inv_freq, interleaved, mscale=1.0):
    """x [rows, heads, hd] f64 turned to positions pos [rows]."""
    half = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()
    z = torch.polar(torch.full_like(ang, mscale), ang)[:, None]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.clone()
    w = torch.complex(x[..., a], x[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


class Pages:
    """The page operations on plain lists, the definitions restated."""

    def __init__(self, table, lens, refs, page):
        self.table = [list(r) for r in table]
        self.lens, self.refs, self.page = list(lens), list(refs), page

    def cells(self, n):
        return -(-n // self.page)

    def fork(self, parents, width):
        table = []
        for r, n in zip(self.table, self.lens):
            for p in r[: self.cells(n)]:
                self.refs[p] -= 1
        lens = []
        for p in parents:
            row = self.table[p][: self.cells(self.lens[p])] if p >= 0 else []
            for c in row:
                self.refs[c] += 1
            table.append(row + [-1] * (width - len(row)))
            lens.append(self.lens[p] if p >= 0 else 0)
        self.table, self.lens = table, lens

    def resize(self, new):
        """The copies made, [(src, dst)], and the number of missing pages."""
        for s, (n, t) in enumerate(zip(self.lens, new)):
            if t <= n:
                for x in range(self.cells(t), self.cells(n)):
                    self.refs[self.table[s][x]] -= 1
                    self.table[s][x] = -1
                self.lens[s] = t
        refs, copies, grants = list(self.refs), [], []
        need = 0
        plan = []
        for s, t in enumerate(new):
            n = self.lens[s]
            if t <= n:
                continue
            cow = False
            if n % self.page:
                tail = self.table[s][n // self.page]
                if refs[tail] > 1:
                    refs[tail] -= 1
                    cow = True
            more = self.cells(t) - self.cells(n)
            need += cow + more
            plan.append((s, t, cow, more))
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if need > len(free):
            return [], need - len(free)
        take = iter(free)
        for s, t, cow, more in plan:
            n = self.lens[s]
            if cow:
                src, dst = self.table[s][n // self.page], next(take)
                self.refs[src] -= 1
                self.refs[dst] = 1
                self.table[s][n // self.page] = dst
                copies.append((src, dst))
            for x in range(more):
                p = next(take)
                self.refs[p] = 1
                self.table[s][self.cells(n) + x] = p
            self.lens[s] = t
        return copies, 0

    def compact(self):
        used = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(used)
        moves = list(zip([p for p in used if p >= n], [p for p in range(n) if self.refs[p] == 0]))
        to = dict(moves)
        for s, r in enumerate(self.table):
            for x in range(self.cells(self.lens[s])):
                r[x] = to.get(r[x], r[x])
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        return moves, n
