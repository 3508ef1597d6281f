"""Plain forms in 64 bits of the attention-side operators (lib.kv_append, lib.attn, lib.spec_verify), and steps to run them on."""
import math

import numpy as np
import torch

from dsgx10_amd import lib

BF16 = torch.bfloat16
E4M3_MAX = 448.0


class Step:
    """A cache with a batch over it: rows[b] rows and lens[b] own tokens a sequence behind `prefix` shared ones, pages handed out in a
    shuffled order. What no token fills holds `junk`. layout: "thd" pools [page][token][head][D], "htd" [page][head][token][D], "kv"
    keys and values in one tensor [page][2][token][head][D]."""

    def __init__(self, rows, lens, prefix=0, Hq=8, Hkv=2, D=128, page=16, fmt="bf16", layout="thd", seed=0, junk=float("nan"), device="cuda", max_rows=None, max_len=None, cu=True,
                 spare=2, kscale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.P, self.Hq, self.Hkv, self.D, self.page, self.fmt, self.device = rows, lens, prefix, Hq, Hkv, D, page, fmt, device
        B = len(rows)
        per = max(1, max(-(-n // page) for n in lens))
        own, pre = [-(-n // page) for n in lens], -(-prefix // page)
        self.npages = sum(own) + pre + spare
        order = torch.randperm(self.npages, generator=g).tolist()
        self.prefix_pages = order[:pre]
        at = pre
        self.table_rows = []
        for n in own:
            self.table_rows.append(order[at:at + n])
            at += n
        # places past a sequence's pages hold numbers that must not be followed
        table = torch.tensor([r + [-1 if i % 2 else 2 ** 31 - 1 for i in range(per - len(r))] for r in self.table_rows], dtype=torch.int32)
        shape = {"thd": (self.npages, page, Hkv, D), "htd": (self.npages, Hkv, page, D), "kv": (self.npages, 2, page, Hkv, D)}[layout]
        dt = BF16 if fmt == "bf16" else torch.uint8
        fill = junk if fmt == "bf16" else (0x7F if math.isnan(junk) else 0)
        pools = [torch.full(shape, fill, dtype=dt, device=device)] * 2 if layout == "kv" else [torch.full(shape, fill, dtype=dt, device=device) for _ in range(2)]
        if layout == "kv":
            self.kpool, self.vpool = pools[0][:, 0], pools[0][:, 1]
        else:
            self.kpool, self.vpool = (p if layout == "thd" else p.permute(0, 2, 1, 3) for p in pools)
        self.pools = pools
        self.ks = self.vs = None
        if fmt == "e4m3":
            self.ks, self.vs = (torch.rand(Hkv, generator=g).mul(0.02).add(0.01).to(device) for _ in range(2))
        self.g, self.kscale = g, kscale
        total = lambda n: torch.randn(n, Hkv, D, generator=g)  # noqa: E731
        self.pre_kv = [self._held(total(prefix), s) for s in (self.ks, self.vs)]
        self.own_kv = [[self._held(total(n), s) for s in (self.ks, self.vs)] for n in lens]
        self.store()
        self.R = sum(rows)
        cu_rows = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.first = cu_rows
        self.t_lens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.t_table = table.to(device)
        self.t_cu = torch.from_numpy(cu_rows).to(device) if cu else None
        self.t_prefix = torch.tensor(self.prefix_pages, dtype=torch.int32, device=device) if prefix else None
        self.cache = lib.kv_cache(self.kpool, self.vpool, self.ks, self.vs)
        self.batch = lib.kv_batch(self.R, max_rows or max(1, max(rows)), max(lens) if max_len is None else max_len, self.t_lens, self.t_table, cu_rows=self.t_cu, prefix_len=prefix,
                                  prefix=self.t_prefix)
        self.q = (torch.randn(self.R, Hq, D, generator=g) * 1.5).to(BF16)

    def _held(self, x, scale):
        """values as a cache's element type holds them"""
        x = x * self.kscale
        if self.fmt == "bf16":
            return x.to(BF16)
        return (x / scale.cpu()[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)

    def _put(self, pool, pages, x):
        if x.shape[0] == 0:
            return
        t = torch.arange(x.shape[0])
        pg = torch.tensor(pages)[t // self.page].to(pool.device)
        raw = x if self.fmt == "bf16" else x.view(torch.uint8)
        pool[pg, (t % self.page).to(pool.device)] = raw.to(pool.device)

    def store(self):
        """the tokens' keys and values into their places"""
        for i, pool in enumerate((self.kpool, self.vpool)):
            self._put(pool, self.prefix_pages, self.pre_kv[i])
            for b, pages in enumerate(self.table_rows):
                self._put(pool, pages, self.own_kv[b][i])

    def values(self, b):
        """prefix's and sequence b's keys and values, f64 [tokens][Hkv][D]"""
        out = []
        for i, s in enumerate((self.ks, self.vs)):
            x = torch.cat([self.pre_kv[i].double(), self.own_kv[b][i].double()])
            out.append(x if s is None else x * s.cpu().double()[:, None])
        return out

    def run(self, scale=None, ld_extra=0, lse=True, out=None, stream=None, ws=None):
        scale = self.D ** -0.5 if scale is None else scale
        n, ld = self.Hq * self.D, self.Hq * self.D + ld_extra
        q = torch.full((max(self.R, 1), ld), float("nan"), dtype=BF16, device=self.device)
        q[:self.R, :n] = self.q.reshape(self.R, n).to(self.device)
        out = torch.full((max(self.R, 1), ld), 7.0, dtype=BF16, device=self.device) if out is None else out
        z = torch.full((max(self.R, 1), self.Hq), 7.0, device=self.device) if lse else None
        if ws is None:
            ws = torch.zeros(lib.attn_ws_bytes(self.cache, self.batch, self.Hq), dtype=torch.uint8, device=self.device)
        lib.attn(self.cache, self.batch, q, ld, self.Hq, scale, out, ld, ws, lse=z, stream=stream)
        torch.cuda.synchronize()
        return out.cpu(), None if z is None else z.cpu()


def attn64(s, scale=None):
    """(out, sum of p |v|, lse, bound on a score's f32 error) of every row's head in 64 bits, shapes [R][Hq][D] and [R][Hq]"""
    scale = s.D ** -0.5 if scale is None else scale
    G = s.Hq // s.Hkv
    o, mag, lse, err = (torch.zeros(s.R, s.Hq, s.D, dtype=torch.float64), torch.zeros(s.R, s.Hq, s.D, dtype=torch.float64),
                        torch.full((s.R, s.Hq), -math.inf, dtype=torch.float64), torch.zeros(s.R, s.Hq, dtype=torch.float64))
    for b, (n, L) in enumerate(zip(s.rows, s.lens)):
        k, v = s.values(b)
        for i in range(n):
            r, seen = int(s.first[b]) + i, s.P + max(0, L - n + i + 1)
            if seen == 0:
                continue
            for h in range(s.Hkv):
                q = s.q[r, h * G:(h + 1) * G].double()
                kk, vv = k[:seen, h], v[:seen, h]
                a = q @ kk.T * scale
                z = torch.logsumexp(a, -1)
                p = (a - z[:, None]).exp()
                o[r, h * G:(h + 1) * G], mag[r, h * G:(h + 1) * G], lse[r, h * G:(h + 1) * G] = p @ vv, p @ vv.abs(), z
                # f32 sums of D exact products in any order, the scaling and the exponent's subtraction
                err[r, h * G:(h + 1) * G] = ((q.abs() @ kk.abs().T * abs(scale)).amax(-1) * (s.D + 8) + z.abs()) * 2.0 ** -24
    return o, mag, lse, err


def check_attn(s, out, lse, scale=None, rows=None):
    """Against the 64-bit form. Roundings: the result's to bf16 (2^-8 of it), the numerators' to bf16 (2^-8 of p each, so 2^-8 sum p |v|),
    a score's error e as a factor 1 +- e on p and on the sum, and f32 sums over a few hundred blocks and ranges (2^-14)."""
    o, mag, z, err = attn64(s, scale)
    got = out[:s.R, :s.Hq * s.D].double().view(s.R, s.Hq, s.D)
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -14 + 3 * err[..., None]) * mag + 1e-30
    rows = slice(None) if rows is None else rows
    bad = ((got - o).abs() > tol)[rows] | ~torch.isfinite(got[rows])
    assert not bad.any(), "%d values off, worst %.3g of the bound" % (int(bad.sum()), float(((got - o).abs() / tol)[rows].max()))
    if lse is not None:
        lse = lse[:s.R].double()
        none = torch.isinf(z)
        assert torch.equal(torch.isinf(lse)[rows], none[rows]) and bool((lse[rows][none[rows]] < 0).all())
        d = torch.where(none, torch.zeros_like(z), lse - z).abs()[rows]
        assert bool((d <= (2 * err + 2.0 ** -20 * (1 + z.abs().nan_to_num(posinf=0)))[rows]).all()), float(d.max())


# ---- kv_append -------------------------------------------------------------------------------------------------------------
def append64(x, w, cs, rot, off, pairs, eps):
    """x f64 [H][D] of one row; cs f64 [rot]: (y, the magnitude that its f32 errors are relative to)"""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y, mag = x.clone(), x.abs()
    if rot:
        i = torch.arange(0, rot, 2) if pairs else torch.arange(rot // 2)
        a, b = off + i, off + (i + 1 if pairs else i + rot // 2)
        co, si = cs[:rot // 2], cs[rot // 2:]
        y[:, a], y[:, b] = x[:, a] * co - x[:, b] * si, x[:, b] * co + x[:, a] * si
        m = x[:, a].abs() + x[:, b].abs()
        mag = mag.clone()
        mag[:, a], mag[:, b] = m, m
    return y, mag


def rope_table(n, rot, base=10000.0):
    a = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat([a.cos(), a.sin()], 1).float()


# ---- spec_verify -----------------------------------------------------------------------------------------------------------
def verify64(target, draft, u, us, rows, q=None, temp=None, probs=False):
    """the definition, a sequence at a time, numpy f64: (tokens, accepted)"""
    R, V = target.shape
    tokens, accepted = np.full(R, -1, np.int32), np.zeros(len(rows), np.int32)
    r0 = 0

    def dist(r, T):
        x = target[r].astype(np.float64)
        if probs:
            return x
        if T <= 0:
            p = np.zeros(V)
            p[int(np.argmax(x))] = 1.0 if not np.isnan(x).any() else np.nan
            return p
        with np.errstate(all="ignore"):
            e = np.exp((x - x.max()) / T)
            return e / e.sum()

    for b, n in enumerate(rows):
        T = 1.0 if temp is None else float(np.float32(temp[b]))
        for i in range(n):
            r = r0 + i
            p, d = dist(r, T), int(draft[r])
            w = p
            if i < n - 1:
                known = 0 <= d < V
                qd = 1.0 if q is None else float(q[r, d]) if known else 0.0
                if known and float(u[r]) * qd < p[d]:
                    tokens[r] = d
                    accepted[b] += 1
                    continue
                less = q[r].astype(np.float64) if q is not None else (np.arange(V) == d).astype(np.float64)
                rest = p - less
                rest = np.where(rest > 0, rest, np.where(np.isnan(rest), np.nan, 0.0))
                w = p if rest.sum() <= 0 else rest
            c = np.cumsum(w)
            if c[-1] > 0 and np.isfinite(c[-1]):
                above = np.nonzero(c > float(us[b]) * c[-1])[0]
                tokens[r] = above[0] if len(above) else np.nonzero(w > 0)[0][-1]
            break
        r0 += n
    return tokens, accepted
