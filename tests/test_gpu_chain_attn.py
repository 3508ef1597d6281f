"""The attention side in its place: decode layers with their own paged caches, chained (dsgx10_amd/chain.py), then the head and the
verification of the step's drafts, over several steps of sequences that share a prefix and draft different numbers of tokens. Every
stage against its plain form in 64 bits, fed with the GPU's own inputs of that stage; then the whole step captured and replayed."""
import numpy as np
import pytest
import torch

from dsgx10_amd import abi, lib
from dsgx10_amd.chain import Attention, LayerChain
from tests import gpu, kv, orc
from tests.helpers import check_sums, make_layer
from tests.test_gpu_layer_step import _chain_weights

pytestmark = pytest.mark.gpu

H, QL, I, E, TOPK, NL, V, VP = 2048, 256, 1024, 16, 4, 2, 1003, 1008
PAGE, P, PER, ROT = 16, 21, 5, 32


def bf(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16).copy()).view(torch.bfloat16)


class Model:
    """NL layers with weights, norms and caches of their own, and a head; B sequences of rows[b] rows a step"""

    def __init__(self, rows, Hq, Hkv, D, cache, fmt=abi.FMT_FP8):
        self.rows, self.B, self.M, self.Hq, self.Hkv, self.D, self.fmt = rows, len(rows), sum(rows), Hq, Hkv, D, cache
        self.NQ, self.XR = Hq * D, QL + 2 * Hkv * D + 64
        g = torch.Generator().manual_seed(5)
        self.g = g
        pages = 2 + self.B * PER + 1
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.prefix, self.table = order[:2].cuda(), order[2:2 + self.B * PER].view(self.B, PER).contiguous().cuda()
        self.lens = torch.zeros(self.B, dtype=torch.int32, device="cuda")
        cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.first, self.cu = cu, torch.from_numpy(cu).cuda()
        self.rope = kv.rope_table(P + PER * PAGE, ROT).cuda()
        self.batch = lib.kv_batch(self.M, max(rows), PER * PAGE, self.lens, self.table, cu_rows=self.cu, prefix_len=P, prefix=self.prefix)
        self.keep, self.W, self.pools = [], [], []
        mat = lambda parts: dict(fmt=fmt, w=parts[0], s=parts[1], zp=parts[2] if len(parts) > 2 else None)  # noqa: E731
        for l in range(NL):
            hw = _chain_weights(7, l, fmt, H, self.XR, QL, self.NQ, E)
            dl = make_layer(fmt, H, I, E, TOPK, NS=4, seed=40 + l, shared="fp8").upload()
            shape = (pages, PAGE, Hkv, D)
            k, v = (torch.randn(shape, generator=g) for _ in range(2))
            ks, vs = (torch.rand(Hkv, generator=g).mul(0.02).add(0.02) for _ in range(2))
            if cache == "e4m3":
                k, v = ((t / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8).cuda() for t, s in ((k, ks), (v, vs)))
                scales = ks.cuda(), vs.cuda()
            else:
                k, v, scales = k.to(kv.BF16).cuda(), v.to(kv.BF16).cuda(), (None, None)
            w = {n: gpu.dev(hw[n]) for n in ("attn_norm", "ffn_norm", "xproj", "router")}
            qn, kn = ((torch.randn(D, generator=g) * 0.1 + 1.0).to(kv.BF16).cuda() for _ in range(2))
            qb, op = ([gpu.dev(p) for p in hw[n]] for n in ("qb", "oproj"))
            w.update(qb=mat(qb), oproj=mat(op), moe=dl.w, ws=gpu.empty(lib.decode_ws_bytes(dl.w), 0), cache=lib.kv_cache(k, v, *scales), q_norm=qn, k_norm=kn)
            self.W.append(w)
            self.pools.append((k, v, scales))
            self.keep.append((hw, dl))
        self.head_h = orc.normal_bf16(7, 997, (VP, H), 0.03)
        self.head = dict(fmt=abi.FMT_BF16, w=gpu.dev(self.head_h), s=None, zp=None)
        self.fin = gpu.dev(orc.f32_to_bf16(1.0 + orc.normal_f32(7, 998, (H,), 0.1)))
        self.ws = torch.zeros(lib.attn_ws_bytes(self.W[0]["cache"], self.batch, Hq), dtype=torch.uint8, device="cuda")
        self.att = Attention(self.batch, Hq, self.ws, rope=self.rope, rot=ROT)
        self.vws = torch.zeros(lib.spec_verify_ws_bytes(self.B, self.M, V), dtype=torch.uint8, device="cuda")
        self.draft, self.tokens = (torch.zeros(self.M, dtype=torch.int32, device="cuda") for _ in range(2))
        self.accepted = torch.zeros(self.B, dtype=torch.int32, device="cuda")
        self.u, self.us = torch.zeros(self.M, device="cuda"), torch.zeros(self.B, device="cuda")
        self.qprob, self.temp = torch.zeros(self.M, V, device="cuda"), torch.ones(self.B, device="cuda")
        self.x0 = torch.zeros(self.M * H, dtype=kv.BF16, device="cuda")
        self.ch = LayerChain(self.M, H, self.XR, QL, self.NQ, E, 1.0, lambda n: gpu.empty(n, 0), V=VP)

    def inputs(self, step, lens):
        """a step's residual rows, drafts, random numbers and lengths, in place"""
        g = torch.Generator().manual_seed(100 + step)
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.x0.copy_(torch.randn(self.M * H, generator=g))
        self.draft.copy_(torch.randint(0, V, (self.M,), generator=g))
        self.qprob.copy_(torch.softmax(torch.randn(self.M, V, generator=g) * 0.5, -1))
        self.u.copy_(torch.rand(self.M, generator=g) * 0.6)
        self.us.copy_(torch.rand(self.B, generator=g))
        self.temp.copy_(torch.tensor([0.0 if b == 1 else 0.8 for b in range(self.B)]))

    def step(self, tap=None, fused=False):
        ch = self.ch
        ch.res[ch.cur].view(kv.BF16).copy_(self.x0)
        ch.yr.zero_()
        for l, w in enumerate(self.W):
            ch.layer(w, fused=fused, up=0, attn=self.att, tap=None if tap is None else lambda name, l=l: tap(l, name))
        ch.finish(self.fin)
        ch.cur ^= 1   # (the next step begins in the same buffers, so that a captured one is the same call)
        ch.head(self.head, V, self.draft, self.u, self.us, self.tokens, self.accepted, self.vws, max(self.rows), cu_rows=self.cu, q=self.qprob, temp=self.temp)

    def results(self):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.tokens, self.accepted, self.ch.xn, self.ch.vocab, self.ch.att)] + [t.clone() for k, v, _ in self.pools for t in (k, v)]


def _rows_of(m, lens):
    return [(b, i, int(m.first[b]) + i, lens[b] - n + i) for b, n in enumerate(m.rows) for i in range(n)]


def _check_append(m, l, lens, q_in, xg, before):
    """queries, and the cache's places of the step's rows, to an f32 chain's error and one rounding; every other place as it was"""
    w, (k, v, (ks, vs)) = m.W[l], m.pools[l]
    q_out = m.ch.q.view(kv.BF16).view(m.M, m.Hq, m.D).cpu().double()
    D, Hkv = m.D, m.Hkv
    half = {"bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}[m.fmt]
    # f32 norm of D squares, its root, two products and a rotation: below D + 16 roundings of 2^-24 of the pair's size
    f32 = (D + 16) * 2.0 ** -24
    new = [t.clone() for t in before]
    for b, i, r, t in _rows_of(m, lens):
        cs = m.rope[P + t].cpu().double()
        y, mag = kv.append64(q_in[r], w["q_norm"].cpu(), cs, ROT, 0, False, 1e-5)
        assert bool(((q_out[r] - y).abs() <= 2.0 ** -8 * y.abs() + 2 * f32 * mag + 1e-30).all()), (l, r, "queries")
        kx, vx = (xg[r, QL + j * Hkv * D:QL + (j + 1) * Hkv * D].view(Hkv, D) for j in range(2))
        y, mag = kv.append64(kx, w["k_norm"].cpu(), cs, ROT, 0, False, 1e-5)
        page, at = int(m.table[b, t // PAGE]), t % PAGE
        for pool, was, x, s, mg in ((k, new[0], y, ks, mag), (v, new[1], vx, vs, vx.abs())):
            got = pool[page, at].cpu()
            sc = torch.ones(Hkv, 1, dtype=torch.float64) if s is None else s.cpu().double()[:, None]
            d = got.double() if s is None else got.view(torch.float8_e4m3fn).double()
            want = (x / sc).clamp(-kv.E4M3_MAX, kv.E4M3_MAX) if s is not None else x
            tiny = 0.0 if s is None else 2.0 ** -10    # e4m3's subnormal step is 2^-9
            assert bool(((d - want).abs() <= half * want.abs() * (1 + 1e-6) + 2 * f32 * mg / sc + tiny + 1e-30).all()), (l, r, "cache")
            was[page, at] = pool[page, at]
    assert torch.equal(new[0], k) and torch.equal(new[1], v), (l, "a place of no row changed")


def _check_attn(m, l, lens):
    k, v, (ks, vs) = m.pools[l]
    val = lambda pool, s: (pool.double() if s is None else pool.view(torch.float8_e4m3fn).double() * s.double()[:, None]).cpu()  # noqa: E731
    kk, vv = val(k, ks), val(v, vs)
    q, got = (t.view(kv.BF16).view(m.M, m.Hq, m.D).cpu().double() for t in (m.ch.q, m.ch.att))
    G, pre = m.Hq // m.Hkv, m.prefix.cpu().long()
    for b, i, r, t in _rows_of(m, lens):
        mine = m.table[b].cpu().long()
        kt, vt = (torch.cat([x[pre].reshape(-1, m.Hkv, m.D)[:P], x[mine].reshape(-1, m.Hkv, m.D)[:t + 1]]) for x in (kk, vv))
        for h in range(m.Hq):
            a = kt[:, h // G] @ q[r, h] * m.D ** -0.5
            p = torch.softmax(a, 0)
            o, mag = p @ vt[:, h // G], p @ vt[:, h // G].abs()
            err = float((q[r, h].abs() @ kt[:, h // G].abs().T).amax()) * m.D ** -0.5 * (m.D + 8) * 2.0 ** -24
            assert bool(((got[r, h] - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -14 + 3 * err) * mag + 1e-30).all()), (l, r, h)


@pytest.mark.parametrize("Hq,Hkv,D,cache", [(8, 2, 128, "bf16"), (8, 2, 128, "e4m3"), (4, 1, 256, "bf16"), (10, 5, 64, "e4m3")])
def test_steps_of_drafting_sequences(Hq, Hkv, D, cache):
    m = Model([3, 1, 4], Hq, Hkv, D, cache)
    lens = [3 + 13, 1, 4 + 29]
    for step in range(3):
        m.inputs(step, lens)
        before, q_in, xg = {}, {}, {}

        def tap(l, name):
            torch.cuda.synchronize()
            if name == "qb":
                before[l] = [t.clone() for t in m.pools[l][:2]]
                q_in[l] = m.ch.q.view(kv.BF16).view(m.M, Hq, D).cpu().double()
                xg[l] = m.ch.xg.view(kv.BF16).view(m.M, m.XR).cpu().double()
            elif name == "append":
                _check_append(m, l, lens, q_in[l], xg[l], before[l])
            elif name == "attn":
                _check_attn(m, l, lens)
            elif name == "oproj":   # the projection reads attention's rows
                x, hw = gpu.host(m.ch.att, np.uint16, (m.M, m.NQ)), m.keep[l][0]["oproj"]
                o = orc.gemv(x, abi.FMT_FP8, hw[0], hw[1], None, H, m.NQ, abi.OUT_F32)
                worst, bad = check_sums(gpu.host(m.ch.part, np.float32, (m.M, H)), o["yd"], o["ymag"], 1e-4)
                assert bad == 0, (l, worst)
        m.step(tap)
        torch.cuda.synchronize()
        logits = gpu.host(m.ch.vocab, np.float32, (m.M, VP))
        o = orc.gemv(gpu.host(m.ch.xn, np.uint16, (m.M, H)), abi.FMT_BF16, m.head_h, None, None, VP, H, abi.OUT_F32)
        worst, bad = check_sums(logits, o["yd"], o["ymag"], 1e-4)
        assert bad == 0, ("head", worst)
        want = kv.verify64(logits[:, :V], m.draft.cpu().numpy(), m.u.cpu().numpy(), m.us.cpu().numpy(), m.rows, q=m.qprob.cpu().numpy(), temp=m.temp.cpu().numpy())
        assert np.array_equal(m.tokens.cpu().numpy(), want[0]) and np.array_equal(m.accepted.cpu().numpy(), want[1]), (step, want)
        # what was refused is not a token of the sequence: the next step's rows take its places
        lens = [L - n + 1 + int(a) + n for L, n, a in zip(lens, m.rows, want[1])]
        assert max(lens) <= PER * PAGE


@pytest.mark.parametrize("fused", [False, True])
def test_a_captured_step_replays_as_the_eager_one(fused):
    m = Model([2, 3], 8, 2, 128, "e4m3")
    start = [[t.clone() for t in p[:2]] for p in m.pools]
    plans = [[20, 3], [47, 80], [2, 33], [80, 61]]

    def reset():
        for p, s in zip(m.pools, start):
            p[0].copy_(s[0]), p[1].copy_(s[1])
    want = []
    for i, lens in enumerate(plans):
        reset()
        m.inputs(i, lens)
        m.step(fused=fused)
        want.append(m.results())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.step(fused=fused)
    for i, lens in list(enumerate(plans)) + [(1, plans[1])]:
        reset()
        m.inputs(i, lens)
        g.replay()
        for a, b in zip(m.results(), want[i]):
            assert torch.equal(a, b), (i, a.shape)
        torch.randn(1 << 16, device="cuda").sum().item()


def test_chain_refuses_what_does_not_fit():
    m = Model([2, 2], 8, 2, 128, "bf16")
    other = lib.kv_batch(3, 2, 16, m.lens, m.table, cu_rows=m.cu)
    for att in (Attention(other, 8, m.ws), Attention(m.batch, 4, m.ws)):
        with pytest.raises(lib.DsgxError):
            m.ch.layer(m.W[0], up=0, attn=att)
    with pytest.raises(lib.DsgxError):
        m.ch.head(m.head, VP + 1, m.draft, m.u, m.us, m.tokens, m.accepted, m.vws, 2)
    with pytest.raises(lib.DsgxError):
        m.ch.head(m.head, V, m.draft, m.u, m.us, m.tokens[:3], m.accepted, m.vws, 2)
    torch.cuda.synchronize()
