"""lib.kv_append against the definition in 64 bits: norm and rotation forms, cache formats and layouts, rows that are not stored."""
import pytest
import torch

from dsgx10_amd import lib
from tests import kv

pytestmark = pytest.mark.gpu


def _run(s, rot, off, pairs, norm, eps=1e-5, seed=1, pos=None, table=None, in_place=False, with_q=True, scale=1.7, dead_rows=()):
    """appends random rows and checks q and both pools whole, bit for bit where nothing was to be written"""
    g = torch.Generator().manual_seed(seed)
    Hq, Hkv, D, R = s.Hq, s.Hkv, s.D, s.R
    W = (Hq + 2 * Hkv) * D + 8                      # rows of a fused projection, with something behind them
    x = (torch.randn(R, W, generator=g) * scale).to(kv.BF16)
    dx = x.cuda()
    wq, wk = ((torch.randn(D, generator=g) * 0.1 + 1).to(kv.BF16) for _ in range(2)) if norm else (None, None)
    rope = kv.rope_table(s.P + max(s.lens) + 3, rot) if rot and table is None else table
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    qo = dx if in_place else torch.full((R, Hq * D), 7.0, dtype=kv.BF16, device="cuda")
    before = [p.clone() for p in (s.kpool, s.vpool)]
    keep = [up(wq), up(wk), up(rope), up(pos)]
    q_args = dict(q=dx, ldq=W, Hq=Hq, q_out=qo, ldqo=W if in_place else Hq * D) if with_q else {}
    lib.kv_append(s.cache, s.batch, dx[:, Hq * D:], W, dx[:, (Hq + Hkv) * D:], W, q_norm=keep[0], k_norm=keep[1], eps=eps, rope=keep[2], rot=rot, rot_off=off, pairs=pairs, pos=keep[3],
                  **q_args)
    torch.cuda.synchronize()
    xd = x.double()
    want = [p.clone().cpu() for p in before]
    for b, n in enumerate(s.rows):
        for i in range(n):
            r, t = int(s.first[b]) + i, s.lens[b] - n + i
            at = s.P + t if pos is None else int(pos[r])
            cs = rope[at].double() if rot else None
            heads = xd[r, :(Hq + 2 * Hkv) * D].view(-1, D)
            if with_q:
                y, mag = kv.append64(heads[:Hq], wq, cs, rot, off, pairs, eps)
                got = qo[r, :Hq * D].cpu().double().view(Hq, D)
                assert bool(((got - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -19 * mag).all()), (r, float((got - y).abs().max()))
            if r in dead_rows:
                continue
            page = s.table_rows[b][t // s.page]
            for j, (pool, sc) in enumerate(((s.kpool, s.ks), (s.vpool, s.vs))):
                h = heads[Hq + j * Hkv:Hq + (j + 1) * Hkv]
                y, mag = kv.append64(h, wk if j == 0 else None, cs, rot if j == 0 else 0, off, pairs, eps) if j == 0 else (h, h.abs())
                raw = pool[page, t % s.page].cpu()
                if s.fmt == "bf16":
                    tol = 2.0 ** -8 * y.abs() + (2.0 ** -19 * mag if j == 0 else 0.0)
                    if j == 1:
                        assert torch.equal(raw.double(), y)
                    assert bool(((raw.double() - y).abs() <= tol).all())
                else:
                    # e4m3: half a step (2^-4 of the value, 2^-10 among the smallest), past +-448 the end
                    c = (y / sc.cpu().double()[:, None]).clamp(-448, 448)
                    m = mag / sc.cpu().double()[:, None]
                    got = raw.view(torch.float8_e4m3fn).double()
                    assert bool(((got - c).abs() <= 2.0 ** -4 * c.abs() + 2.0 ** -10 + 2.0 ** -18 * m).all())
                want[j][page, t % s.page] = raw
    for pool, w in zip((s.kpool, s.vpool), want):   # every other place of the pools as it was
        as_int = (lambda t: t.contiguous().view(torch.int16) if s.fmt == "bf16" else t.contiguous())
        assert torch.equal(as_int(pool.cpu()), as_int(w))
    return qo


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,rot,off", [(8, 2, 128, 128, 0), (64, 1, 256, 64, 192), (4, 4, 64, 64, 0), (5, 5, 64, 32, 16), (6, 3, 128, 16, 112), (3, 1, 256, 256, 0), (7, 7, 128, 64, 0)])
def test_forms(Hq, Hkv, D, rot, off, norm, pairs, fmt):
    s = kv.Step([1, 3], [1, 40], prefix=9, Hq=Hq, Hkv=Hkv, D=D, fmt=fmt, seed=D + rot)
    _run(s, rot, off, pairs, norm)


@pytest.mark.parametrize("layout", ["thd", "htd", "kv"])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_layouts(page, layout):
    for fmt in ("bf16", "e4m3"):
        s = kv.Step([5, 1, 17], [5, 1, 50], page=page, layout=layout, fmt=fmt, seed=page)
        _run(s, 64, 0, False, True)


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 130])
def test_batches(B):
    s = kv.Step([(b * 7) % 4 for b in range(B - 1)] + [3], [(b * 7) % 4 + b for b in range(B - 1)] + [20], Hq=4, Hkv=1, seed=B)
    _run(s, 128, 0, False, True)


def test_rows_without_cu():
    s = kv.Step([3, 3], [3, 77], cu=False, seed=2)
    _run(s, 128, 0, True, True)


def test_a_prompt():
    s = kv.Step([300], [333], Hq=8, Hkv=2, page=64, seed=3)
    _run(s, 64, 0, False, True)


def test_in_place_no_rotation_and_keys_alone():
    _run(kv.Step([2, 2], [2, 30], seed=4), 128, 0, False, True, in_place=True)
    _run(kv.Step([2, 2], [2, 30], seed=5), 0, 0, False, True)
    _run(kv.Step([2, 2], [2, 30], seed=6), 0, 0, False, False)
    _run(kv.Step([2, 2], [2, 30], seed=7), 64, 0, False, True, with_q=False)


def test_given_positions():
    s = kv.Step([2, 3], [9, 30], seed=8)
    _run(s, 128, 0, False, True, pos=torch.tensor([5, 0, 900, 901, 17], dtype=torch.int32), table=kv.rope_table(1000, 128))


def test_far_positions_of_a_table():
    s = kv.Step([1], [3], seed=9)
    _run(s, 64, 0, False, False, pos=torch.tensor([131071], dtype=torch.int32), table=kv.rope_table(131072, 64))


def test_saturation_nan_and_tiny_values():
    s = kv.Step([1], [4], Hq=2, Hkv=1, fmt="e4m3", seed=10)
    _run(s, 0, 0, False, False, scale=40.0)
    _run(s, 0, 0, False, False, scale=1e-4)
    x = torch.zeros(1, 4 * s.D, dtype=kv.BF16, device="cuda")
    x[0, 2 * s.D:2 * s.D + 4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0], device="cuda")
    qo = torch.zeros(1, 2 * s.D, dtype=kv.BF16, device="cuda")
    lib.kv_append(s.cache, s.batch, x[:, 2 * s.D:], 4 * s.D, x[:, 3 * s.D:], 4 * s.D, q=x, ldq=4 * s.D, Hq=2, q_out=qo, ldqo=2 * s.D)
    got = s.kpool[s.table_rows[0][0], 3, 0, :4].view(torch.float8_e4m3fn).float().cpu()
    assert got[0] == 448 and got[1] == -448 and torch.isnan(got[2]) and got[3] == 0


def test_tokens_without_a_place_are_not_stored():
    # a bad page, a table that ends, more rows than tokens: q is made all the same
    s = kv.Step([3, 2, 3], [20, 40, 5], page=16, Hq=4, Hkv=2, seed=11)
    s.t_table[1, 2] = s.npages          # tokens 38, 39 of sequence 1
    s.table_rows[1][2] = 0
    _run(s, 64, 0, False, True, dead_rows=(3, 4))
    s = kv.Step([2, 1], [2, 20], page=16, Hq=4, Hkv=2, seed=12)
    s.t_lens[0] = 1                      # row 0 has no token, row 1 is token 0
    s.t_lens[1] = 2 ** 30                # past the table
    pos = torch.tensor([0, 1, 2], dtype=torch.int32)
    before = [p.clone() for p in (s.kpool, s.vpool)]
    dx = torch.randn(3, 8 * s.D).to(kv.BF16).cuda()
    qo, rope = torch.zeros(3, 4 * s.D, dtype=kv.BF16, device="cuda"), kv.rope_table(40, 64).cuda()
    lib.kv_append(s.cache, s.batch, dx[:, 4 * s.D:], 8 * s.D, dx[:, 6 * s.D:], 8 * s.D, q=dx, ldq=8 * s.D, Hq=4, q_out=qo, ldqo=4 * s.D, rope=rope, rot=64, pos=pos.cuda())
    torch.cuda.synchronize()
    page = s.table_rows[0][0]
    for j, (pool, old) in enumerate(zip((s.kpool, s.vpool), before)):
        assert bool(torch.isfinite(pool[page, 0]).all())
        old[page, 0] = pool[page, 0]
        assert torch.equal(pool.view(torch.int16), old.view(torch.int16))
    assert bool(torch.isfinite(qo).all())
    assert torch.equal(s.vpool[page, 0].reshape(-1).cpu(), dx[1, 6 * s.D:].cpu())


def test_a_position_outside_the_table():
    s = kv.Step([3], [20], Hq=2, Hkv=1, seed=13)
    before = s.kpool.clone()
    dx = torch.randn(3, 4 * s.D).to(kv.BF16).cuda()
    qo, rope = torch.zeros(3, 2 * s.D, dtype=kv.BF16, device="cuda"), kv.rope_table(10, 64).cuda()
    pos = torch.tensor([10, -1, 9], dtype=torch.int32, device="cuda")
    lib.kv_append(s.cache, s.batch, dx[:, 2 * s.D:], 4 * s.D, dx[:, 3 * s.D:], 4 * s.D, q=dx, ldq=4 * s.D, Hq=2, q_out=qo, ldqo=2 * s.D, rope=rope, rot=64, pos=pos)
    torch.cuda.synchronize()
    qv = qo.float().view(3, 2, s.D).cpu()
    assert bool(torch.isnan(qv[:2, :, :64]).all()) and bool(torch.isfinite(qv[:2, :, 64:]).all()) and bool(torch.isfinite(qv[2]).all())
    page = s.table_rows[0][1]
    changed = (s.kpool.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1).nonzero().cpu().tolist()
    assert changed == [[page, 3]]        # token 19 alone


def test_captured_append_replays():
    s = kv.Step([2], [40], Hq=4, Hkv=2, seed=15)
    dx = torch.randn(2, 8 * s.D).to(kv.BF16).cuda()
    qo, rope = torch.zeros(2, 4 * s.D, dtype=kv.BF16, device="cuda"), kv.rope_table(64, 128).cuda()
    call = lambda: lib.kv_append(s.cache, s.batch, dx[:, 4 * s.D:], 8 * s.D, dx[:, 6 * s.D:], 8 * s.D, q=dx, ldq=8 * s.D, Hq=4, q_out=qo, ldqo=4 * s.D, rope=rope, rot=128)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for L in (40, 2, 17, 40):
        s.t_lens.fill_(L)
        call()
        torch.cuda.synchronize()
        want, pools = qo.clone(), [p.clone() for p in (s.kpool, s.vpool)]
        for p in (s.kpool, s.vpool):
            p.zero_()
        qo.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want)
        for p, w in zip((s.kpool, s.vpool), pools):
            for t in (L - 2, L - 1):
                at = (s.table_rows[0][t // s.page], t % s.page)
                assert torch.equal(p[at], w[at])
