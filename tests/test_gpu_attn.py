"""lib.attn against the definition in 64 bits: head layouts, cache formats and layouts, lengths from nothing to many ranges, prefixes that end
inside a page, rows that see nothing, places that hold NaN, captured and replayed steps."""
import pytest
import torch

from dsgx10_amd import lib
from tests import kv

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (4, 4, 64), (6, 2, 64), (64, 1, 256), (12, 2, 256), (5, 5, 128), (48, 4, 128), (16, 1, 64), (32, 8, 128)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_heads_and_formats(Hq, Hkv, D, fmt):
    s = kv.Step([1, 3, 2], [37, 300, 65], Hq=Hq, Hkv=Hkv, D=D, fmt=fmt, seed=Hq + D)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 2049])
def test_lengths(length, fmt):
    s = kv.Step([1, min(4, length)], [length, length], page=32, fmt=fmt, seed=length)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 100, 128, 257, 1100])
@pytest.mark.parametrize("Hq,Hkv,D,fmt", [(8, 2, 128, "bf16"), (8, 1, 64, "e4m3"), (64, 1, 256, "bf16"), (12, 4, 256, "e4m3")])
def test_prefix(prefix, Hq, Hkv, D, fmt):
    s = kv.Step([2, 1, 5, 1, 3], [40, 1, 129, 16, 70], prefix=prefix, Hq=Hq, Hkv=Hkv, D=D, fmt=fmt, page=16 if prefix % 2 else 64, seed=prefix)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,n,G,max_len", [(9, 1, 8, None), (5, 3, 8, None), (4, 1, 16, 40000), (3, 1, 8, 1), (1, 2, 4, None), (2, 8, 8, None), (1, 12, 8, 9000), (1, 6, 8, None)])
def test_prefix_and_own_tokens_by_every_pair_of_kernels(B, n, G, max_len, D, fmt):
    s = kv.Step([n] * B, [n + (37 * b) % 290 for b in range(B)], prefix=700, Hq=2 * G, Hkv=2, D=D, fmt=fmt, page=16, seed=B + n, max_len=max_len)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("B,n", [(1, 1), (3, 7), (40, 1), (70, 2), (130, 4)])
def test_many_rows_behind_a_prefix(B, n):
    s = kv.Step([n] * B, [n + (7 * b) % 50 for b in range(B)], prefix=333, Hq=16, Hkv=2, D=128, page=16, seed=B)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["thd", "htd", "kv"])
def test_pages_and_layouts(page, layout):
    for fmt in ("bf16", "e4m3"):
        s = kv.Step([2, 1], [page + 3, 2 * page + 17], prefix=page // 2 + 1, page=page, layout=layout, fmt=fmt, seed=page)
        kv.check_attn(s, *s.run())


def test_rows_of_other_strides():
    s = kv.Step([2, 3], [90, 33], prefix=20, seed=4)
    out, lse = s.run(ld_extra=24)
    kv.check_attn(s, out, lse)
    assert bool((out[:, s.Hq * s.D:] == 7).all())  # what lies between the rows stays
    out2, _ = s.run(ld_extra=24, lse=False)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("prefix", [0, 40])
def test_sequences_without_tokens_or_rows(prefix):
    # a sequence without tokens, one with fewer tokens than rows (its first rows see the prefix alone), one without rows, one ordinary
    s = kv.Step([2, 3, 0, 1], [0, 2, 50, 9], prefix=prefix, seed=8)
    out, lse = s.run()
    kv.check_attn(s, out, lse)
    if not prefix:
        assert bool((out[:3] == 0).all()) and bool(torch.isinf(lse[:3]).all())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_unseen_drafts_hold_infinities_and_nans(fmt, D):
    """the keys and values of a later row of the step do not reach an earlier one, whatever they hold"""
    for rows, L in ((4, 41), (7, 130), (3, 3), (6, 20)):
        s = kv.Step([rows, 1], [L, 30], prefix=5, D=D, fmt=fmt, seed=L)
        want = kv.attn64(s)
        for b, hidden in ((0, rows - 2), (0, rows - 1)):
            t = L - rows + hidden
            for i in range(2):
                raw = s.own_kv[b][i]
                if fmt == "bf16":
                    raw[t] = float("nan") if i == 0 else float("inf")
                else:
                    raw.view(torch.uint8)[t] = 0x7F
        s.store()
        out, lse = s.run()
        o, mag, z, err = want
        keep = [i for i in range(s.R) if not (rows - 2 <= i < rows)]
        got = out.double().view(s.R, s.Hq, s.D)[keep]
        tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -14 + 3 * err[..., None]) * mag + 1e-30
        assert bool(((got - o[keep]).abs() <= tol[keep]).all()), (rows, L)
        assert bool(torch.isnan(out.double().view(s.R, s.Hq, s.D)[rows - 2:rows]).all())  # the rows that see them show it


def test_bounds_are_only_plans():
    """more rows and tokens than max_rows and max_len announce"""
    s = kv.Step([9, 2], [700, 900], prefix=70, Hq=16, Hkv=2, max_rows=1, max_len=64, seed=3)
    kv.check_attn(s, *s.run())


def test_bad_pages_are_not_there():
    s = kv.Step([2, 1], [100, 80], prefix=40, page=16, seed=12)
    # sequence 0 loses its pages 1 and 3, the prefix its page 0: as if those tokens did not exist
    s.t_table[0, 1], s.t_table[0, 3], s.t_prefix[0] = -5, s.npages, -1
    out, lse = s.run()
    keep = [t for t in range(100) if t // 16 not in (1, 3)]
    for i in range(2):
        s.pre_kv[i] = s.pre_kv[i][16:]
        s.own_kv[0][i] = s.own_kv[0][i][keep]
    s.P -= 16
    s.lens[0] = len(keep)
    kv.check_attn(s, out, lse)


def test_rows_of_no_sequence_stay():
    s = kv.Step([2, 2, 1], [20, 30, 40], seed=5)
    s.t_cu.copy_(torch.tensor([0, 2, 2, 5], dtype=torch.int32))     # sequence 1 has none; sequence 2 rows 2 .. 4
    s.t_cu[3] = 4                                                    # row 4 belongs to nobody
    s.rows, s.first = [2, 0, 2], [0, 2, 2, 4]
    out, lse = s.run()
    kv.check_attn(s, out, lse, rows=slice(0, 4))
    assert bool((out[4] == 7).all()) and bool((lse[4] == 7).all())
    # bounds out of order or past the rows: those sequences are left out, the others are right
    s.t_cu.copy_(torch.tensor([0, 2, -3, 99], dtype=torch.int32))
    out, lse = s.run()
    kv.check_attn(s, out, lse, rows=slice(0, 2))
    assert bool((out[2:] == 7).all())


def test_lengths_are_cut_to_the_table():
    s = kv.Step([1, 1], [64, 33], page=16, seed=6)
    want = s.run()
    s.t_lens.copy_(torch.tensor([64, -4], dtype=torch.int32))
    out, lse = s.run()
    assert torch.equal(out[0], want[0][0]) and bool((out[1] == 0).all())
    s.t_lens.copy_(torch.tensor([2 ** 31 - 1, 33], dtype=torch.int32))
    out, lse = s.run()
    assert torch.equal(out[0], want[0][0]) and torch.equal(out[1], want[0][1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-3])
def test_scales(scale):
    s = kv.Step([2], [150], seed=7, kscale=0.5)
    kv.check_attn(s, *s.run(scale=scale), scale=scale)


def test_large_scores():
    """scores far apart and far from zero: the maximum is subtracted before anything is raised"""
    for c in (30.0, -30.0):
        s = kv.Step([3], [200], prefix=50, Hq=4, Hkv=2, seed=9, kscale=abs(c))
        kv.check_attn(s, *s.run(scale=c / 30), scale=c / 30)


def test_offsets_past_32_bits():
    """pages that lie more than 2^32 values into the pools"""
    page, Hkv, D = 64, 8, 128
    n = 2 ** 32 // (page * Hkv * D) + 40
    s = kv.Step([2, 1], [200, 90], prefix=70, Hq=16, Hkv=Hkv, D=D, page=page, fmt="e4m3", seed=10)
    pools = [torch.empty(n, page, Hkv, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    shift = n - s.npages
    for pool, old in zip(pools, (s.kpool, s.vpool)):
        pool[shift:] = old
    s.kpool, s.vpool = pools
    s.t_table += shift
    s.t_prefix += shift
    s.cache = lib.kv_cache(*pools, s.ks, s.vs)
    kv.check_attn(s, *s.run())


def test_same_inputs_same_bits_and_shared_workspace():
    s = kv.Step([1, 4, 2], [900, 333, 70], prefix=600, Hq=32, Hkv=4, seed=11)
    other = kv.Step([3], [1500], Hq=32, Hkv=4, seed=13)
    ws = torch.zeros(max(lib.attn_ws_bytes(x.cache, x.batch, 32) for x in (s, other)), dtype=torch.uint8, device="cuda")
    a, za = s.run(ws=ws)
    other.run(ws=ws)
    b, zb = s.run(ws=ws)
    assert torch.equal(a, b) and torch.equal(za, zb)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    c, zc = s.run(ws=ws, stream=stream)
    assert torch.equal(a, c) and torch.equal(za, zc)


def test_captured_step_replays_with_other_lengths():
    """lens, tables and rows are read when the graph runs"""
    s = kv.Step([2, 2], [400, 90], prefix=100, page=16, Hq=16, Hkv=2, seed=14)
    n = s.Hq * s.D
    q, out = s.q.reshape(s.R, n).cuda(), torch.zeros(s.R, n, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(s.R, s.Hq, device="cuda")
    ws = torch.zeros(lib.attn_ws_bytes(s.cache, s.batch, s.Hq), dtype=torch.uint8, device="cuda")
    call = lambda: lib.attn(s.cache, s.batch, q, n, s.Hq, s.D ** -0.5, out, n, ws, lse=lse)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([400, 90], [33, 2], [257, 64], [400, 90]):
        s.t_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        full = s.lens, s.own_kv
        s.lens = lens
        s.own_kv = [[x[:L] for x in pair] for pair, L in zip(full[1], lens)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, z = out.cpu(), lse.cpu()
        kv.check_attn(s, got, z)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out.cpu()) and torch.equal(z, lse.cpu())
        s.lens, s.own_kv = full


@pytest.mark.parametrize("D,Hq,Hkv,L", [(64, 8, 8, 20011), (128, 8, 2, 12000), (256, 4, 1, 9000)])
def test_one_row_over_many_ranges(D, Hq, Hkv, L):
    s = kv.Step([1], [L], Hq=Hq, Hkv=Hkv, D=D, page=64, seed=D)
    kv.check_attn(s, *s.run())


@pytest.mark.parametrize("B,prefix,cu", [(300, 0, True), (300, 40, True), (257, 0, False), (65, 0, False)])
def test_many_sequences(B, prefix, cu):
    rows = [2] * B if not cu else [1 + b % 3 if b % 7 else 0 for b in range(B)]
    s = kv.Step(rows, [rows[b] + (53 * b) % 700 for b in range(B)], prefix=prefix, Hq=4, Hkv=2, D=64, page=32, seed=B, cu=cu)
    kv.check_attn(s, *s.run())


def test_a_prefix_too_long_for_the_wider_form():
    s = kv.Step([1] * 7, [40 + 90 * b for b in range(7)], prefix=32800, Hq=8, Hkv=1, D=64, page=128, fmt="e4m3", seed=21)
    kv.check_attn(s, *s.run())


def _bound(s):
    n = s.Hq * s.D
    t = dict(q=s.q.reshape(s.R, n).cuda(), out=torch.zeros(s.R, n, dtype=torch.bfloat16, device="cuda"), lse=torch.zeros(s.R, s.Hq, device="cuda"))
    return t, lambda ws, stream=None: lib.attn(s.cache, s.batch, t["q"], n, s.Hq, s.D ** -0.5, t["out"], n, ws, lse=t["lse"], stream=stream)


def test_graphs_of_different_batches_share_a_workspace():
    steps = [kv.Step([2, 1, 3], [700, 90, 1300], prefix=500, Hq=16, Hkv=2, seed=31), kv.Step([1] * 5, [900, 20, 3000, 7, 600], Hq=8, Hkv=2, seed=32),
             kv.Step([9], [2000], prefix=300, Hq=16, Hkv=2, seed=33)]
    ws = torch.zeros(max(lib.attn_ws_bytes(s.cache, s.batch, s.Hq) for s in steps), dtype=torch.uint8, device="cuda")
    calls, want, graphs = [_bound(s) for s in steps], [], []
    for s, (t, call) in zip(steps, calls):
        call(ws)
        torch.cuda.synchronize()
        kv.check_attn(s, t["out"].cpu(), t["lse"].cpu())
        want.append((t["out"].clone(), t["lse"].clone()))
    for t, call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(ws)
        graphs.append(g)
    for i in (0, 1, 2, 1, 0, 2, 2, 0):
        calls[i][0]["out"].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(calls[i][0]["out"], want[i][0]) and torch.equal(calls[i][0]["lse"], want[i][1]), i
        torch.randn(1 << 16, device="cuda").sum().item()


def test_two_calls_at_once_on_streams_of_their_own():
    steps = [kv.Step([2, 1, 3], [700, 90, 1300], prefix=500, Hq=16, Hkv=2, seed=31), kv.Step([1] * 5, [900, 20, 3000, 7, 600], Hq=8, Hkv=2, seed=32)]
    calls = [_bound(s) for s in steps]
    wss = [torch.zeros(lib.attn_ws_bytes(s.cache, s.batch, s.Hq), dtype=torch.uint8, device="cuda") for s in steps]
    want = []
    for (t, call), ws in zip(calls, wss):
        call(ws)
        torch.cuda.synchronize()
        want.append(t["out"].clone())
        t["out"].zero_()
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(20):
        for (t, call), ws, st in zip(calls, wss, streams):
            call(ws, stream=st)
    torch.cuda.synchronize()
    for (t, _), w in zip(calls, want):
        assert torch.equal(t["out"], w)
