"""lib.spec_verify against the definition in f64 (tokens and counts equal), and the distribution that it draws from."""
import ctypes as C

import numpy as np
import pytest
import torch

from dsgx10_amd import abi, lib
from tests import kv

pytestmark = pytest.mark.gpu


def _inputs(rows, V, kind, seed, sharp=False, temps=None, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    R = sum(rows)
    logits = torch.randn(R, V, generator=g) * spread
    T = torch.ones(len(rows)) if temps is None else torch.tensor(temps)
    of = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    near = torch.softmax(logits / T[of, None].clamp(min=0.3) + 0.5 * torch.randn(R, V, generator=g), -1)
    draft = (near.argmax(-1) if sharp else torch.multinomial(near, 1, generator=g)[:, 0]).to(torch.int32)
    target = logits.to(torch.bfloat16) if kind == "bf16" else torch.softmax(logits, -1) if kind == "prob" else logits
    return dict(target=target, draft=draft, u=torch.rand(R, generator=g), us=torch.rand(len(rows), generator=g), q=None if sharp else near,
                temp=None if temps is None or kind == "prob" else T, probs=kind == "prob", rows=rows)


def _call(d, ld=0, cu=True, stream=None, ws=None):
    rows, V = d["rows"], d["target"].shape[1]
    R, B = sum(rows), len(rows)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    t = d["target"]
    if ld:
        t = torch.cat([t, torch.full((R, ld), float("nan"), dtype=t.dtype)], 1)
    c = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32).cuda() if cu else None
    tokens, accepted = torch.full((R,), 99, dtype=torch.int32, device="cuda"), torch.full((B,), 99, dtype=torch.int32, device="cuda")
    if ws is None:
        ws = torch.zeros(lib.spec_verify_ws_bytes(B, R, V), dtype=torch.uint8, device="cuda")
    keep = [up(t), up(d["draft"]), up(d["u"]), up(d["us"]), up(d["q"]), up(d["temp"])]
    lib.spec_verify(keep[0], V, keep[1], keep[2], keep[3], tokens, accepted, ws, max(rows), cu_rows=c, q=keep[4], temp=keep[5], probs=d["probs"], ldt=V + ld, stream=stream)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), accepted.cpu().numpy()


def _want(d):
    n = lambda t: None if t is None else t.numpy()  # noqa: E731
    return kv.verify64(d["target"].float().numpy(), n(d["draft"]), n(d["u"]), n(d["us"]), d["rows"], n(d["q"]), n(d["temp"]), d["probs"])


def _check(d, **kw):
    got, want = _call(d, **kw), _want(d)
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    return got


@pytest.mark.parametrize("sharp", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16", "prob"])
@pytest.mark.parametrize("V", [1, 2, 7, 63, 1000, 4095, 4096, 4097, 8200, 32768, 100003])
def test_vocabularies(V, kind, sharp):
    rows = [1, 2, 5, 3, 8] if V < 20000 else [5, 1, 3]
    for seed in range(3 if V < 20000 else 1):
        _check(_inputs(rows, V, kind, 10 * V + seed, sharp))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_temperatures_and_greedy_streams(kind):
    for seed in range(6):
        _check(_inputs([3, 4, 1, 6, 2], 5000, kind, seed, seed % 2 == 1, [0.7, 0.0, 1.3, 0.0, 0.25]))


def test_greedy_ties_go_to_the_lowest_id():
    d = _inputs([2, 1], 9000, "bf16", 3, True, [0.0, 0.0])
    d["target"][:, [17, 4096, 8999]] = 50.0
    d["draft"][0] = 17
    tokens, accepted = _check(d)
    assert accepted[0] == 1 and tokens[1] == 17 and tokens[2] == 17


def test_rows_of_other_strides_and_without_cu():
    for kind in ("f32", "bf16", "prob"):
        for ld in (1, 3, 8):
            _check(_inputs([3, 3], 1001, kind, ld), ld=ld, cu=False)


def test_masked_ids_are_never_drawn():
    d = _inputs([3, 2, 1], 5000, "f32", 5)
    d["target"][:, 100:] = -float("inf")
    tokens, _ = _check(d)
    assert tokens.max() < 100
    d["target"][:, :] = -float("inf")
    d["target"][:, 4500] = 1.0
    tokens, _ = _check(d)
    assert set(tokens) <= {4500, -1} or d["draft"].eq(4500).any()


def test_random_numbers_at_the_ends():
    for kind in ("f32", "prob"):
        d = _inputs([4, 2], 3000, kind, 6)
        for u, us in ((0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (0.0, 1 - 2.0 ** -24)):
            d["u"].fill_(u)
            d["us"].fill_(us)
            _check(d)


def test_a_drafter_equal_to_the_target_is_always_accepted():
    d = _inputs([6, 3], 2000, "prob", 7)
    d["q"] = d["target"].clone()
    d["u"].fill_(0.999)
    _, accepted = _check(d)
    assert list(accepted) == [5, 2]


def test_nothing_left_of_the_difference_draws_from_the_target():
    d = _inputs([2], 50, "prob", 8)
    d["q"] = d["target"] * 2
    d["u"].fill_(0.9)                    # 0.9 * 2p >= p: refused, and p - q is nowhere positive
    _, accepted = _check(d)
    assert accepted[0] == 0


def test_bad_drafts_and_rows_that_cannot_be_drawn_from():
    d = _inputs([3, 3, 3, 2], 700, "f32", 9)
    d["draft"][0], d["draft"][3] = -1, 700
    d["target"][6, 5] = float("nan")     # sequence 2's first row
    d["target"][9, 5] = float("inf")     # sequence 3's
    tokens, accepted = _call(d)
    assert accepted[0] == accepted[1] == accepted[2] == accepted[3] == 0
    assert 0 <= tokens[0] < 700 and 0 <= tokens[3] < 700 and tokens[6] == -1 and tokens[9] == -1
    assert list(tokens[1:3]) == [-1, -1]
    d = _inputs([2], 700, "bf16", 9, True, [0.0])
    d["target"][0, 3] = float("nan")
    tokens, accepted = _call(d)
    assert accepted[0] == 0 and tokens[0] == -1


def test_sequences_without_rows():
    d = _inputs([2, 3], 300, "f32", 10)
    want = _want(d)
    d["rows"] = [2, 0, 3]
    d["us"] = torch.tensor([d["us"][0], 0.5, d["us"][1]])
    tokens, accepted = _call(d)
    assert np.array_equal(tokens, want[0]) and list(accepted) == [want[1][0], 0, want[1][1]]


def test_the_draws_follow_the_target():
    """Whatever the drafter, the first token of a sequence has the target's distribution: over N sequences an id of probability p is
    counted N p times, give or take five standard deviations (a wrong result once in 10^6 ids)."""
    N, V = 4000, 12
    g = torch.Generator().manual_seed(11)
    p, q = (torch.softmax(torch.randn(V, generator=g) * 1.2, -1) for _ in range(2))
    d = dict(target=p.repeat(2 * N, 1), q=q.repeat(2 * N, 1), draft=torch.multinomial(q, 2 * N, True, generator=g).to(torch.int32), u=torch.rand(2 * N, generator=g),
             us=torch.rand(N, generator=g), temp=None, probs=True, rows=[2] * N)
    tokens, _ = _check(d)
    counts = np.bincount(tokens[0::2], minlength=V)
    sd = np.sqrt(N * p.numpy() * (1 - p.numpy()))
    assert np.all(np.abs(counts - N * p.numpy()) <= 5 * sd)


def test_captured_call_replays_on_new_numbers():
    d = _inputs([4, 2, 1], 9001, "f32", 12, temps=[1.0, 0.6, 0.9])
    R, B, V = 7, 3, 9001
    dev = {k: v.cuda() for k, v in d.items() if isinstance(v, torch.Tensor)}
    cu = torch.tensor([0, 4, 6, 7], dtype=torch.int32, device="cuda")
    tokens, accepted = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    ws = torch.zeros(lib.spec_verify_ws_bytes(B, R, V), dtype=torch.uint8, device="cuda")
    call = lambda: lib.spec_verify(dev["target"], V, dev["draft"], dev["u"], dev["us"], tokens, accepted, ws, 4, cu_rows=cu, q=dev["q"], temp=dev["temp"])  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        d["u"], d["us"] = torch.rand(R, generator=g), torch.rand(B, generator=g)
        dev["u"].copy_(d["u"])
        dev["us"].copy_(d["us"])
        graph.replay()
        torch.cuda.synchronize()
        want = _want(d)
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(accepted.cpu().numpy(), want[1])
        assert np.array_equal(_call(d, ws=ws)[0], want[0])


@pytest.mark.parametrize("kind", ["f32", "bf16", "prob"])
@pytest.mark.parametrize("rows,V", [([3] * 40, 70001), ([4, 1, 7] * 100, 9000), ([2], 200003)])
def test_pieces_of_several_chunks(rows, V, kind):
    d = _inputs(rows, V, kind, 77, False, None if kind == "prob" else [0.0 if b % 5 == 1 else 0.9 for b in range(len(rows))])
    if kind != "prob":
        # a maximum that rises from chunk to chunk, and a first chunk that holds nothing
        d["target"] += torch.arange(V) // 4096 * 0.125
        d["target"][1::2, :4096] = -float("inf")
    _check(d)


@pytest.mark.parametrize("where", [5, 69000])
def test_a_nan_or_infinity_in_any_chunk_refuses_the_row(where):
    rows = [3] * 40
    for value in (float("nan"), float("inf")):
        d = _inputs(rows, 70001, "f32", 78, True, [0.7] * 40)
        d["target"][0, where] = value
        tokens, accepted = _call(d)
        assert accepted[0] == 0 and tokens[0] == -1
        want = _want({**d, "target": d["target"].nan_to_num(0.0, posinf=0.0)})
        assert np.array_equal(tokens[3:], want[0][3:]) and np.array_equal(accepted[1:], want[1][1:])


@pytest.mark.parametrize("T", [1e-3, 1e-6, 3e-9, 1e-10, 1e-30, 1e-44])
def test_temperatures_near_zero(T):
    """down to where 700 T is less than a step of the maximum; then only the largest logits' ids are left, evenly"""
    for sharp in (False, True):
        d = _inputs([3, 2, 4], 6000, "f32", 79, sharp, [T] * 3)
        d["target"][2, [7, 4500]] = 30.0
        _check(d)


@pytest.mark.parametrize("T", [1e6, 1e30, 3e38])
def test_temperatures_that_flatten_everything(T):
    for sharp in (False, True):
        d = _inputs([3, 2, 4], 6000, "f32", 80, sharp, [T] * 3)
        d["target"][:, 100:4500] = -float("inf")
        _check(d)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_drafts_border_without_probabilities(kind):
    """u on either side of p(draft), 4 * 10^-6 of it away: the border moves by 10^-6 at most, u is rounded to 2^-24"""
    d = _inputs([2] * 60, 30011, kind, 95, True, [0.4 + 0.05 * b for b in range(60)])
    p = torch.softmax(d["target"].double() / d["temp"].double().repeat_interleave(2)[:, None], -1)
    at = p.gather(1, d["draft"].long()[:, None])[:, 0]
    side = torch.where(torch.arange(120) // 2 % 2 == 0, 1 - 4e-6, 1 + 4e-6)
    d["u"] = (at * side).float()
    tokens, accepted = _check(d)
    assert accepted.tolist() == [1, 0] * 30


def test_no_rows_at_all():
    z = lambda n, t=torch.float32: torch.zeros(n, dtype=t, device="cuda")  # noqa: E731
    ids, ws = z(4, torch.int32), z(lib.spec_verify_ws_bytes(3, 0, 500), torch.uint8)
    for kind in (torch.float32, torch.bfloat16):
        accepted = torch.full((3,), 9, dtype=torch.int32, device="cuda")
        a = abi.VerifyIn(z(500, kind).data_ptr(), None, ids.data_ptr(), ids.data_ptr(), z(4).data_ptr(), z(3).data_ptr(), None, 500, 500, int(kind == torch.bfloat16), 500, 3, 0, 2)
        assert lib.lib().dsgx_spec_verify(C.byref(a), ids.data_ptr(), accepted.data_ptr(), ws.data_ptr(), None) == abi.OK
        torch.cuda.synchronize()
        assert accepted.tolist() == [0, 0, 0] and ids.tolist() == [0] * 4


def test_graphs_of_different_sizes_share_a_workspace():
    ds = [_inputs([3] * 40, 70001, "f32", 91, False, [0.8] * 40), _inputs([2, 5], 900, "bf16", 92, True), _inputs([1, 4, 2], 20000, "prob", 93)]
    sizes = [(len(d["rows"]), sum(d["rows"]), d["target"].shape[1]) for d in ds]
    ws = torch.zeros(max(lib.spec_verify_ws_bytes(*n) for n in sizes), dtype=torch.uint8, device="cuda")
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    calls, outs, graphs = [], [], []
    for d, (B, R, V) in zip(ds, sizes):
        g = {k: up(d[k]) for k in ("target", "draft", "u", "us", "q", "temp")}
        cu = torch.tensor(np.concatenate([[0], np.cumsum(d["rows"])]), dtype=torch.int32).cuda()
        tokens, accepted = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
        outs.append((tokens, accepted))
        calls.append(lambda g=g, V=V, o=outs[-1], cu=cu, d=d: lib.spec_verify(g["target"], V, g["draft"], g["u"], g["us"], *o, ws, max(d["rows"]), cu_rows=cu, q=g["q"], temp=g["temp"],
                                                                             probs=d["probs"]))
    for call in calls:
        call()
    torch.cuda.synchronize()
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    for i in (0, 1, 2, 2, 1, 0, 0):
        outs[i][0].fill_(77), outs[i][1].fill_(77)
        graphs[i].replay()
        torch.cuda.synchronize()
        want = _want(ds[i])
        assert np.array_equal(outs[i][0].cpu().numpy(), want[0]) and np.array_equal(outs[i][1].cpu().numpy(), want[1]), i
        torch.randn(1 << 16, device="cuda").sum().item()
