"""What the attention-side operators refuse, on the CPU: every check fails before a launch."""
import ctypes as C

import pytest
import torch

from dsgx10_amd import abi, lib


def _cache(**kw):
    c = abi.KvCache(0x1000, 0x2000, None, None, 16 * 2 * 128, 2 * 128, 128, abi.FMT_BF16, 2, 128, 16, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _batch(**kw):
    b = abi.KvBatch(0x100, 0x200, 0x300, None, 2, 4, 2, 100, 8, 0)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


BAD_CACHE = [(dict(k=None), abi.EINVAL), (dict(fmt=0), abi.EFORMAT), (dict(fmt=16), abi.EFORMAT), (dict(fmt=abi.KV_E4M3), abi.EINVAL), (dict(D=96), abi.EINVAL), (dict(D=0), abi.EINVAL),
             (dict(page=8), abi.EINVAL), (dict(page=48), abi.EINVAL), (dict(page=2048), abi.EINVAL), (dict(page=0), abi.EINVAL), (dict(Hkv=0), abi.EINVAL), (dict(npages=0), abi.EINVAL),
             (dict(k=0x1008), abi.EINVAL), (dict(tok_stride=252), abi.EINVAL), (dict(tok_stride=64), abi.EINVAL), (dict(head_stride=4), abi.EINVAL), (dict(page_stride=-8), abi.EINVAL)]
BAD_BATCH = [dict(lens=None), dict(table=None), dict(B=0), dict(B=70000), dict(rows=-1), dict(max_rows=0), dict(max_len=-1), dict(table_ld=0), dict(cu_rows=None, rows=5), dict(prefix_len=-1),
             dict(prefix_len=10), dict(table_ld=1 << 27)]


def _append(c, b, **kw):
    a = abi.KvAppendIn(0x1000, 0x2000, 0x3000, 0x4000, None, None, 0x5000, None, 1024, 256, 256, 1024, 8, 64, 0, 0, 100, 1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib().dsgx_kv_append(C.byref(c), C.byref(b), C.byref(a), None)


def _attn(c, b, q=0x1000, ldq=1024, Hq=8, out=0x2000, ldo=1024, ws=0x3000):
    return lib.lib().dsgx_attn(C.byref(c), C.byref(b), q, ldq, Hq, 1.0, out, ldo, None, ws, None)


@pytest.mark.parametrize("bad,code", BAD_CACHE)
def test_caches(bad, code):
    assert _append(_cache(**bad), _batch()) == code and _attn(_cache(**bad), _batch()) == code
    assert lib.lib().dsgx_last_error()
    assert lib.attn_ws_bytes(_cache(**bad), _batch(), 8) == 0


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_batches(bad):
    assert _append(_cache(), _batch(**bad)) == abi.EINVAL and _attn(_cache(), _batch(**bad)) == abi.EINVAL
    assert lib.attn_ws_bytes(_cache(), _batch(**bad), 8) == 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(Hq=0), dict(Hq=-1), dict(rot=8), dict(rot=-16), dict(rot=144), dict(rot_off=8), dict(rot_off=80),
                                 dict(rope=None), dict(rope_len=0), dict(k=0x2002), dict(rope=0x5004), dict(q_norm=0x7002), dict(ldk=252), dict(ldk=128), dict(ldq=1000), dict(ldqo=1020)])
def test_append_arguments(bad):
    assert _append(_cache(), _batch(), **bad) == abi.EINVAL


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(ws=None), dict(Hq=0), dict(Hq=7), dict(Hq=-2), dict(q=0x1008), dict(ws=0x3008), dict(ldq=1000), dict(ldo=1028), dict(ldq=1016)])
def test_attn_arguments(bad):
    assert _attn(_cache(), _batch(), **bad) == abi.EINVAL


def test_no_rows_is_no_launch():
    assert _attn(_cache(), _batch(rows=0)) == abi.OK and _append(_cache(), _batch(rows=0)) == abi.OK


def _verify(tokens=0x100, accepted=0x200, ws=0x300, **kw):
    a = abi.VerifyIn(0x1000, None, 0x2000, 0x3000, 0x4000, 0x5000, None, 1000, 1000, 0, 1000, 2, 6, 3)
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib().dsgx_spec_verify(C.byref(a), tokens, accepted, ws, None)


@pytest.mark.parametrize("bad", [dict(target=None), dict(us=None), dict(tokens=None), dict(accepted=None), dict(ws=None), dict(kind=3), dict(kind=-1), dict(V=0), dict(B=0), dict(rows=70000),
                                 dict(max_rows=0), dict(cu_rows=None, rows=5), dict(draft=None), dict(u=None), dict(ldt=999), dict(q=0x6000, ldq=10), dict(ws=0x304), dict(target=0x1002),
                                 dict(q=0x6002)])
def test_verify_arguments(bad):
    assert _verify(**bad) == abi.EINVAL


def test_python_handles_refuse_what_is_no_cache():
    k = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    assert lib.kv_cache(k, k).Hkv == 2
    for a, b, ks in ((k, k[:3], None), (k, k.permute(0, 2, 1, 3), None), (k.float(), k.float(), None), (k.half(), k.half(), None), (k, k, torch.ones(2)), (k[..., ::2], k[..., ::2], None), (k.to(torch.uint8), k.to(torch.uint8), None)):
        with pytest.raises(lib.DsgxError):
            lib.kv_cache(a, b, ks, ks)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 8, dtype=torch.int32)
    lib.kv_batch(2, 1, 10, lens, table)
    for bad in (dict(lens=lens.long()), dict(table=table[:, ::2]), dict(cu_rows=lens.float())):
        with pytest.raises(lib.DsgxError):
            lib.kv_batch(2, 1, 10, bad.get("lens", lens), bad.get("table", table), cu_rows=bad.get("cu_rows"))


def test_packed_arguments_are_the_structs():
    a = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, -13, 14, 15, 1, 17, 0.5)
    assert lib._APPEND(*a) == bytes(abi.KvAppendIn(*a))
    a = (1, 2, 3, 4, 5, 6, 7, 8, 1 << 40, 2, -11, 12, 13, 14)
    assert lib._VERIFY(*a) == bytes(abi.VerifyIn(*a))


def test_types_of_tensors():
    c, b = _cache(), _batch()
    t = lambda *n, d=torch.float32: torch.zeros(*n, dtype=d)  # noqa: E731
    for kw in (dict(rope=t(4, 16, d=torch.bfloat16), rot=16), dict(pos=t(4, d=torch.int64))):
        with pytest.raises(lib.DsgxError):
            lib.kv_append(c, b, t(64), 256, t(64), 256, **kw)
    i32 = torch.int32
    ok = dict(draft=t(3, d=i32), u=t(3), us=t(1), tokens=t(3, d=i32), accepted=t(1, d=i32), temp=None, cu_rows=None)
    for bad in (dict(draft=t(3, d=torch.int64)), dict(u=t(3, d=torch.float64)), dict(us=t(1, d=torch.bfloat16)), dict(tokens=t(3, d=torch.int64)), dict(accepted=t(1, d=torch.int16)),
                dict(temp=t(1, d=torch.float16)), dict(cu_rows=t(2, d=torch.int64)), dict(us=t(0)), dict(draft=t(2, d=i32)), dict(u=t(1)), dict(cu_rows=t(1, d=i32)), dict(temp=t(0))):
        a = {**ok, **bad}
        with pytest.raises(lib.DsgxError):
            lib.spec_verify(t(3, 50), 50, a["draft"], a["u"], a["us"], a["tokens"], a["accepted"], t(8), 3, cu_rows=a["cu_rows"], temp=a["temp"])


def test_batches_that_miss_lengths():
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    lib.kv_batch(4, 2, 16, i(2), i(2, 3), cu_rows=i(3))
    for kw in (dict(lens=i(1)), dict(cu_rows=i(2)), dict(table=i(6))):
        a = dict(dict(lens=i(2), table=i(2, 3), cu_rows=i(3)), **kw)
        with pytest.raises(lib.DsgxError):
            lib.kv_batch(4, 2, 16, a["lens"], a["table"], cu_rows=a["cu_rows"])


@pytest.mark.parametrize("D,fmt,Hkv,G", [(64, abi.FMT_BF16, 5, 3), (128, abi.FMT_BF16, 8, 8), (128, abi.FMT_BF16, 1, 1), (256, abi.FMT_BF16, 1, 64)])
def test_the_largest_batch_sizes_the_workspace(D, fmt, Hkv, G):
    c = _cache(Hkv=Hkv, D=D, head_stride=D, tok_stride=Hkv * D, page_stride=16 * Hkv * D)
    need = lambda **kw: lib.attn_ws_bytes(c, _batch(**kw), Hkv * G)  # noqa: E731
    whole = need(B=40, rows=200, max_rows=8, max_len=100)
    assert whole == need(B=40, rows=200, max_rows=200, max_len=90000, prefix_len=50000, prefix=0x400, table_ld=9000)
    for B in (1, 7, 40):
        for rows in (B, 2 * B, 200):
            assert 0 < need(B=B, rows=rows, max_rows=rows) <= whole
