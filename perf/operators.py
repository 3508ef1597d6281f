"""The operators between a decode layer's projections and after its head, as cases to be timed: the step's queries and keys
normed, rotated and appended to a paged cache (lib.kv_append), attention over that cache for a batch that may share a prefix
(lib.attn), and the verification of drafted tokens against the target's distribution (lib.spec_verify).

Shapes: 64 query heads of 256 over one head of keys and values are the chained layers' own projections (q_b gives 16384 values,
the x-projection the 512 beside its q latent); the others are generic: heads of 64, 128 and 256 in groups of 1 to 16, pages of 16
to 128 tokens, BF16 and e4m3 caches. draw() spreads over the sizes around them.

The plain form computes in f32 (probabilities and their sums in f64) and rounds once at the end; with `own` the public entry
points are called instead."""
import math

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-5
MOST_BYTES, MOST_FLOPS, MOST_POOL = 4e8, 2e11, 1.5e8  # of a drawn case; MOST_POOL: values of keys


def listed():
    return [
        # the smallest call: one token of one stream into its cache; the launch is the time
        dict(name="append 1 row", kind="append", B=1, rows="1", lens="777", prefix=0, Hq=64, Hkv=1, D=256, page=64, cache="bf16", rot=64, style="pairs", norm=True),
        # a step of many streams with a few drafted tokens each, e4m3 cache behind a shared prompt
        dict(name="append 40 drafting streams e4m3", kind="append", B=40, rows="1-6", lens="20-3000", prefix=1000, Hq=32, Hkv=8, D=128, page=16, cache="e4m3", rot=128, style="halves",
             norm=True),
        # a prompt's chunk of the largest size a call takes, beside two short ones
        dict(name="append three prompts' chunks", kind="append", B=3, rows="200-7600", lens="7600-8200", prefix=0, Hq=64, Hkv=8, D=128, page=64, cache="bf16", rot=64, style="halves",
             norm=True),
        # one stream, one token, a short context: latency
        dict(name="attn 1 row 301 tokens", kind="attn", B=1, rows="1", lens="301", prefix=0, Hq=32, Hkv=8, D=128, page=16, cache="bf16"),
        # speculative decoding far into a long document: five rows of the layers' own 64 x 256 heads over one cached head
        dict(name="attn 5 rows 50001 tokens", kind="attn", B=1, rows="5", lens="50001", prefix=0, Hq=64, Hkv=1, D=256, page=64, cache="bf16"),
        # a serving batch of ragged contexts, one to four rows each, e4m3 cache
        dict(name="attn 32 ragged streams e4m3", kind="attn", B=32, rows="1-4", lens="150-12000", prefix=0, Hq=32, Hkv=8, D=128, page=16, cache="e4m3"),
        # the same system prompt in front of every stream, short contexts of their own
        dict(name="attn prefix 8011 of 48 streams", kind="attn", B=48, rows="1", lens="37-600", prefix=8011, Hq=64, Hkv=8, D=128, page=64, cache="bf16"),
        # the largest: a long shared document, 100 streams with three rows each, where the matrix unit is the time
        dict(name="attn prefix 32768 of 100 streams", kind="attn", B=100, rows="3", lens="100-1500", prefix=32768, Hq=32, Hkv=4, D=128, page=128, cache="e4m3"),
        # one draft of one stream
        dict(name="verify 1 draft", kind="verify", B=1, drafts="1", V=32768, target="f32", sharp=False, temp=0.7),
        # a batch of streams with four drafts each, the drafter's probabilities kept
        dict(name="verify 16 x 4 drafts", kind="verify", B=16, drafts="4", V=131072, target="f32", sharp=False, temp=0.8),
        # many ragged streams, an odd vocabulary, bf16 logits; a drafter that picks its best token
        dict(name="verify 48 ragged bf16", kind="verify", B=48, drafts="0-7", V=100003, target="bf16", sharp=True, temp=1.0),
        # probabilities that the sampler's filters have left
        dict(name="verify 32 x 3 probabilities", kind="verify", B=32, drafts="3", V=65537, target="prob", sharp=False, temp=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return "%d-%d" % (a, b) if a < b else str(a)


def _heads(rng):
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 5, 8])
    G = rng.choice([1, 2, 3, 4, 6, 8, 8, 16])
    if rng.random() < 0.15:
        return 64, 1, 256
    return Hkv * G, Hkv, D


def draw(rng):
    while True:
        kind = rng.choice(["append", "attn", "attn", "verify"])
        if kind == "verify":
            c = dict(kind=kind, B=_log(rng, 1, 48), drafts=rng.choice(["0-7", "1", "2", "3", "1-5", "7"]), V=_log(rng, 2000, 160000), target=rng.choice(["f32", "f32", "bf16", "prob"]),
                     sharp=rng.random() < 0.4, temp=rng.choice([0.5, 0.8, 1.0, 1.3]))
        else:
            Hq, Hkv, D = _heads(rng)
            c = dict(kind=kind, B=_log(rng, 1, 100), rows=_span(rng, 1, 8), lens=_span(rng, 30, 60000), prefix=rng.choice([0, 0, _log(rng, 16, 32768)]), Hq=Hq, Hkv=Hkv, D=D,
                     page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["bf16", "e4m3"]))
            if kind == "append":
                c.update(rot=rng.choice([D, D, D // 2, 32]), style=rng.choice(["halves", "pairs"]), norm=rng.random() < 0.7, lens=_span(rng, 30, 4000))
                if rng.random() < 0.4:
                    n = _log(rng, 100, 8000)
                    c.update(B=1, rows=str(n), lens=str(n + rng.randint(0, 300)), prefix=0)
            if sum(_step(c)[1]) * c["Hkv"] * D > MOST_POOL:
                continue
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def _ints(text, n, salt):
    """n whole numbers spread over the span `text` ("7" or "2-90"): the ends first, the rest by a fixed rule"""
    if "-" not in text:
        return [int(text)] * n
    a, b = map(int, text.split("-"))
    f = [(0.61803398875 * (k + 1) + 0.37 * salt) % 1.0 for k in range(n)]
    return [[a, b][k] if k < 2 and n > 2 else int(round(a * (b / a) ** f[k])) if a > 0 else int(a + f[k] * (b - a + 1)) for k in range(n)]


def _step(c):
    """rows and own tokens of every sequence"""
    rows = _ints(c["rows"], c["B"], 1)
    lens = [max(n, L) for n, L in zip(rows, _ints(c["lens"], c["B"], 2))]
    return rows, lens


def _verify_rows(c):
    return [n + 1 for n in _ints(c["drafts"], c["B"], 3)]


def work(c):
    if c["kind"] == "verify":
        R, B, V = sum(_verify_rows(c)), c["B"], c["V"]
        # logits: every row's sum is needed; probabilities: only the row that is sampled from, and the drafter's beside it
        each = {"f32": 4, "bf16": 2, "prob": 4}[c["target"]]
        read = (B if c["target"] == "prob" else R) * V * each + (0 if c["sharp"] else B * V * 4)
        return {"bytes": read + 24 * R, "flops": 8 * (R + 2 * B) * V}
    rows, lens = _step(c)
    R, Hq, Hkv, D, e = sum(rows), c["Hq"], c["Hkv"], c["D"], 2 if c["cache"] == "bf16" else 1
    if c["kind"] == "append":
        return {"bytes": R * D * (Hq * 4 + Hkv * 2 * (2 + e)) + R * c["rot"] * 4, "flops": R * D * (8 * Hq + 10 * Hkv)}
    P = c["prefix"]
    seen = sum(n * P + n * L - n * (n - 1) // 2 for n, L in zip(rows, lens))
    return {"bytes": (P + sum(lens)) * Hkv * D * 2 * e + R * Hq * (4 * D + 4), "flops": 4 * D * Hq * seen}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "verify":
        return _prepare_verify(c, g)
    rows, lens = _step(c)
    B, R, P, page, Hq, Hkv, D = c["B"], sum(rows), c["prefix"], c["page"], c["Hq"], c["Hkv"], c["D"]
    per = -(-max(lens) // page)
    own_pages, pre_pages = [-(-L // page) for L in lens], -(-P // page)
    total = sum(own_pages) + pre_pages
    order = torch.randperm(total + 3, generator=g, device="cuda")[:total].to(torch.int32)
    table = torch.full((B, per), -1, dtype=torch.int32, device="cuda")
    fill = (torch.arange(per, device="cuda")[None, :] < _i32(own_pages)[:, None])
    table[fill] = order[pre_pages:]
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    s = dict(c=c, R=R, max_rows=max(rows), max_len=max(lens), cu=_i32(cu), lens=_i32(lens), table=table, prefix=order[:pre_pages].contiguous(), total=total + 3)
    shape = (s["total"], page, Hkv, D)
    if c["cache"] == "bf16":
        s["k"], s["v"], s["ks"], s["vs"] = _normal(g, *shape), _normal(g, *shape), None, None
    else:
        s["ks"] = torch.rand(Hkv, generator=g, device="cuda") * 0.02 + 0.01
        s["vs"] = torch.rand(Hkv, generator=g, device="cuda") * 0.02 + 0.01
        s["k"] = (_normal(g, *shape, dtype=torch.float32) / s["ks"][:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        s["v"] = (_normal(g, *shape, dtype=torch.float32) / s["vs"][:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if c["kind"] == "attn":
        # scores with a standard deviation of about 2.5: some keys matter, as after training
        s["q"] = _normal(g, R, Hq * D, scale=2.5)
        s["scale"] = D ** -0.5
        s["out"] = torch.empty(R, Hq * D, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.empty(R, Hq, dtype=torch.float32, device="cuda")
        return s
    # the projections' rows, queries, keys and values side by side
    s["qkv"] = _normal(g, R, (Hq + 2 * Hkv) * D, scale=1.7)
    s["wq"], s["wk"] = (_normal(g, D, scale=0.1) + 1.0 for _ in range(2)) if c["norm"] else (None, None)
    rot = c["rot"]
    angle = torch.arange(P + max(lens), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
    s["q_out"] = torch.empty(R, Hq * D, dtype=torch.bfloat16, device="cuda")
    return s


def _prepare_verify(c, g):
    n = _verify_rows(c)
    B, R, V = c["B"], sum(n), c["V"]
    cu = [0]
    for k in n:
        cu.append(cu[-1] + k)
    logits = _normal(g, R, V, scale=2.5, dtype=torch.float32)
    # the drafter is near the target, so that most drafts pass
    near = torch.softmax(logits / c["temp"] + 0.4 * torch.randn(R, V, generator=g, device="cuda"), -1)
    draft = near.argmax(-1) if c["sharp"] else torch.multinomial(near, 1, generator=g)[:, 0]
    s = dict(c=c, B=B, R=R, V=V, max_rows=max(n), cu=_i32(cu), draft=draft.to(torch.int32), q=None if c["sharp"] else near, u=torch.rand(R, generator=g, device="cuda"),
             us=torch.rand(B, generator=g, device="cuda"), temp=torch.full((B,), c["temp"], device="cuda"), tokens=torch.empty(R, dtype=torch.int32, device="cuda"),
             accepted=torch.empty(B, dtype=torch.int32, device="cuda"))
    if B > 4 and c["target"] != "prob":
        s["temp"][B // 2] = 0.0  # one stream of the batch decodes greedily
    if c["target"] == "prob":
        # what a filter of the least likely tokens leaves
        p = torch.softmax(logits / c["temp"], -1)
        p = torch.where(p < 0.02 * p.max(-1, keepdim=True).values, torch.zeros_like(p), p)
        s["target"] = p / p.sum(-1, keepdim=True)
    else:
        s["target"] = logits if c["target"] == "f32" else logits.to(torch.bfloat16)
    return s


def run(state):
    s, c = state, state["c"]
    if own:
        return {"append": _own_append, "attn": _own_attn, "verify": _own_verify}[c["kind"]](s, c)
    if c["kind"] == "append":
        return _plain_append(s, c, torch.float32)
    if c["kind"] == "attn":
        return _plain_attn(s, c)
    return _plain_verify(s)


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _cache_and_batch(s, c):
    """the handles that a program keeps with its cache and its batch"""
    from dsgx10_amd import lib
    if "cache" not in s:
        s["cache"] = lib.kv_cache(s["k"], s["v"], s["ks"], s["vs"])
        s["batch"] = lib.kv_batch(s["R"], s["max_rows"], s["max_len"], s["lens"], s["table"], cu_rows=s["cu"], prefix_len=c["prefix"], prefix=s["prefix"] if c["prefix"] else None)
    return s["cache"], s["batch"]


def _own_append(s, c):
    from dsgx10_amd import lib
    cache, batch = _cache_and_batch(s, c)
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    x, ld = s["qkv"], (Hq + 2 * Hkv) * D
    lib.kv_append(cache, batch, x[:, Hq * D:], ld, x[:, (Hq + Hkv) * D:], ld, q=x, ldq=ld, Hq=Hq, q_out=s["q_out"], ldqo=Hq * D, q_norm=s["wq"], k_norm=s["wk"], eps=EPS, rope=s["rope"],
                  rot=c["rot"], pairs=c["style"] == "pairs")
    return s["q_out"], _stored(s["k"]), _stored(s["v"])


def _own_attn(s, c):
    from dsgx10_amd import lib
    cache, batch = _cache_and_batch(s, c)
    if "ws" not in s:
        s["ws"] = torch.zeros(lib.attn_ws_bytes(cache, batch, c["Hq"]), dtype=torch.uint8, device="cuda")
    ld = c["Hq"] * c["D"]
    lib.attn(cache, batch, s["q"], ld, c["Hq"], s["scale"], s["out"], ld, s["ws"], lse=s["lse"])
    return s["out"], s["lse"]


def _own_verify(s, c):
    from dsgx10_amd import lib
    if "ws" not in s:
        s["ws"] = torch.zeros(lib.spec_verify_ws_bytes(s["B"], s["R"], s["V"]), dtype=torch.uint8, device="cuda")
    lib.spec_verify(s["target"], s["V"], s["draft"], s["u"], s["us"], s["tokens"], s["accepted"], s["ws"], s["max_rows"], cu_rows=s["cu"], q=s["q"], temp=s["temp"],
                    probs=c["target"] == "prob")
    return s["tokens"], s["accepted"]


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _stored(t):
    return t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t


def _places(s):
    """of every row: its sequence and its token among that sequence's own"""
    r = torch.arange(s["R"], device="cuda", dtype=torch.int32)
    b = torch.bucketize(r, s["cu"][1:], right=True)
    return b, (s["lens"][b] - (s["cu"][b + 1] - r)).long()


def _norm_rotate(x, w, cs, rot, pairs):
    """x [R][H][D] in the arithmetic's type; cs [R][rot]: cosines, then sines"""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    co, si = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * co - b * si, b * co + a * si
    y = torch.stack([ra, rb], -1).flatten(-2) if pairs else torch.cat([ra, rb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _append_rows(s, c, dtype):
    Hq, Hkv, D, R = c["Hq"], c["Hkv"], c["D"], s["R"]
    x = s["qkv"].to(dtype).view(R, Hq + 2 * Hkv, D)
    b, t = _places(s)
    cs = s["rope"].to(dtype)[c["prefix"] + t]
    pairs = c["style"] == "pairs"
    q = _norm_rotate(x[:, :Hq], s["wq"], cs, c["rot"], pairs)
    k = _norm_rotate(x[:, Hq:Hq + Hkv], s["wk"], cs, c["rot"], pairs)
    return q.reshape(R, Hq * D), k, x[:, Hq + Hkv:], s["table"][b, t // c["page"]].long(), t % c["page"]


def _plain_append(s, c, dtype):
    q, k, v, page, at = _append_rows(s, c, dtype)
    for pool, x, scale in ((s["k"], k, s["ks"]), (s["v"], v, s["vs"])):
        if c["cache"] == "bf16":
            pool[page, at] = x.to(torch.bfloat16)
        else:
            pool[page, at] = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.to(torch.bfloat16), _stored(s["k"]), _stored(s["v"])


def _tokens(pool, scale, pages, dtype):
    """pages [...][n] -> their tokens [...][n * page][Hkv][D] in the arithmetic's type"""
    t = _stored(pool[pages.clamp(min=0).long()]).to(dtype)
    t = t.flatten(-4, -3)
    return t if scale is None else t * scale.to(dtype)[:, None]


def _plain_attn(s, c):
    Hq, Hkv, D, B, P, R, N = c["Hq"], c["Hkv"], c["D"], c["B"], c["prefix"], s["R"], s["max_rows"]
    G = Hq // Hkv
    n = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(N, device="cuda")
    at = (s["cu"][:-1, None] + i).clamp(max=R - 1).long()                                     # [B][N]: the row, where there is one
    q = s["q"].view(R, Hkv, G, D).float()
    own_k, own_v = (_tokens(s[x], s[x + "s"], s["table"], torch.float32).permute(0, 2, 1, 3).contiguous() for x in "kv")   # [B][Hkv][L][D]
    qb = q[at].permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D)
    score = torch.matmul(qb, own_k.transpose(2, 3).contiguous()).mul_(s["scale"]).view(B, Hkv, N, G, -1)
    seen = (s["lens"] - n)[:, None] + i                                                       # the last token that row i sees
    t = torch.arange(score.shape[-1], device="cuda")
    score.masked_fill_(~(t <= seen[..., None])[:, None, :, None], -math.inf)
    top = score.amax(-1)
    if P:
        pre_k, pre_v = (_tokens(s[x], s[x + "s"], s["prefix"], torch.float32)[:P].permute(1, 0, 2).contiguous() for x in "kv")  # [Hkv][P][D]
        qp = q.permute(1, 0, 2, 3).reshape(Hkv, R * G, D)
        pre = torch.matmul(qp, pre_k.transpose(1, 2).contiguous()).mul_(s["scale"])
        pre_top = pre.amax(-1)
        pick = lambda x: x.view(Hkv, R, G, -1)[:, at].permute(1, 0, 2, 3, 4)                  # noqa: E731  [Hkv][R G][.] -> [B][Hkv][N][G][.]
        top = torch.maximum(top, pick(pre_top)[..., 0])
        r = torch.arange(R, device="cuda", dtype=torch.int32)
        b = torch.bucketize(r, s["cu"][1:], right=True)
        top_r = top[b, :, r - s["cu"][b]]                                                     # [R][Hkv][G]
        pre.sub_(top_r.permute(1, 0, 2).reshape(Hkv, R * G, 1)).exp_()
        pre_sum, pre_out = pre.sum(-1), torch.matmul(pre, pre_v)
    score.sub_(top[..., None]).exp_()
    total, out = score.sum(-1), torch.matmul(score.view(B, Hkv, N * G, -1), own_v).view(B, Hkv, N, G, D)
    if P:
        total, out = total + pick(pre_sum)[..., 0], out + pick(pre_out)
    out, lse = out / total[..., None], top + total.log()
    real = i < n[:, None]
    return out.permute(0, 2, 1, 3, 4)[real].reshape(R, Hq * D).to(torch.bfloat16), lse.permute(0, 2, 1, 3)[real].reshape(R, Hq)


def _plain_verify(s):
    c, R, B, V, cu = s["c"], s["R"], s["B"], s["V"], s["cu"].long()
    r = torch.arange(R, device="cuda")
    b = torch.bucketize(r, cu[1:], right=True)
    ids = torch.arange(V, device="cuda")
    if c["target"] == "prob":
        p = s["target"].double()
    else:
        # a sum over the vocabulary stands next to a border that a random number may fall on either side of: 64 bits
        x, temp = s["target"].double(), s["temp"].double()[b, None]
        best = x.amax(-1, keepdim=True)
        first = torch.where(x == best, ids, V).amin(-1, keepdim=True)
        e = ((x - best) / torch.where(temp > 0, temp, 1.0)).exp()
        p = torch.where(temp > 0, e / e.sum(-1, keepdim=True), (ids == first).double())
    d = s["draft"].long()
    pd = p.gather(1, d[:, None])[:, 0]
    qd = s["q"].gather(1, d[:, None])[:, 0].double() if s["q"] is not None else torch.ones_like(pd)
    last = r == cu[b + 1] - 1
    stop = ~(s["u"].double() * qd < pd) | last
    end = torch.where(stop, r, R).new_full((B,), R).scatter_reduce(0, b, torch.where(stop, r, R), "amin")     # the row that the last token comes from
    w = p[end]
    less = s["q"][end].double() if s["q"] is not None else (ids == d[end, None]).double()
    rest = (w - less).clamp(min=0)
    w = torch.where(last[end][:, None] | (rest.sum(-1, keepdim=True) <= 0), w, rest)
    total = w.cumsum(-1)
    token = (total <= s["us"].double()[:, None] * total[:, -1:]).sum(-1)
    tokens = torch.where(r < end[b], d, torch.where(r == end[b], token[b], -1))
    return tokens.to(torch.int32), (end - cu[:-1]).to(torch.int32)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "verify":
        return None  # whole numbers only
    rows, lens = _step(c)
    Hq, Hkv, D, page, P = c["Hq"], c["Hkv"], c["D"], c["page"], c["prefix"]
    if c["kind"] == "append":
        return _exact_append(s, c, rows, lens)
    if work(c)["flops"] > 2.5e11:
        return None
    G, res, lses = Hq // Hkv, [], []
    val = lambda x, h, pages: _stored(s[x][pages.long()])[:, :, h].double().reshape(-1, D) * (1.0 if s[x + "s"] is None else s[x + "s"][h].double())  # noqa: E731
    q = s["q"].double().view(s["R"], Hkv, G, D)
    for h in range(Hkv):
        pk, pv = (val(x, h, s["prefix"])[:P] for x in "kv")
        o, l, r = [], [], 0
        for b, (n, L) in enumerate(zip(rows, lens)):
            mine = s["table"][b, :-(-L // page)]
            k, v = (torch.cat([pre, val(x, h, mine)[:L]]) for x, pre in (("k", pk), ("v", pv)))
            a = torch.einsum("ngd,td->ngt", q[r:r + n, h], k) * s["scale"]
            hidden = torch.arange(P + L, device="cuda")[None, :] > P + L - n + torch.arange(n, device="cuda")[:, None]
            a = a.masked_fill(hidden[:, None, :], -math.inf)
            z = torch.logsumexp(a, -1)
            o.append(torch.einsum("ngt,td->ngd", (a - z[..., None]).exp(), v))
            l.append(z)
            r += n
        res.append(torch.cat(o))
        lses.append(torch.cat(l))
    return torch.stack(res, 1).reshape(s["R"], Hq * D), torch.stack(lses, 1).reshape(s["R"], Hq)


def _exact_append(s, c, rows, lens):
    Hq, Hkv, D, page, P, rot = c["Hq"], c["Hkv"], c["D"], c["page"], c["prefix"], c["rot"]
    b = torch.tensor([b for b, n in enumerate(rows) for _ in range(n)], device="cuda")
    t = torch.tensor([L - n + i for n, L in zip(rows, lens) for i in range(n)], device="cuda")
    x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
    out = x.clone()
    for lo, hi, w in ((0, Hq, s["wq"]), (Hq, Hq + Hkv, s["wk"])):
        y = x[:, lo:hi]
        if w is not None:
            y = y / (y.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        # each pair as a complex number, turned by its angle
        first = torch.arange(0, rot, 2, device="cuda") if c["style"] == "pairs" else torch.arange(rot // 2, device="cuda")
        second = first + 1 if c["style"] == "pairs" else first + rot // 2
        turn = torch.complex(s["rope"][P + t, :rot // 2].double(), s["rope"][P + t, rot // 2:].double())
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
        out[:, lo:hi] = y
        out[:, lo:hi, first], out[:, lo:hi, second] = z.real, z.imag
    pools = []
    for name, lo in (("k", Hq), ("v", Hq + Hkv)):
        pool, new = _stored(s[name]).double(), out[:, lo:lo + Hkv]
        scale = s[name + "s"]
        pool[s["table"][b, t // page].long(), t % page] = new if scale is None else (new / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        pools.append(pool)
    return out[:, :Hq].reshape(-1, Hq * D), pools[0], pools[1]
