"""One decode layer's dense projections and MoE step chained as the reference's runner chains them
(altar1-4xgx10-switchless/engine/model/model.cu:229-352), on the C ABI. Every launch, shape and dependency of the GEMVs and of
the MoE half is the runner's:

    x-projection   BF16 [XR][H], K split 4                 model.cu:236-247   <- RMSNorm(res + the layer before's yr)
    q_b            INT4 or FP8 [NQ][QL] on the first QL columns of the x-projection's output        model.cu:262-267
    attention      with an Attention handle: the keys and values behind the x-projection's first QL columns, and q_b's queries,
                   normed, rotated and appended to the layer's paged cache; then the queries over the cache
    o_proj         INT4 or FP8 [H][NQ], f32 partials                                                 model.cu:291-294
    add + norm     h = bf16(res + part), xn = RMSNorm(h) with the layer's ffn norm                   model.cu:299
    router         BF16 [E][H], f32 logits, K split 4                                                model.cu:311-313
    experts        routing, shared expert and yr += ys fused                                         model.cu:334-343
    add + norm     the next layer's attention norm                                                   model.cu:346-352

fused = True runs the add + norm in front of the router as the prologue of the router's GEMV (dsgx_add_norm_gemv): six
launches a layer (seven with the MFMA variant's ordered sum) instead of seven (eight); the bits are the same. fuse_xproj does
the same for the x-projection: right for the bits, but that GEMV has ten times the router's workgroups, each of which would
redo the rows' norm, and the layer gets slower (measured: +4 us at hidden 4096, +10 us at 6144), so it is off by default.

The runner's own attention, between its q_b and o_proj, reads a compressed latent through an indexer (the absorbed per-head
W_UK / W_UV products, sparse attention); that is not here. Without an Attention handle q_b's output goes to o_proj directly; with one, whole
heads attend: NQ = Hq D, and the x-projection has the 2 Hkv D values of a row's keys and values behind its first QL columns.
After the last layer, head() is the vocabulary's GEMV and the verification of the step's drafted tokens."""
from . import abi, lib


class Attention:
    """What the layers of a step share between q_b and o_proj. batch: lib.kv_batch of the step's rows; Hq query heads; ws: zeroed
    workspace of lib.attn_ws_bytes of the layers' caches (of one shape); scale: of the scores, 1 / sqrt(D) by default; rope f32
    [tokens][rot], rot, rot_off, pairs, eps and pos as in lib.kv_append. A layer's own cache and norms are in its W."""

    def __init__(self, batch, Hq, ws, scale=None, rope=None, rot=0, rot_off=0, pairs=False, eps=1e-5, pos=None):
        self.batch, self.Hq, self.ws, self.scale, self.eps = batch, Hq, ws, scale, eps
        self.rope = dict(rope=rope, rot=rot, rot_off=rot_off, pairs=pairs, pos=pos)


class LayerChain:
    def __init__(self, M, H, XR, QL, NQ, E, route_scale, alloc, V=0):
        """alloc(nbytes) -> a zeroed device buffer (the caller's allocator: torch in the tests and the bench); V: rows of the head's
        matrix, if head() is to be called"""
        self.M, self.H, self.XR, self.QL, self.NQ, self.E, self.route_scale = M, H, XR, QL, NQ, E, route_scale
        self.res = [alloc(M * H * 2), alloc(M * H * 2)]   # the residual stream, ping-pong (a fused add + norm reads one, writes the other)
        self.xn = alloc(M * H * 2)
        self.xg = alloc(M * XR * 2)
        self.q = alloc(M * NQ * 2)
        self.att = alloc(M * NQ * 2)   # attention's output
        self.V = V
        self.vocab = alloc(M * V * 4) if V else None
        self.part = alloc(M * H * 4)
        self.logits = alloc(M * E * 4)
        self.yr = alloc(M * H * 4)
        self.ys = alloc(M * H * 4)
        self.cur = 0

    def layer(self, W, fused=True, up=-1, stream=None, tap=None, fuse_xproj=False, attn=None):
        """W: dict(attn_norm, ffn_norm bf16 [H]; xproj bf16 [XR][H]; qb, oproj: dict(fmt, w, s, zp) [NQ][QL], [H][NQ]; router bf16
        [E][H]; moe: a dsgx_layer_w; ws: its decode workspace; with attn, an Attention: cache a lib.kv_cache, q_norm, k_norm
        bf16 [D] or absent). Reads res[cur] and yr, leaves the new residual in res[cur].
        tap(name): called after each stage (tests read the stage's buffers then)."""
        M, H, XR, QL, NQ, E = self.M, self.H, self.XR, self.QL, self.NQ, self.E
        a, b = self.res[self.cur], self.res[self.cur ^ 1]
        tap = tap or (lambda name: None)
        xp = [dict(fmt=abi.FMT_BF16, w=W["xproj"], n=XR, y=self.xg, ldy=XR)]
        if fused and fuse_xproj:
            lib.add_norm_gemv(self.yr, None, a, b, W["attn_norm"], 1e-5, None, M, H, xp, abi.OUT_BF16, splitk=2, stream=stream)
        else:
            lib.add_norm(self.yr, None, M, H, a, b, W["attn_norm"], 1e-5, self.xn, stream=stream)
            tap("norm1")
            # (K over 2 waves: 7.2 / 9.1 us for the two layers' shapes against 8.7 / 11.2 over 4 and 8.0 / 10.1 unsplit, measured)
            lib.gemv(self.xn, H, M, H, xp, abi.OUT_BF16, splitk=2, stream=stream)
        tap("xproj")
        lib.gemv(self.xg, XR, M, QL, [dict(W["qb"], n=NQ, y=self.q, ldy=NQ)], abi.OUT_BF16, stream=stream)
        tap("qb")
        y = self.q
        if attn is not None:
            y = self._attend(W, attn, stream, tap)
        lib.gemv(y, NQ, M, NQ, [dict(W["oproj"], n=H, y=self.part, ldy=H)], abi.OUT_F32, stream=stream)
        tap("oproj")
        rt = [dict(fmt=abi.FMT_BF16, w=W["router"], n=E, y=self.logits, ldy=E)]
        if fused:
            lib.add_norm_gemv(self.part, None, b, a, W["ffn_norm"], 1e-5, self.xn, M, H, rt, abi.OUT_F32, splitk=4, stream=stream)
        else:
            lib.add_norm(self.part, None, M, H, b, a, W["ffn_norm"], 1e-5, self.xn, stream=stream)
            tap("norm2")
            lib.gemv(self.xn, H, M, H, rt, abi.OUT_F32, splitk=4, stream=stream)
        tap("router")
        lib.moe_decode(W["moe"], self.xn, None, None, M, W["ws"], self.yr, self.ys, logits=self.logits, route_scale=self.route_scale,
                       ysum=True, up=up, stream=stream)
        tap("experts")
        # (the new residual is in res[cur] again: two add + norms a layer)

    def _attend(self, W, attn, stream, tap):
        """q_b's output and the x-projection's columns behind QL through the layer's cache -> o_proj's input"""
        M, XR, QL, NQ, cache = self.M, self.XR, self.QL, self.NQ, W["cache"]
        w = cache.Hkv * cache.D
        if attn.batch.rows != M or attn.Hq * cache.D != NQ or QL + 2 * w > XR:
            raise lib.DsgxError(abi.EINVAL, "chain: %d rows of %d heads of %d over %d heads, in a chain of %d rows, %d values of q and %d columns behind q_b's" %
                                (attn.batch.rows, attn.Hq, cache.D, cache.Hkv, M, NQ, XR - QL))
        k, v = self.xg[2 * QL:], self.xg[2 * (QL + w):]
        lib.kv_append(cache, attn.batch, k, XR, v, XR, q=self.q, ldq=NQ, Hq=attn.Hq, q_out=self.q, ldqo=NQ, q_norm=W.get("q_norm"), k_norm=W.get("k_norm"), eps=attn.eps,
                      stream=stream, **attn.rope)
        tap("append")
        lib.attn(cache, attn.batch, self.q, NQ, attn.Hq, cache.D ** -0.5 if attn.scale is None else attn.scale, self.att, NQ, attn.ws, stream=stream)
        tap("attn")
        return self.att

    def finish(self, norm_w, stream=None):
        """the add + norm after the last layer: the final residual into res[cur ^ 1], its norm into xn"""
        lib.add_norm(self.yr, None, self.M, self.H, self.res[self.cur], self.res[self.cur ^ 1], norm_w, 1e-5, self.xn, stream=stream)
        self.cur ^= 1

    def head(self, W, V, draft, u, us, tokens, accepted, ws, max_rows, cu_rows=None, q=None, temp=None, stream=None):
        """After finish(): the vocabulary's logits of the normed rows (W: dict(fmt, w, s, zp), [self.V][H]; the first V columns count)
        and the step's drafts judged by them, as lib.spec_verify does it. ws: zeroed, lib.spec_verify_ws_bytes(sequences, M, V)."""
        import torch
        if not 0 < V <= self.V or tokens.numel() != self.M:
            raise lib.DsgxError(abi.EINVAL, "chain: a vocabulary of %d in a chain made for %d, %d tokens of %d rows" % (V, self.V, tokens.numel(), self.M))
        lib.gemv(self.xn, self.H, self.M, self.H, [dict(W, n=self.V, y=self.vocab, ldy=self.V)], abi.OUT_F32, stream=stream)
        lib.spec_verify(self.vocab.view(torch.float32), V, draft, u, us, tokens, accepted, ws, max_rows, cu_rows=cu_rows, q=q, temp=temp, ldt=self.V, stream=stream)
