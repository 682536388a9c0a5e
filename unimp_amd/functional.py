"""Autograd building blocks of the Flamingo step, each one a fused forward/backward over the HIP kernels.

Granularity is the residual sub-block (x -> x + f(LN(x))) so that the residual gradient add is fused into
the LayerNorm backward kernel and no eager PyTorch arithmetic sits on the hot path.  Weight gradients are
only computed for parameters whose ``requires_grad`` is set at call time (the LM tower is frozen in UniMP,
so its backward is dX-only; SURVEY.md §0.6 / §7 "honour flags at step time").

Arithmetic restated (reference file:line):
  mlp_block          CLIPMLP clip.py:144-156 / GPTNeoXMLP / open_flamingo FeedForward (+ tanh gate)
  neox_attn_block    GPTNeoXAttention + residual (transformers gpt_neox modelling :180-283)
  gated_xattn        open_flamingo MaskedCrossAttention + attn_gate
  perceiver_attn     open_flamingo PerceiverAttention (A.2)
  focal_ce           UniMP/mmrec.py:190-213
"""
import math
import os as _os
import weakref
import torch
from torch.autograd import Function

from . import ops

bf16 = torch.bfloat16


def _need(ctx, i):
    return ctx.needs_input_grad[i]


# Weight-gradient sink (train.Trainer installs one around backward): an object with ``view_of(weight)`` -> the weight's
# [out, in] view of the flat bf16 gradient buffer, or None, and ``done(weight)``.  With a sink the dW GEMM adds its fp32
# accumulators straight into that view (epilogue ``accumulate``) and autograd gets no gradient for the weight -- no temporary,
# no ``.grad +=`` pass, one bf16 rounding instead of two; ``done`` then plays the post-accumulate hook for the data-parallel
# bucketer (the weight's gradient is complete: every weight routed here is used once per step).  Without a sink (tests that
# call ``loss.backward()`` themselves) the gradient is returned as usual.
WGRAD_SINK = None
ROPE_FUSE = _os.environ.get("UNIMP_ROPE_FUSE", "1") != "0"      # backward: dq / dk rotated back inside the attention kernels' epilogues


def _dw(ctx, idx, w, a, b, gate=None):
    """weight gradient a^T b ([out, tokens] x [tokens, in], both token-major) of forward input ``idx``."""
    if not _need(ctx, idx):
        return None
    sink = WGRAD_SINK
    if sink is not None:
        out = sink.view_of(w)
        if out is not None:
            ops.gemm(a, b, a_ks=True, b_ks=True, gate=gate, out=out, accumulate=True)
            sink.done(w)
            return None
    return ops.gemm(a, b, a_ks=True, b_ks=True, gate=gate)


def _ln_bwd(dy, x2, w, b, mean, rstd, need_w, need_b, has_beta=True, **kw):
    """ops.layernorm_bwd with the weight gradients routed through the sink (added straight into gamma's / beta's slots of the
    flat gradient buffer) when there is one; returns (dx, dgamma, dbeta) with None for what went to the sink."""
    want = need_w or (has_beta and need_b)
    sink = WGRAD_SINK
    if (want and sink is not None and need_w and (need_b or not has_beta) and sink.has(w) and (not has_beta or (b is not None and sink.has(b)))):
        vg = sink.view_of(w)
        vb = sink.view_of(b) if has_beta else None
        dx, _, _ = ops.layernorm_bwd(dy, x2, w, mean, rstd, want_wgrad=True, has_beta=has_beta, dg_out=vg, db_out=vb, **kw)
        sink.done(w)
        if has_beta:
            sink.done(b)
        return dx, None, None
    return ops.layernorm_bwd(dy, x2, w, mean, rstd, want_wgrad=want, has_beta=has_beta, **kw)


def _gate_grad(dy, raw, gate):
    """d/d gate of tanh(gate) * raw contracted with dy."""
    d = ops.dot(dy, raw)
    t = torch.tanh(gate.float())
    return (d * (1 - t * t)).to(gate.dtype).view_as(gate)


def _no_bias_grad(ctx, idx, name):
    if idx is not None and _need(ctx, idx):
        raise NotImplementedError(f"gradient w.r.t. dense-layer bias '{name}' is not implemented in unimp_amd "
                                  "(no trainable Linear bias exists in the UniMP configuration)")


# ----------------------------------------------------------------------------------------------- packed token order (opt-in)
# collate_rec.py:38-74 right-pads every sequence of a batch to the longest; the reference then runs every row-wise operation of the
# language tower (LayerNorm, the QKV / out / MLP / gated feed-forward projections) over the <PAD> rows too.  In packed mode
# (Trainer(packed=True), bench.py --packed, UNIMP_PACKED=1) the tower's residual stream holds the VALID tokens only, as [1, M, H] with
# M = the valid count rounded up to PACK_ROUND rows (default: 1/16 of B * L), sequence after sequence.  The attention kernels take that layout directly
# (include/unimp_hip.h q_row_off / k_row_off: sequence b = rows off[b] .. off[b] + len[b] - 1), the QKV projection's rotary epilogue
# reads each row's position from a table: nothing is gathered or scattered between the embedding and the final hidden state.
# Every valid row goes through the same arithmetic as in the padded run; nothing reads the rows that are skipped.
PACKED = _os.environ.get("UNIMP_PACKED", "0") == "1"
PACK_ROUND = None           # M granularity in rows; None: 1/16 of B * L in multiples of 256 (2 048 at b = 64, L = 512) -- keeps the number of
                            # distinct GEMM shapes (autotune keys) per batch size at two or three
PACK = None                 # the Pack of the forward in progress (set by the tower's forward)


class Pack:
    """idx int32 [M]: flat position b * L + j of packed row r (rows beyond the valid count point at one <PAD> position: they are
    computed by the row-wise kernels, never read back, and hold exact zeros in every gradient); inv int32 [B * L]: packed row of a
    position, -1 at <PAD>; rows: the sequences as row ranges (ops.PackedRows); pos int32 [M]: position of a row inside its sequence.
    Needs RIGHT-padded sequences (pipeline/train/data.py:274 ``tokenizer.padding_side = "right"``): a sequence is one row range."""

    def __init__(self, attention_mask):
        B, L = attention_mask.shape
        m = attention_mask != 0
        flat = m.reshape(-1)
        pos = flat.nonzero().view(-1)                      # host sync: the valid count
        nv = pos.numel()
        rnd = PACK_ROUND or max(256, B * L // 16 // 256 * 256)
        M = min(B * L, (nv + rnd - 1) // rnd * rnd)
        self.B, self.L, self.nv, self.M = B, L, nv, M
        self.useful = nv > 0 and M < B * L
        if not self.useful:
            return
        if bool((m[:, 1:] & ~m[:, :-1]).any()):
            raise ValueError("packed token order needs right-padded sequences (every attention_mask row a prefix of ones)")
        dev = attention_mask.device
        dummy = (~flat).nonzero()[0]                        # exists: M < B * L
        idx = torch.cat([pos, dummy.expand(M - nv)]) if M > nv else pos
        self.idx_long = idx
        self.idx = idx.to(torch.int32).contiguous()
        inv = torch.full((B * L,), -1, dtype=torch.int32, device=dev)
        inv[pos] = torch.arange(nv, dtype=torch.int32, device=dev)
        self.inv = inv
        lens = m.sum(1).to(torch.int32)
        off = (torch.cumsum(lens, 0) - lens).to(torch.int32)
        self.rows = ops.PackedRows(B, L, off, lens, nv)
        self.pos = (idx % L).to(torch.int32).contiguous()
        self._seg = None

    def seg(self, seg):
        """a per-token int32 [B, L] map (media_time of the gated cross-attention) in the packed row order; one gather per forward"""
        if self._seg is None or self._seg[0] is not seg:
            self._seg = (seg, seg.reshape(-1)[self.idx_long].contiguous())
        return self._seg[1]


class PackRowsFn(Function):
    """padded [B * L, D] -> packed [M, D]"""

    @staticmethod
    def forward(ctx, x, pack):
        ctx.pack = pack
        return ops.gather_rows(x, pack.idx)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        return ops.gather_rows(dy.contiguous(), ctx.pack.inv), None


class UnpackRowsFn(Function):
    """packed [M, D] -> padded [B * L, D], zeros at <PAD>"""

    @staticmethod
    def forward(ctx, x, pack):
        ctx.pack = pack
        return ops.gather_rows(x, pack.inv)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        return ops.gather_rows(dy.contiguous(), ctx.pack.idx), None


# ----------------------------------------------------------------------------------------------- LayerNorm
class LayerNormFn(Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, rms):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        y, mean, rstd = ops.layernorm_fwd(x2, w, b, eps, rms=rms)
        ctx.save_for_backward(x2, w, mean, rstd)
        ctx.rms, ctx.has_b, ctx.shp, ctx.b_ref = rms, b is not None, shp, b
        return y.view(shp)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, w, mean, rstd = ctx.saved_tensors
        dy2 = dy.reshape(-1, ctx.shp[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dx, dg, db = _ln_bwd(dy2, x2, w, ctx.b_ref, mean, rstd, _need(ctx, 1), ctx.has_b and _need(ctx, 2), has_beta=ctx.has_b, rms=ctx.rms)
        return dx.view(ctx.shp), dg, db, None, None


def layer_norm(x, w, b, eps=1e-5, rms=False):
    return LayerNormFn.apply(x, w, b, eps, rms)


# ----------------------------------------------------------------------------------------------- Linear (lm head etc.)
class LinearFn(Function):
    """y = x W^T (+ b); optional padded leading dimension for odd N (the vocabulary)."""

    @staticmethod
    def forward(ctx, x, w, b, ldc):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        y = ops.gemm(x2, w, bias=b, ldc=ldc)
        ctx.save_for_backward(x2, w)
        ctx.shp, ctx.b_idx = shp, (2 if b is not None else None)
        return y.view(*shp[:-1], w.shape[0]) if ldc in (None, w.shape[0]) else \
            y.as_strided((*shp[:-1], w.shape[0]), _lead_strides(shp[:-1], ldc) + (1,), y.storage_offset())

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, w = ctx.saved_tensors
        _no_bias_grad(ctx, ctx.b_idx, "bias")
        N = w.shape[0]
        dy2 = _as_matrix(dy, N)
        dx = ops.gemm(dy2, w, b_ks=True).view(ctx.shp) if _need(ctx, 0) else None
        dw = _dw(ctx, 1, w, dy2, x2)
        return dx, dw, None, None


def _lead_strides(lead, ld):
    st, acc = [], ld
    for n in reversed(lead):
        st.append(acc)
        acc *= n
    return tuple(reversed(st))


def _as_matrix(t, N):
    """[..., N] gradient -> 2-D bf16 matrix with unit inner stride and ld % 8 == 0 (repack only if needed)."""
    if t.dtype != bf16:
        t = t.to(bf16)
    lead = t.shape[:-1]
    rows = 1
    for n in lead:
        rows *= n
    ld = t.stride(-2) if t.dim() >= 2 else N
    uniform = t.stride(-1) == 1 and ld % 8 == 0 and t.data_ptr() % 16 == 0 and \
        all(t.stride(i) == t.stride(i + 1) * t.shape[i + 1] for i in range(t.dim() - 2))
    if uniform:
        return t.as_strided((rows, N), (ld, 1), t.storage_offset())
    ldp = (N + 7) // 8 * 8
    buf = torch.zeros((rows, ldp), dtype=bf16, device=t.device)
    buf[:, :N].copy_(t.reshape(rows, N))
    return buf[:, :N]


def linear(x, w, b=None, ldc=None):
    return LinearFn.apply(x, w, b, ldc)


def _frozen_t(w):
    """k-strided copy W^T [in, out] of a FROZEN weight, cached on the parameter and rebuilt when the weight is written to
    (load_state_dict copies in place and bumps `_version`).  The forward MLP GEMMs run 5-8 % faster with the weight operand
    in that form (tools/bench_gemm_ab.py, the W^T rows); trainable weights keep the reference layout -- a copy would have to follow every
    optimizer step."""
    c = getattr(w, "_unimp_wt", None)
    if c is None or c[0] != w._version or c[1].data_ptr() == 0:
        c = (w._version, w.detach().t().contiguous())
        w._unimp_wt = c
    return c[1]


# Rotary epilogue of the fused QKV projection (frozen towers, training path): the projection's rows are permuted ONCE so that
# the rotation pairs (i, i + rot/2) of every q and k head vector become adjacent -- index 8g + j pairs with 8g + 4 + j -- and the
# QKV GEMM rotates them in its epilogue (ops.gemm(rope=...), csrc/gemm_tile.h): the read + write pass of rope_ over the fused
# [B L, 3H] buffer is gone, and the backward kernels rotate dq / dk back in the same layout without tables.  Attention only ever
# takes q . k, which a common permutation of their dims leaves unchanged; v keeps its order.  UNIMP_ROPE_EPILOGUE=0 disables it.
ROPE_EPILOGUE = _os.environ.get("UNIMP_ROPE_EPILOGUE", "1") != "0"


def _rope_perm_index(nh, hd, rot, interleaved, device):
    """row index map new -> old of the fused projection [3H, H] for the adjacent-pair layout"""
    half = rot // 2
    p = torch.arange(hd)
    g, j = p // 8, p % 8
    d = torch.where(j < 4, 4 * g + j, half + 4 * g + (j - 4))
    d = torch.where(p < rot, d, p)                               # dims beyond the rotary part keep their place
    ident = torch.arange(hd)
    if interleaved:            # rows [nh][q | k | v][hd]
        per_head = torch.cat([d, hd + d, 2 * hd + ident])
        idx = (torch.arange(nh)[:, None] * 3 * hd + per_head[None]).reshape(-1)
    else:                      # rows [q | k | v][nh][hd]
        H = nh * hd
        qk = (torch.arange(nh)[:, None] * hd + d[None]).reshape(-1)
        idx = torch.cat([qk, H + qk, 2 * H + torch.arange(H)])
    return idx.to(device)


def _frozen_rope_perm(t, nh, hd, rot, interleaved):
    """rows of a FROZEN fused QKV projection weight [3H, H] (or bias [3H]) in the adjacent-pair order; cached on the tensor like _frozen_t"""
    key = (t._version, nh, hd, rot, interleaved)
    c = getattr(t, "_unimp_rope_perm", None)
    if c is None or c[0] != key:
        c = (key, t.detach().index_select(0, _rope_perm_index(nh, hd, rot, interleaved, t.device)).contiguous())
        t._unimp_rope_perm = c
    return c[1]


def _frozen_pk(w, b_ks=False):
    """fragment-ordered image of a FROZEN weight for the packed-B ping-pong GEMM (ops.pack_b), one per orientation: b_ks=False
    serves y = x W^T, b_ks=True serves dx = dy W.  Cached on the parameter like _frozen_t; costs one extra copy of the frozen
    weights per orientation in HBM (4b-instruct: 2 x 5 GB)."""
    if not FROZEN_PK or w.requires_grad:
        return None
    key = "_unimp_pk_t" if b_ks else "_unimp_pk"
    c = getattr(w, key, None)
    if c is None or c[0] != w._version:
        c = (w._version, ops.pack_b(w.detach(), b_ks))
        setattr(w, key, c)
    return c[1]


# opt-in: frozen weights also kept as packed-B images (the B operand bypasses the LDS).  Measured (tools/bench_packed.py, b = 64): +3 %
# over the best unpacked variant on the MLP up-projection, equal or slower on the other seven tower shapes -- the fragment loads
# wait on L2 latency every half-step where the LDS-DMA ring does not -- so it is NOT the default (it also costs a second copy
# of the frozen weights per orientation)
FROZEN_PK = _os.environ.get("UNIMP_FROZEN_PK", "0") == "1"
# Forward GEMMs of FROZEN layers read a cached transposed copy W^T [in, out] of the weight (default since round 4; UNIMP_FROZEN_WT=0: off,
# =1: MLP weights only).  A k-strided B operand is staged in whole 512-byte rows per LDS-DMA instruction where the k-contiguous [out, in]
# form is fetched as 64-byte pieces of 16 different rows: +1.5 ... +4.8 % on every forward shape of the towers (tools/bench_gemm_ab.py,
# profiles/r04_gemm_ab_forms.txt), and EVERY kernel variant sums the two forms in the same order -- the same bits as the [out, in] form on
# all nine variants (tools/check_ks_bits.py; round 3 kept this opt-in on the belief that the 128 x 128 kernel differed).  Costs one
# extra copy of the frozen weights in HBM (4b-instruct: 5.6 GB of 288).
_FW = int(_os.environ.get("UNIMP_FROZEN_WT", "2"))
FROZEN_WT = _FW >= 1      # frozen MLP weights (LM, ViT)
FROZEN_WT_ATTN = _FW >= 2    # frozen qkv / attention-out projections (LM, ViT), incl. the row-permuted copy of the rotary epilogue


# ----------------------------------------------------------------------------------------------- MX-fp8 frozen towers (F4)
FP8_FROZEN = _os.environ.get("UNIMP_FP8", "0") == "1"   # opt-in (bench.py --fp8): frozen Linear layers of the towers run on the MX-fp8 GEMM


# A weight takes the MX path only if BOTH its dimensions reach FP8_MIN_DIM (each is the contraction depth of the forward or of dX).  At
# K = 1024 a 256 x 256 MX tile is 8 K-steps of 128 bytes -- prologue and epilogue outweigh the loop -- and the bf16 ping-pong kernel is the
# faster one: the ViT-L/14's four projections ran at 0.53-1.11 PF on the MX kernel against 0.86-1.22 PF in bf16, before the cost of
# quantising their activations (profiles/r04_mx_step_shapes.txt).  So "fp8 frozen towers" means the language tower (4096 x 4096 ... 16384);
# UNIMP_FP8_MIN_DIM=128 restores MX everywhere (the tiny-tower tests do).
FP8_MIN_DIM = int(_os.environ.get("UNIMP_FP8_MIN_DIM", "2048"))
MX_FUSED_OUT = _os.environ.get("UNIMP_MX_FUSED_OUT", "1") != "0"     # MLP-internal activations leave their GEMM as MX operands (A/B knob; same bits)


def _mx_ok(w, M):
    """the MX path serves a FROZEN weight whose two dimensions are multiples of 128 (contraction of the forward and of dX) and at
    least FP8_MIN_DIM, for row counts the decode kernel does not take"""
    return (FP8_FROZEN and not w.requires_grad and M > 64 and w.shape[0] % 128 == 0 and w.shape[1] % 128 == 0
            and min(w.shape[0], w.shape[1]) >= FP8_MIN_DIM)


def _frozen_mx(w, transposed=False):
    """e4m3 + E8M0 copy of a frozen weight, quantised ONCE along the contraction dimension of the product it serves:
    W [out, in] along `in` for y = x W^T; W^T [in, out] along `out` for dx = dy W.  Cached on the parameter, rebuilt when the
    weight is written to (like _frozen_t)."""
    key = "_unimp_mx_t" if transposed else "_unimp_mx"
    c = getattr(w, key, None)
    if c is None or c[0] != w._version:
        src = w.detach().t().contiguous() if transposed else w.detach()
        c = (w._version, ops.mx_quantize(src))
        setattr(w, key, c)
    return c[1]


# ----------------------------------------------------------------------------------------------- MLP sub-block
DERIV_U8 = _os.environ.get("UNIMP_DERIV_U8", "1") != "0"      # the stored act'(z) of the MLP blocks in 8 bits; 0: bf16


class MLPBlockFn(Function):
    """out = res + tanh(gate) * (act(LN(x) W1^T + b1) W2^T + b2);  res defaults to x, gate to 1."""

    @staticmethod
    def forward(ctx, x, res, ln_w, ln_b, w1, b1, w2, b2, gate, act, eps):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        r2 = x2 if res is None else res.reshape(-1, shp[-1])
        M, F = x2.shape[0], w1.shape[0]
        w1g, w2g = w1.requires_grad, w2.requires_grad
        bwd = any(ctx.needs_input_grad)            # frozen tower on constant inputs (the ViT): no act'(z) output, nothing saved
        mx = gate is None and _mx_ok(w1, M) and _mx_ok(w2, M)
        ln_mx = mx and MX_FUSED_OUT and shp[-1] % 32 == 0 and shp[-1] <= 4096
        h, mean, rstd = ops.layernorm_fwd_mx(x2, ln_w, ln_b, eps) if ln_mx else ops.layernorm_fwd(x2, ln_w, ln_b, eps)
        # act'(z) for the backward: uint8 (ops / common.h DERIV_U8: step 1 / 202, 0 and 1 exact) unless the decode-row kernel (M <= 64) writes it
        pre = torch.empty((M, F), dtype=torch.uint8 if (DERIV_U8 and F % 8 == 0 and M > 64) else bf16, device=x.device) if bwd else None
        t1, t2 = FROZEN_WT and not w1g and M > 64, FROZEN_WT and not w2g and M > 64      # M <= 64: the weight-streaming decode kernel
        if mx:      # frozen tower on the MX-fp8 path: activations quantised on the fly (e4m3 + E8M0 per 32), fp32 accumulate
            # the up-projection's output only feeds the down-projection (both frozen): it leaves its GEMM already quantised
            # (MX_FUSED_OUT: the bytes mx_quantize would make of the bf16 tensor, without that tensor and without the quantiser pass)
            fused = MX_FUSED_OUT and F % 32 == 0
            a = ops.gemm_mx(h if ln_mx else ops.mx_quantize(h), _frozen_mx(w1), bias=b1, act=act, pre=pre, out_mx=fused)
            raw = None
            out = ops.gemm_mx(a if fused else ops.mx_quantize(a), _frozen_mx(w2), bias=b2, res=r2)
            a = None
        else:
            a = ops.gemm(h, _frozen_t(w1) if t1 else w1, b_ks=t1, bias=b1, act=act, pre=pre, pre_deriv=bwd,   # pre <- act'(z): backward needs no transcendental
                         b_pk=None if t1 or M <= 64 else _frozen_pk(w1))
            raw = torch.empty_like(x2) if gate is not None and bwd else None
            out = ops.gemm(a, _frozen_t(w2) if t2 else w2, b_ks=t2, bias=b2, gate=gate, res=r2, pre=raw,
                           b_pk=None if t2 or M <= 64 else _frozen_pk(w2))
        if bwd:
            ctx.save_for_backward(x2, ln_w, mean, rstd, w1, w2, gate, pre, h if w1g else None, a if w2g else None, raw)
        ctx.act, ctx.shp, ctx.res_is_x, ctx.has_lnb, ctx.mx, ctx.ln_b_ref = act, shp, res is None, ln_b is not None, mx, ln_b
        return out.view(shp)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, ln_w, mean, rstd, w1, w2, gate, pre, h, a, raw = ctx.saved_tensors
        _no_bias_grad(ctx, 5, "b1")
        _no_bias_grad(ctx, 7, "b2")
        dy2 = dy.reshape(-1, ctx.shp[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dgate = _gate_grad(dy2, raw, gate) if gate is not None and _need(ctx, 8) else None
        if ctx.mx:      # dX through the frozen MLP on the MX path: the same e4m3 weights, quantised along the other dimension
            fused = MX_FUSED_OUT and w2.shape[1] % 32 == 0
            dpre = ops.gemm_mx(ops.mx_quantize(dy2), _frozen_mx(w2, True), aux=pre, out_mx=fused)
            dw1 = dw2 = None
            dh = ops.gemm_mx(dpre if fused else ops.mx_quantize(dpre), _frozen_mx(w1, True))
        else:
            dpre = ops.gemm(dy2, w2, b_ks=True, gate=gate, aux=pre, dact="deriv", b_pk=_frozen_pk(w2, True))   # [M,F]  (dy tanh(g) W2) * act'(z)
            dw2 = _dw(ctx, 6, w2, dy2, a, gate=gate)
            dw1 = _dw(ctx, 4, w1, dpre, h)
            dh = ops.gemm(dpre, w1, b_ks=True, b_pk=_frozen_pk(w1, True))
        del dpre
        dx, dg, db = _ln_bwd(dh, x2, ln_w, ctx.ln_b_ref, mean, rstd, _need(ctx, 2), ctx.has_lnb and _need(ctx, 3), has_beta=ctx.has_lnb,
                             dres=dy2 if ctx.res_is_x else None)
        dres = None if ctx.res_is_x else dy
        return dx.view(ctx.shp), dres, dg, db, dw1, None, dw2, None, dgate, None, None


def mlp_block(x, ln_w, ln_b, w1, b1, w2, b2, act, gate=None, res=None, eps=1e-5):
    if not torch.is_grad_enabled() and x.numel() // x.shape[-1] <= 16 and _ln_fusable(x.numel() // x.shape[-1], x.shape[-1], False):
        # a cached decode step (M <= 16 rows, autograd off -- decided HERE: inside a Function.forward grad mode is always off and
        # needs_input_grad follows requires_grad, so the trainable gated blocks would look like training): two launches, the LayerNorm
        # inside the up-projection's weight-streaming GEMM, no act'(z) output, nothing saved
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        r2 = x2 if res is None else res.reshape(-1, shp[-1])
        a = ops.gemm(x2, w1, bias=b1, act=act, ln=(ln_w, ln_b, eps))
        return ops.gemm(a, w2, bias=b2, gate=gate, res=r2).view(shp)
    return MLPBlockFn.apply(x, res, ln_w, ln_b, w1, b1, w2, b2, gate, act, eps)


class SwiGLUBlockFn(Function):
    """out = x + down( silu(gate(RMSNorm(x))) * up(RMSNorm(x)) )   (UniMP/xformers_model/llama.py:185-199,311-380).
    w_gu is the row-concatenation [gate_proj; up_proj] so one GEMM yields [gate | up]."""

    @staticmethod
    def forward(ctx, x, ln_w, w_gu, w_down, eps):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1])
        F = w_gu.shape[0] // 2
        h, _, rstd = ops.layernorm_fwd(x2, ln_w, None, eps, rms=True)
        gu = ops.gemm(h, w_gu)
        a = ops.swiglu_fwd(gu, F)
        out = ops.gemm(a, w_down, res=x2)
        ctx.save_for_backward(x2, ln_w, rstd, w_gu, w_down, gu, h if w_gu.requires_grad else None, a if w_down.requires_grad else None)
        ctx.shp, ctx.F = shp, F
        return out.view(shp)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, ln_w, rstd, w_gu, w_down, gu, h, a = ctx.saved_tensors
        dy2 = dy.reshape(-1, ctx.shp[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        da = ops.gemm(dy2, w_down, b_ks=True)
        dwd = ops.gemm(dy2, a, a_ks=True, b_ks=True) if _need(ctx, 3) else None
        dgu = ops.swiglu_bwd(gu, da, ctx.F)
        dwgu = ops.gemm(dgu, h, a_ks=True, b_ks=True) if _need(ctx, 2) else None
        dh = ops.gemm(dgu, w_gu, b_ks=True)
        dx, dg, _ = ops.layernorm_bwd(dh, x2, ln_w, None, rstd, dres=dy2, want_wgrad=_need(ctx, 1), has_beta=False, rms=True)
        return dx.view(ctx.shp), dg, dwgu, dwd, None


def swiglu_block(x, ln_w, w_gu, w_down, eps=1e-6):
    return SwiGLUBlockFn.apply(x, ln_w, w_gu, w_down, eps)


# ----------------------------------------------------------------------------------------------- GPT-NeoX / OPT / Llama self-attention sub-block
class SelfAttnBlockFn(Function):
    """out = res + dense(causal_attn(rope(qkv(LN(x)))));  qkv layout [B, L, nh, 3*hd] (GPT-NeoX per-head interleave)
    or [B, L, 3, nh, hd] (blocked q|k|v: OPT / Llama / ViT)."""

    @staticmethod
    def forward(ctx, x, res, ln_w, ln_b, wqkv, bqkv, wd, bd, rope, kv_len, nh, interleaved, causal, eps, rms, q_scale, alibi=None,
                qk_ln=None):
        """qk_ln = (q_ln weight, k_ln weight, eps): LayerNorm over the full d_model vectors of q and of k before the heads are split
        (the QK-LayerNorm MPT of mmrec.py:475-494's "3b" towers, mosaic_gpt ``attn_qk_ln``); frozen gains only, blocked q|k|v layout."""
        pack = PACK
        if pack is not None:
            return SelfAttnBlockFn._forward_packed(ctx, pack, x, res, ln_w, ln_b, wqkv, bqkv, wd, bd, rope, kv_len, nh, interleaved, causal, eps,
                                                   rms, q_scale, alibi, qk_ln)
        ctx.pack = None
        B, L, H = x.shape
        hd = H // nh
        x2 = x.reshape(B * L, H)
        r2 = x2 if res is None else res.reshape(B * L, H)
        mx = _mx_ok(wqkv, B * L) and _mx_ok(wd, B * L)
        ln_mx = mx and MX_FUSED_OUT and H % 32 == 0 and H <= 4096            # the normalised rows only feed the frozen MX projection: they leave LayerNorm quantised
        h, mean, rstd = ops.layernorm_fwd_mx(x2, ln_w, ln_b, eps, rms=rms) if ln_mx else ops.layernorm_fwd(x2, ln_w, ln_b, eps, rms=rms)
        tq = FROZEN_WT_ATTN and not wqkv.requires_grad and B * L >= 1024
        td = FROZEN_WT_ATTN and not wd.requires_grad and B * L >= 1024
        # rotary epilogue: frozen projection, bf16 path, a kernel variant that serves it, positions 0 .. L-1 per sequence
        fused = None
        if (ROPE_EPILOGUE and rope is not None and len(rope) > 3 and not mx and not wqkv.requires_grad and not FROZEN_PK
                and (bqkv is None or not bqkv.requires_grad) and rope[2] % 8 == 0 and hd % 8 == 0 and B * L < (1 << 24)
                and ops.attn_generation() >= 2 and ops.gemm_rope_variant(B * L, 3 * H, H, tq, x.device) is not None):
            rot = rope[2]
            fused = dict(rot=rot, hd=hd, period=3 * hd if interleaved else 3 * H, span=2 * hd if interleaved else 2 * H, L=L,
                         log2_base=math.log2(rope[3]))
        if fused is not None:
            wp = _frozen_rope_perm(wqkv, nh, hd, fused["rot"], interleaved)
            bp = _frozen_rope_perm(bqkv, nh, hd, fused["rot"], interleaved) if bqkv is not None else None
            qkv = ops.gemm(h, _frozen_t(wp) if tq else wp, b_ks=tq, bias=bp, rope=fused)
        else:
            qkv = ops.gemm_mx(h if ln_mx else ops.mx_quantize(h), _frozen_mx(wqkv), bias=bqkv) if mx else \
                ops.gemm(h, _frozen_t(wqkv) if tq else wqkv, b_ks=tq, bias=bqkv, b_pk=None if tq else _frozen_pk(wqkv))
        q, k, v, hs, offs = _split_qkv(qkv, B, L, nh, hd, interleaved)
        qk_raw = qk_stats = None
        if qk_ln is not None:
            if interleaved or rope is not None or qk_ln[0].requires_grad or qk_ln[1].requires_grad:
                raise NotImplementedError("qk_ln: blocked q|k|v layout, no rotary, frozen gains (the MPT-1B towers)")
            qk_raw = qkv[:, :2 * H].clone()                 # the backward of the two LayerNorms needs their inputs
            _, qm, qr = ops.layernorm_fwd(qk_raw[:, :H], qk_ln[0], None, qk_ln[2], out=qkv[:, :H])
            _, km, kr = ops.layernorm_fwd(qk_raw[:, H:], qk_ln[1], None, qk_ln[2], out=qkv[:, H:2 * H])
            qk_stats = (qm, qr, km, kr)
        if rope is not None and fused is None:
            cos, sin, rot = rope[:3]
            ops.rope_(qkv, L, nh, hs, rot, offs, cos, sin)
        o, lse = ops.attn_fwd(q, k, v, q_scale, ops.MASK_CAUSAL if causal else ops.MASK_NONE, kv_len, alibi=alibi)
        o2 = o.view(B * L, H)
        out = ops.gemm_mx(ops.mx_quantize(o2), _frozen_mx(wd), bias=bd, res=r2) if mx else \
            ops.gemm(o2, _frozen_t(wd) if td else wd, b_ks=td, bias=bd, res=r2, b_pk=None if td else _frozen_pk(wd))
        ctx.save_for_backward(x2, ln_w, mean, rstd, wqkv, wd, qkv, o, lse, kv_len, h if wqkv.requires_grad else None,
                              rope[0] if rope is not None else None, rope[1] if rope is not None else None, alibi)
        ctx.cfg = (B, L, H, nh, hd, interleaved, causal, rms, q_scale, rope[2] if rope is not None else 0, res is None,
                   ln_b is not None)
        ctx.mx = mx
        ctx.rope_fused = fused
        ctx.qk_ln = None if qk_ln is None else (qk_ln[0], qk_ln[1], qk_raw) + qk_stats
        return out.view(B, L, H)

    @staticmethod
    def _forward_packed(ctx, pack, x, res, ln_w, ln_b, wqkv, bqkv, wd, bd, rope, kv_len, nh, interleaved, causal, eps, rms, q_scale, alibi, qk_ln):
        """x [1, M, H] packed rows (functional.Pack): LayerNorm, both projections and the attention kernels on the packed rows; the
        rotation takes each row's position from pack.pos (the QKV GEMM's rotary epilogue under the same static criteria as the padded
        path, else the table pass)."""
        if qk_ln is not None:
            raise NotImplementedError("packed token order: qk_ln towers are not wired")
        B, L, M = pack.B, pack.L, pack.M
        H = x.shape[-1]
        hd = H // nh
        x2 = x.reshape(M, H)
        r2 = x2 if res is None else res.reshape(M, H)
        h, mean, rstd = ops.layernorm_fwd(x2, ln_w, ln_b, eps, rms=rms)
        tq = FROZEN_WT_ATTN and not wqkv.requires_grad and M >= 1024       # the padded path's criteria on the packed row count
        td = FROZEN_WT_ATTN and not wd.requires_grad and M >= 1024
        fused = None
        if (ROPE_EPILOGUE and rope is not None and len(rope) > 3 and not wqkv.requires_grad and not FROZEN_PK
                and (bqkv is None or not bqkv.requires_grad) and rope[2] % 8 == 0 and hd % 8 == 0 and M < (1 << 24)
                and ops.attn_generation() >= 2 and ops.gemm_rope_variant(M, 3 * H, H, tq, x.device) is not None):
            fused = dict(rot=rope[2], hd=hd, period=3 * hd if interleaved else 3 * H, span=2 * hd if interleaved else 2 * H, L=L,
                         log2_base=math.log2(rope[3]), pos=pack.pos)
        if fused is not None:
            wp = _frozen_rope_perm(wqkv, nh, hd, fused["rot"], interleaved)
            bp = _frozen_rope_perm(bqkv, nh, hd, fused["rot"], interleaved) if bqkv is not None else None
            qkv = ops.gemm(h, _frozen_t(wp) if tq else wp, b_ks=tq, bias=bp, rope=fused)
        else:
            qkv = ops.gemm(h, _frozen_t(wqkv) if tq else wqkv, b_ks=tq, bias=bqkv)
        q, k, v, hs, offs = _split_qkv(qkv, 1, M, nh, hd, interleaved)
        if rope is not None and fused is None:
            ops.rope_(qkv, L, nh, hs, rope[2], offs, rope[0], rope[1], pos=pack.pos)
        o, lse = ops.attn_fwd(q, k, v, q_scale, ops.MASK_CAUSAL if causal else ops.MASK_NONE, alibi=alibi, q_rows=pack.rows, k_rows=pack.rows)
        out = ops.gemm(o.view(M, H), _frozen_t(wd) if td else wd, b_ks=td, bias=bd, res=r2)
        ctx.save_for_backward(x2, ln_w, mean, rstd, wqkv, wd, qkv, o, lse, kv_len, h if wqkv.requires_grad else None,
                              rope[0] if rope is not None else None, rope[1] if rope is not None else None, alibi)
        ctx.cfg = (B, L, H, nh, hd, interleaved, causal, rms, q_scale, rope[2] if rope is not None else 0, res is None, ln_b is not None)
        ctx.mx, ctx.rope_fused, ctx.qk_ln, ctx.pack = False, fused, None, pack
        return out.view(1, M, H)

    @staticmethod
    def _backward_packed(ctx, dy):
        x2, ln_w, mean, rstd, wqkv, wd, qkv, o, lse, kv_len, h, cos, sin, alibi = ctx.saved_tensors
        B, L, H, nh, hd, interleaved, causal, rms, q_scale, rot, res_is_x, has_lnb = ctx.cfg
        pack = ctx.pack
        M, mask = pack.M, ops.MASK_CAUSAL if causal else ops.MASK_NONE
        _no_bias_grad(ctx, 5, "qkv bias")
        _no_bias_grad(ctx, 7, "dense bias")
        dy2 = dy.reshape(M, H)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        do = ops.gemm(dy2, wd, b_ks=True).view(1, M, nh, hd)
        dwd = ops.gemm(dy2, o.view(M, H), a_ks=True, b_ks=True) if _need(ctx, 6) else None
        q, k, v, hs, offs = _split_qkv(qkv, 1, M, nh, hd, interleaved)
        dqkv = torch.empty_like(qkv)
        if pack.nv < M:
            dqkv[pack.nv:].zero_()                         # the kernels write the sequences' rows only; the dW / dX GEMMs contract over all M
        dq, dk, dv, _, _ = _split_qkv(dqkv, 1, M, nh, hd, interleaved)
        kw = dict(alibi=alibi, q_rows=pack.rows, k_rows=pack.rows)
        if ctx.rope_fused is not None:
            if not ops.attn_rope_fusable(dq, dk, dv, rot // 2, hd, adjacent=True):
                raise RuntimeError("rotary epilogue: the attention backward cannot rotate dq / dk (kernel generation changed after the forward?)")
            ops.attn_bwd(q, k, v, o, lse, do, dq, dk, dv, q_scale, mask, rope=(rot // 2, ctx.rope_fused["log2_base"]), **kw)
            dh = ops.gemm(dqkv, _frozen_rope_perm(wqkv, nh, hd, rot, interleaved), b_ks=True)
            dwqkv = None
        else:
            fuse = ROPE_FUSE and cos is not None and cos.shape[0] >= L and cos.shape[1] * 2 == rot and ops.attn_rope_fusable(dq, dk, dv, rot // 2, hd)
            ops.attn_bwd(q, k, v, o, lse, do, dq, dk, dv, q_scale, mask, rope=(cos, sin) if fuse else None, **kw)
            if cos is not None and not fuse:
                ops.rope_(dqkv, L, nh, hs, rot, offs, cos, sin, inverse=True, pos=pack.pos)
            dwqkv = ops.gemm(dqkv, h, a_ks=True, b_ks=True) if _need(ctx, 4) else None
            dh = ops.gemm(dqkv, wqkv, b_ks=True)
        wg = _need(ctx, 2) or (has_lnb and _need(ctx, 3))
        dx, dg, db = ops.layernorm_bwd(dh, x2, ln_w, mean, rstd, dres=dy2 if res_is_x else None, want_wgrad=wg, has_beta=has_lnb, rms=rms)
        dres = None if res_is_x else dy
        return (dx.view(1, M, H), dres, dg, db, dwqkv, None, dwd, None) + (None,) * 10

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        if ctx.pack is not None:
            return SelfAttnBlockFn._backward_packed(ctx, dy)
        x2, ln_w, mean, rstd, wqkv, wd, qkv, o, lse, kv_len, h, cos, sin, alibi = ctx.saved_tensors
        B, L, H, nh, hd, interleaved, causal, rms, q_scale, rot, res_is_x, has_lnb = ctx.cfg
        _no_bias_grad(ctx, 5, "qkv bias")
        _no_bias_grad(ctx, 7, "dense bias")
        dy2 = dy.reshape(B * L, H)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        o2 = o.view(B * L, H)
        do = (ops.gemm_mx(ops.mx_quantize(dy2), _frozen_mx(wd, True)) if ctx.mx else ops.gemm(dy2, wd, b_ks=True, b_pk=_frozen_pk(wd, True))).view(B, L, nh, hd)
        dwd = ops.gemm(dy2, o2, a_ks=True, b_ks=True) if _need(ctx, 6) else None
        q, k, v, hs, offs = _split_qkv(qkv, B, L, nh, hd, interleaved)
        dqkv = torch.empty_like(qkv)
        dq, dk, dv, _, _ = _split_qkv(dqkv, B, L, nh, hd, interleaved)
        if ctx.qk_ln is not None:        # dq / dk of the NORMALISED q, k go to a side buffer; q_ln / k_ln's backward writes the fused one
            dqk_n = torch.empty((B * L, 2 * H), dtype=qkv.dtype, device=qkv.device)
            dq, dk = dqk_n[:, :H].view(B, L, nh, hd), dqk_n[:, H:].view(B, L, nh, hd)
        # the backward kernels rotate dq / dk back on their way out (same arithmetic as the separate pass, no trip through HBM)
        if ctx.rope_fused is not None:
            # q, k were rotated by the QKV GEMM in the adjacent-pair order of the permuted projection: dq / dk come back in that
            # order, rotated back by the attention kernels, and meet the same permuted rows in the dX GEMM
            if not ops.attn_rope_fusable(dq, dk, dv, rot // 2, hd, adjacent=True):
                raise RuntimeError("rotary epilogue: the attention backward cannot rotate dq / dk (kernel generation changed after the forward?)")
            ops.attn_bwd(q, k, v, o, lse, do, dq, dk, dv, q_scale, ops.MASK_CAUSAL if causal else ops.MASK_NONE, kv_len, alibi=alibi,
                         rope=(rot // 2, ctx.rope_fused["log2_base"]))
            dh = ops.gemm(dqkv, _frozen_rope_perm(wqkv, nh, hd, rot, interleaved), b_ks=True)
            dwqkv = None
        else:
            fuse = ROPE_FUSE and cos is not None and cos.shape[0] >= L and cos.shape[1] * 2 == rot and ops.attn_rope_fusable(dq, dk, dv, rot // 2, hd)
            ops.attn_bwd(q, k, v, o, lse, do, dq, dk, dv, q_scale, ops.MASK_CAUSAL if causal else ops.MASK_NONE, kv_len, alibi=alibi,
                         rope=(cos, sin) if fuse else None)
            if cos is not None and not fuse:
                ops.rope_(dqkv, L, nh, hs, rot, offs, cos, sin, inverse=True)
            if ctx.qk_ln is not None:                        # back through q_ln / k_ln, in place in the fused gradient buffer
                qw, kw, qk_raw, qm, qr, km, kr = ctx.qk_ln
                ops.layernorm_bwd(dqk_n[:, :H], qk_raw[:, :H], qw, qm, qr, has_beta=False, dx_out=dqkv[:, :H])
                ops.layernorm_bwd(dqk_n[:, H:], qk_raw[:, H:], kw, km, kr, has_beta=False, dx_out=dqkv[:, H:2 * H])
            dwqkv = ops.gemm(dqkv, h, a_ks=True, b_ks=True) if _need(ctx, 4) else None
            dh = ops.gemm_mx(ops.mx_quantize(dqkv), _frozen_mx(wqkv, True)) if ctx.mx else ops.gemm(dqkv, wqkv, b_ks=True, b_pk=_frozen_pk(wqkv, True))
        wg = _need(ctx, 2) or (has_lnb and _need(ctx, 3))
        dx, dg, db = ops.layernorm_bwd(dh, x2, ln_w, mean, rstd, dres=dy2 if res_is_x else None, want_wgrad=wg,
                                       has_beta=has_lnb, rms=rms)
        dres = None if res_is_x else dy
        return (dx.view(B, L, H), dres, dg, db, dwqkv, None, dwd, None) + (None,) * 10


def _split_qkv(qkv, B, L, nh, hd, interleaved):
    """strided [B, L, nh, hd] views of q, k, v inside the fused projection output + rope addressing."""
    H = nh * hd
    if interleaved:                      # [B, L, nh, 3*hd]
        t = qkv.view(B, L, nh, 3 * hd)
        return t[..., :hd], t[..., hd:2 * hd], t[..., 2 * hd:], 3 * hd, (0, hd)
    t = qkv.view(B, L, 3, nh, hd)        # [B, L, 3, nh, hd]
    return t[:, :, 0], t[:, :, 1], t[:, :, 2], hd, (0, H)


def self_attn_block(x, ln_w, ln_b, wqkv, bqkv, wd, bd, nh, *, rope=None, kv_len=None, interleaved=True, causal=True,
                    eps=1e-5, rms=False, res=None, q_scale=None, alibi=None, qk_ln=None):
    hd = x.shape[-1] // nh
    return SelfAttnBlockFn.apply(x, res, ln_w, ln_b, wqkv, bqkv, wd, bd, rope, kv_len, nh, interleaved, causal, eps, rms,
                                 q_scale if q_scale is not None else hd ** -0.5, alibi, qk_ln)


# ----------------------------------------------------------------------------------------------- KV-cache decode (F1)
DECODE_FUSED = _os.environ.get("UNIMP_DECODE_FUSED", "1") != "0"      # round 6: fused decode-step kernels (rope + cache append; LN inside the skinny GEMM); 0 = the round-5 launches (A/B, tests)


# the decode step's self-attention as one launch (rope + append + attention; UNIMP_DECODE_STEP_ATTN=0: rope-append, split-key partials, merge)
DECODE_STEP_ATTN = _os.environ.get("UNIMP_DECODE_STEP_ATTN", "1") != "0"
# beams: the K rows of a prompt hold identical K / V for the prompt's positions.  1 (default): by ADDRESS -- every row reads those keys from its group's
# first row, so the ten copies of the prompt become one set of lines that L2 and the memory-side cache serve ten times (the bits of the ungrouped form);
# 2: by prefix workgroups of 32 keys inside the same launch (three forms measured, all behind the ungrouped launch at the reference's sizes:
# profiles/r06_negative_results_decode_and_mx.txt); 0: every row reads its own copy
DECODE_STEP_GROUPED = int(_os.environ.get("UNIMP_DECODE_STEP_GROUPED", "1"))


def _ln_fusable(rows, D, rms):
    """decode rows whose LayerNorm the weight-streaming GEMM can take (ops.gemm(ln=...)): M <= 16, D % 512 == 0, D <= 4096, LayerNorm (not RMSNorm)"""
    return DECODE_FUSED and not rms and rows <= 16 and ops.skinny_ln_ok(rows, D)


def linear_ln(x, ln_w, ln_b, eps, w, ldc=None):
    """linear(layer_norm(x), w) for decode rows (no autograd): one launch.  Returns what ``linear`` returns."""
    shp = x.shape
    x2 = x.reshape(-1, shp[-1])
    y = ops.gemm(x2, w, ldc=ldc, ln=(ln_w, ln_b, eps))
    return y.view(*shp[:-1], w.shape[0]) if ldc in (None, w.shape[0]) else \
        y.as_strided((*shp[:-1], w.shape[0]), _lead_strides(shp[:-1], ldc) + (1,), y.storage_offset())


class LayerKV:
    """decode state of one decoder layer: views ``k``, ``v`` [rows, capacity, nh, hd] into the cache's single K/V tensor
    (keys after RoPE) and the gated cross-attention's projected media ``xkv`` [rows, T*n, 2*inner] (constant over a decode)."""
    __slots__ = ("owner", "k", "v", "xkv", "pages")

    def __init__(self, owner):
        self.owner = weakref.proxy(owner)      # no DecodeCache <-> LayerKV cycle: the K/V tensor must die with its last user, not at the next gc pass
        self.k = self.v = self.xkv = None
        self.pages = None                      # Kv4Cache: this layer's pool [n_pages, heads, page bytes] instead of k / v


class StepState:
    """device-resident positions of a static decode step, one per row (rows may sit at different lengths: a batch of
    prompts): ``pos_idx`` int64 [rows] = slot the row's new K/V go to, ``kv_len`` int32 [rows] = keys visible to it
    (pos + 1).  Nothing on the host depends on the positions, so one step can be captured in a HIP graph and replayed
    (decode.py)."""

    def __init__(self, rows, pos, device):
        """pos: int (all rows) or an integer tensor [rows]."""
        if torch.is_tensor(pos):
            self.pos_idx = pos.to(device=device, dtype=torch.long).clone()
        else:
            self.pos_idx = torch.full((rows,), pos, dtype=torch.long, device=device)
        self.kv_len = (self.pos_idx + 1).to(torch.int32)
        self.rows = torch.arange(rows, dtype=torch.long, device=device)

    def advance(self):
        self.pos_idx.add_(1)
        self.kv_len.add_(1)


class DecodeCache:
    """``past_key_values`` of the towers (inference only).  One tensor ``kv`` [layers, 2, rows, capacity, nh, hd] holds
    every layer's keys and values, ``len`` tokens are cached per row; ``media_count`` [rows, 1] int32 is the number of
    <image> tokens in the prompt = the text_time every generated token attends with (open_flamingo ``use_cached_media``,
    SURVEY.md A.3).  ``shared_prefix``: the first tokens are identical in all rows that can exchange hypotheses (the
    beams of one prompt), so a beam reorder only has to move the generated tail."""

    def __init__(self, n_layers, capacity=0):
        self.layers = [LayerKV(self) for _ in range(n_layers)]
        self.len = 0
        self.capacity = capacity
        self.kv = None
        self.media_count = None
        self.row_len = None                # prefill of right-padded prompts: valid tokens per row (device tensor)
        self.shared_prefix = 0
        self.group, self.shared_len = 1, None     # beam search: rows per prompt and int32 [prompts] prefix length whose K / V the rows of a group share
        self.step = None                   # StepState while decoding with device-side positions

    def _reserve(self, like, need):
        R, _, nh, hd = like.shape
        if self.kv is not None and self.kv.shape[3] >= need:
            return
        cap = max(self.capacity, need + 64) if self.kv is None else max(need + 64, 2 * self.kv.shape[3])
        # zeros, not empty: the kernels load whole 64-key tiles and weight the slots beyond kv_len with p = 0, which
        # only cancels finite values (0 * NaN from recycled memory would poison the row)
        new = torch.zeros((len(self.layers), 2, R, cap, nh, hd), dtype=like.dtype, device=like.device)
        if self.kv is not None:
            new[:, :, :, :self.kv.shape[3]].copy_(self.kv)      # a layer may grow it mid-forward: keep every slot
        self.kv = new
        for i, l in enumerate(self.layers):
            l.k, l.v = new[i, 0], new[i, 1]

    def reorder(self, idx):
        """beam search: row r continues the hypothesis that lived in row idx[r].  The projected media are not moved:
        beams of one batch item share their images, and a beam never migrates to another item."""
        if self.kv is not None and self.len > self.shared_prefix:
            tail = self.kv[:, :, :, self.shared_prefix:self.len]
            tail.copy_(tail.index_select(2, idx))
        if self.media_count is not None:
            self.media_count = self.media_count.index_select(0, idx)


class Kv4Cache(DecodeCache):
    """the decode state with K / V on 4-bit pages (ops.kv4_*): ``pages`` uint8 [layers, n_pages, heads, page bytes], ``tables`` int32 [rows, columns] naming each row's
    pages (32 tokens each, the same for all layers).  The rows of a beam group share the pages of their prompt; every row has pages of its own from the one that its first
    generated token goes to.  Made of a finished prefill's bf16 cache: 17 / 64 of its bytes per token, the prompt once instead of once per beam."""

    def __init__(self, prompts, host_len, beams, max_new):
        """prompts: the prefill's DecodeCache (one row per prompt); host_len: the prompts' lengths; max_new: tokens that every row may still take"""
        super().__init__(len(prompts.layers))
        _, _, B, cap, nh, hd = prompts.kv.shape
        if beams > 16:
            raise ValueError(f"the 4-bit cache holds at most 16 beams of a prompt, not {beams}")
        dev, K, P = prompts.kv.device, beams, ops.KV4_PAGE
        cols = [-(-(n + max_new) // P) for n in host_len]
        n_pages = sum(c + (K - 1) * (c - n // P) for c, n in zip(cols, host_len))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        self.pages = torch.empty((len(prompts.layers), n_pages, nh, ops.kv4_page_bytes(hd)), dtype=torch.uint8, device=dev)
        self.tables = torch.full((B * K, max(cols)), -1, dtype=torch.int32, device=dev)
        self.group, self.shared_len = K, i32(host_len) if K > 1 else None
        self.free, self.ones = torch.arange(n_pages, dtype=torch.int32, device=dev), torch.ones(B * K, dtype=torch.int32, device=dev)
        length = i32(host_len).repeat_interleave(K)
        first = (torch.arange(B * K, device=dev) % K == 0).to(torch.int32)
        zero = torch.zeros(B * K, dtype=torch.int32, device=dev)
        self.mapped, self.cursor, slots, cu = ops.page_tables_extend(self.tables, zero, zero, length * first, self.free, zero[:1], sum(host_len), cover=length + max_new,
                                                                     group=K, shared_len=self.shared_len)
        t = torch.arange(cap, device=dev)                      # the packed tokens' slots, spread to the padded rows of the prefill's cache
        at = (cu[:-1:K].long()[:, None] + t).clamp_(max=sum(host_len) - 1)
        slots = torch.where(t < length[::K, None], slots[at], torch.full((), -1, dtype=torch.long, device=dev)).reshape(-1)
        for lk, lp, pages in zip(self.layers, prompts.layers, self.pages):
            lk.pages = pages
            ops.kv4_write(lp.k.view(B * cap, nh, hd), lp.v.view(B * cap, nh, hd), pages, slots)
        self.cached = length                                    # tokens in the cache, per row
        self.slots = None                                       # of the step's new tokens
        if K > 1:                                               # the page in which a prompt ends: every beam goes on in its own copy
            self.reorder_beams(torch.zeros(B * K, dtype=torch.long, device=dev), length.long())

    def reorder(self, idx):
        raise NotImplementedError("Kv4Cache: beams are reordered inside their groups (reorder_beams)")

    def reorder_beams(self, src_local, pos):
        """row j of every group goes on with the hypothesis of row src_local of its group (index inside the group); pos int64 [rows] = tokens cached"""
        ops.kv4_reorder_beams(self.pages, self.tables, self.group, src_local, pos)

    def begin_step(self):
        """the slots of the step's new tokens, one per row, from the rows' lengths (every column is mapped from the start: nothing is taken from the free list)"""
        self.slots = ops.page_tables_extend(self.tables, self.mapped, self.cached, self.ones, self.free, self.cursor, self.tables.shape[0])[2]

    def end_step(self):
        self.cached.add_(1)


def _kv_append(lc, k, v, pos0):
    need = pos0 + k.shape[1]
    lc.owner._reserve(k, need)
    lc.k[:, pos0:need].copy_(k)
    lc.v[:, pos0:need].copy_(v)
    return lc.k[:, :need], lc.v[:, :need]


@torch.no_grad()
def _decode_attn(q, k, v, scale, kv_len, alibi, group=1, shared_len=None):
    """one new token per row against the cache: the split-key kernel (HBM-bound, every CU busy; with ``group`` beams per prompt
    the prompt's keys are read once per prompt), or -- UNIMP_DECODE_ATTN=0, odd layouts -- the training kernel on one query row."""
    if ops.DECODE_ATTN and q.shape[-1] % 8 == 0 and q.shape[-1] <= 128:
        if not ops.DECODE_SHARED_PREFIX:
            group, shared_len = 1, None
        return ops.attn_decode(q, k, v, scale, kv_len, alibi, group=group, shared_len=shared_len)
    return ops.attn_fwd(q, k, v, scale, ops.MASK_NONE, kv_len, alibi=alibi)[0]


def self_attn_block_cached(x, ln_w, ln_b, wqkv, bqkv, wd, bd, nh, lc, pos0, *, rope=None, interleaved=True, eps=1e-5,
                           rms=False, res=None, q_scale=None, alibi=None, qk_ln=None):
    """SelfAttnBlockFn.forward for decoding: the new rows' keys/values are appended to ``lc``; a prefill (pos0 == 0) runs
    the causal kernel on the prompt, a decode step (one new token per row) attends to every cached key.  With
    ``lc.owner.step`` set the position lives on the device (StepState): ``rope`` then holds the one table row of the
    current position, K/V go to slot ``pos_idx`` and the kernel reads the visible length from ``kv_len``."""
    R, Ln, H = x.shape
    hd = H // nh
    step = lc.owner.step
    x2 = x.reshape(R * Ln, H)
    r2 = x2 if res is None else res.reshape(R * Ln, H)
    if _ln_fusable(R * Ln, H, rms) and lc.owner.step is not None:
        qkv = ops.gemm(x2, wqkv, bias=bqkv, ln=(ln_w, ln_b, eps))       # decode rows: the LayerNorm runs inside the weight-streaming GEMM
    else:
        h, _, _ = ops.layernorm_fwd(x2, ln_w, ln_b, eps, rms=rms)
        qkv = ops.gemm(h, wqkv, bias=bqkv)
    q, k, v, hs, offs = _split_qkv(qkv, R, Ln, nh, hd, interleaved)
    if qk_ln is not None:                      # LayerNorm over the whole d_model vector of q and of k, in place (one wave holds a row)
        qn, _, _ = ops.layernorm_fwd(qkv[:, :H], qk_ln[0], None, qk_ln[2])
        kn, _, _ = ops.layernorm_fwd(qkv[:, H:2 * H], qk_ln[1], None, qk_ln[2])
        qkv[:, :H].copy_(qn)
        qkv[:, H:2 * H].copy_(kn)
    scale = q_scale if q_scale is not None else hd ** -0.5
    if step is not None:
        if Ln != 1:
            raise NotImplementedError("a static decode step feeds one new token per row")
        rot = rope[2] if rope is not None else 0
        o3 = (offs[0], offs[1], (2 * hd) if interleaved else 2 * H)       # q, k, v element offsets inside a head slot (_split_qkv)
        if lc.pages is not None:               # 4-bit pages: rotate + quantise + append, then the attention over the pages
            own = lc.owner
            q = ops.kv4_rope_append(qkv, nh, hs, hd, o3, rot, rope[0] if rot else None, rope[1] if rot else None, lc.pages, own.slots)
            o = ops.kv4_attn_decode(q, lc.pages, own.tables, step.kv_len, scale, alibi, own.group, own.shared_len)
            return ops.gemm(o.view(R, H), wd, bias=bd, res=r2).view(R, 1, H)
        fused = DECODE_FUSED and qk_ln is None and ops.decode_rope_append_ok(hd, rot, hs, o3, qkv, lc.k)
        if fused and DECODE_STEP_ATTN and ops.DECODE_ATTN and hd <= 128:
            # the whole attention in ONE launch: rope of the new q / k, the append, every cached key (csrc/decode_attn.hip attn_decode_step_kernel);
            # beam search: the prompt's keys once per prompt, by extra workgroups of the same launch
            grp = lc.owner.group if DECODE_STEP_GROUPED else 1
            o = ops.attn_decode_step(qkv, nh, hs, hd, o3, rot, rope[0] if rot else None, rope[1] if rot else None, lc.k, lc.v, step.pos_idx,
                                     scale, alibi, grp, lc.owner.shared_len if grp > 1 else None, group_mode=1 if DECODE_STEP_GROUPED == 2 else 0)
            return ops.gemm(o.view(R, H), wd, bias=bd, res=r2).view(R, 1, H)
        if fused:
            # one launch: rotate q / k (row r at its own position) and write the rotated k and v into their cache slots
            ops.decode_rope_append(qkv, nh, hs, hd, o3, rot, rope[0] if rot else None, rope[1] if rot else None, lc.k, lc.v, step.pos_idx)
        else:
            if rope is not None:               # rope = the table rows of the R positions: "sequence" of R rows, row r at its own position
                ops.rope_(qkv, R, nh, hs, rope[2], offs, rope[0], rope[1])
            lc.k.index_put_((step.rows, step.pos_idx), k[:, 0])
            lc.v.index_put_((step.rows, step.pos_idx), v[:, 0])
        o = _decode_attn(q, lc.k, lc.v, scale, step.kv_len, alibi, lc.owner.group, lc.owner.shared_len)
        return ops.gemm(o.view(R, H), wd, bias=bd, res=r2).view(R, 1, H)
    if rope is not None:
        cos, sin, rot = rope[:3]
        ops.rope_(qkv, Ln, nh, hs, rot, offs, cos[pos0:], sin[pos0:])
    kc, vc = _kv_append(lc, k, v, pos0)
    if pos0 == 0:
        o, _ = ops.attn_fwd(q, k, v, scale, ops.MASK_CAUSAL, lc.owner.row_len, alibi=alibi)       # row_len: right-padded prompts
    else:
        if Ln != 1:
            raise NotImplementedError("cached decode feeds one new token per row (chunked prefill is not built)")
        o = _decode_attn(q, kc, vc, scale, None, alibi)
    return ops.gemm(o.view(R * Ln, H), wd, bias=bd, res=r2).view(R, Ln, H)


@torch.no_grad()
def gated_xattn_cached(x, media, seg, ln_w, ln_b, wq, wkv, wo, gate, heads, n_lat, lc, eps=1e-5):
    """GatedXAttnFn.forward for decoding: to_kv(media) is projected once per decode and kept in ``lc.xkv``."""
    R, Ln, D = x.shape
    Sk = media.shape[1]
    inner = wq.shape[0]
    dh = inner // heads
    x2 = x.reshape(R * Ln, D)
    if _ln_fusable(R * Ln, D, False) and lc.xkv is not None:
        q = ops.gemm(x2, wq, ln=(ln_w, ln_b, eps))
    else:
        h, _, _ = ops.layernorm_fwd(x2, ln_w, ln_b, eps)
        q = ops.gemm(h, wq)
    if lc.xkv is None:
        lc.xkv = ops.gemm(media.reshape(R * Sk, -1), wkv)
    kv5 = lc.xkv.view(R, Sk, 2, heads, dh)
    o, _ = ops.attn_fwd(q.view(R, Ln, heads, dh), kv5[:, :, 0], kv5[:, :, 1], dh ** -0.5, ops.MASK_SEGMENT, None, seg, n_lat)
    return ops.gemm(o.view(R * Ln, inner), wo, gate=gate, res=x2).view(R, Ln, D)


# ----------------------------------------------------------------------------------------------- gated cross-attention
class GatedXAttnFn(Function):
    """out = x + tanh(gate) * to_out(softmax_seg(to_q(LN(x)) to_kv(media)^T) V)   (open_flamingo MaskedCrossAttention)."""

    @staticmethod
    def forward(ctx, x, media, seg, ln_w, ln_b, wq, wkv, wo, gate, heads, n_lat, eps):
        pack = PACK                               # packed token order: x is [1, M, D]; q, o (and seg) as row ranges of the packed buffer
        ctx.pack = pack
        Sk = media.shape[1]                       # media [B, T*n, Dv]
        B = media.shape[0]
        D = x.shape[-1]
        L = pack.L if pack is not None else x.shape[1]
        rows = pack.M if pack is not None else B * L
        inner = wq.shape[0]
        dh = inner // heads
        x2 = x.reshape(rows, D)
        m2 = media.reshape(B * Sk, -1)
        h, mean, rstd = ops.layernorm_fwd(x2, ln_w, ln_b, eps)
        q = ops.gemm(h, wq)
        kv = ops.gemm(m2, wkv)
        kv5 = kv.view(B, Sk, 2, heads, dh)
        if pack is not None:
            seg = pack.seg(seg)
            o, lse = ops.attn_fwd(q.view(1, rows, heads, dh), kv5[:, :, 0], kv5[:, :, 1], dh ** -0.5, ops.MASK_SEGMENT, None, seg, n_lat, q_rows=pack.rows)
        else:
            o, lse = ops.attn_fwd(q.view(B, L, heads, dh), kv5[:, :, 0], kv5[:, :, 1], dh ** -0.5, ops.MASK_SEGMENT, None, seg, n_lat)
        out = ops.gemm(o.view(rows, inner), wo, gate=gate, res=x2)
        ctx.save_for_backward(x2, m2, seg, ln_w, mean, rstd, wq, wkv, wo, gate, h, q, kv, o, lse)
        ctx.cfg = (B, L, D, Sk, heads, dh, n_lat)
        ctx.ln_b_ref = ln_b
        return out.view(x.shape)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, m2, seg, ln_w, mean, rstd, wq, wkv, wo, gate, h, q, kv, o, lse = ctx.saved_tensors
        B, L, D, Sk, heads, dh, n_lat = ctx.cfg
        pack = ctx.pack
        inner = heads * dh
        dy2 = dy.reshape(-1, D)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        rows = dy2.shape[0]
        o2 = o.view(rows, inner)
        # do is kept UN-gated: d/d gate of tanh(gate) * (o Wo^T) contracted with dy is <dy Wo, o> -- a dot over [B L, inner] instead
        # of one over dy and a saved copy of the un-gated block output (both [B L, D], D = 5 inner: the copy and its store in the
        # forward's epilogue are gone) -- and everything downstream of do is linear in it, so tanh(gate) moves into the epilogues
        # of the four GEMMs that consume dq / dkv (0 at initialisation there exactly as it was here)
        do2 = ops.gemm(dy2, wo, b_ks=True)
        dgate = _gate_grad(do2, o2, gate) if _need(ctx, 8) else None
        dwo = _dw(ctx, 7, wo, dy2, o2, gate=gate)
        dq = torch.empty_like(q)
        dkv = torch.empty_like(kv)
        kv5, dkv5 = kv.view(B, Sk, 2, heads, dh), dkv.view(B, Sk, 2, heads, dh)
        qshape = (B, L, heads, dh) if pack is None else (1, rows, heads, dh)
        if pack is not None and pack.nv < rows:
            dq[pack.nv:].zero_()                         # rows behind the last sequence: not written by the kernels, contracted by dwq / dh_
        ops.attn_bwd(q.view(qshape), kv5[:, :, 0], kv5[:, :, 1], o, lse, do2.view(qshape), dq.view(qshape),
                     dkv5[:, :, 0], dkv5[:, :, 1], dh ** -0.5, ops.MASK_SEGMENT, None, seg, n_lat, q_rows=pack.rows if pack is not None else None)
        dwq = _dw(ctx, 5, wq, dq, h, gate=gate)
        dh_ = ops.gemm(dq, wq, b_ks=True, gate=gate)
        dwkv = _dw(ctx, 6, wkv, dkv, m2, gate=gate)
        dmedia = ops.gemm(dkv, wkv, b_ks=True, gate=gate).view(B, Sk, -1) if _need(ctx, 1) else None
        dx, dg, db = _ln_bwd(dh_, x2, ln_w, ctx.ln_b_ref, mean, rstd, _need(ctx, 3), _need(ctx, 4), dres=dy2)
        return dx.view(dy.shape), dmedia, None, dg, db, dwq, dwkv, dwo, dgate, None, None, None


def gated_xattn(x, media, seg, ln_w, ln_b, wq, wkv, wo, gate, heads, n_lat, eps=1e-5):
    return GatedXAttnFn.apply(x, media, seg, ln_w, ln_b, wq, wkv, wo, gate, heads, n_lat, eps)


# ----------------------------------------------------------------------------------------------- Perceiver attention
class PerceiverAttnFn(Function):
    """out = latents + to_out(softmax(to_q(LN_l(lat)) [to_kv(LN_m(x)); to_kv(LN_l(lat))]^T) V)   (open_flamingo A.2).
    x: [G, n1, D] media tokens of G = b*T images, lat: [G, n2, D]."""

    @staticmethod
    def forward(ctx, x, lat, nm_w, nm_b, nl_w, nl_b, wq, wkv, wo, heads, eps):
        G, n1, D = x.shape
        n2 = lat.shape[1]
        inner = wq.shape[0]
        dh = inner // heads
        S = n1 + n2
        x2, l2 = x.reshape(G * n1, D), lat.reshape(G * n2, D)
        kvin = torch.empty((G * S, D), dtype=bf16, device=x.device)
        _, mean_m, rstd_m = ops.layernorm_fwd(x2, nm_w, nm_b, eps, out=kvin, grp=n1, grp_stride=S, grp_off=0)
        _, mean_l, rstd_l = ops.layernorm_fwd(l2, nl_w, nl_b, eps, out=kvin, grp=n2, grp_stride=S, grp_off=n1)
        hl, _, _ = ops.layernorm_fwd(l2, nl_w, nl_b, eps)
        q = ops.gemm(hl, wq)
        kv = ops.gemm(kvin, wkv)
        kv5 = kv.view(G, S, 2, heads, dh)
        o, lse = ops.attn_fwd(q.view(G, n2, heads, dh), kv5[:, :, 0], kv5[:, :, 1], dh ** -0.5, ops.MASK_NONE)
        out = ops.gemm(o.view(G * n2, inner), wo, res=l2)
        ctx.save_for_backward(x2, l2, nm_w, nl_w, mean_m, rstd_m, mean_l, rstd_l, wq, wkv, wo, kvin, hl, q, kv, o, lse)
        ctx.cfg = (G, n1, n2, D, heads, dh)
        ctx.nm_b_ref, ctx.nl_b_ref = nm_b, nl_b
        return out.view(G, n2, D)

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        x2, l2, nm_w, nl_w, mean_m, rstd_m, mean_l, rstd_l, wq, wkv, wo, kvin, hl, q, kv, o, lse = ctx.saved_tensors
        G, n1, n2, D, heads, dh = ctx.cfg
        inner, S = heads * dh, n1 + n2
        dy2 = dy.reshape(G * n2, D)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        o2 = o.view(G * n2, inner)
        do = ops.gemm(dy2, wo, b_ks=True).view(G, n2, heads, dh)
        dwo = _dw(ctx, 8, wo, dy2, o2)
        dq, dkv = torch.empty_like(q), torch.empty_like(kv)
        kv5, dkv5 = kv.view(G, S, 2, heads, dh), dkv.view(G, S, 2, heads, dh)
        ops.attn_bwd(q.view(G, n2, heads, dh), kv5[:, :, 0], kv5[:, :, 1], o, lse, do, dq.view(G, n2, heads, dh),
                     dkv5[:, :, 0], dkv5[:, :, 1], dh ** -0.5, ops.MASK_NONE)
        dwq = _dw(ctx, 6, wq, dq, hl)
        dhl = ops.gemm(dq, wq, b_ks=True)
        dwkv = _dw(ctx, 7, wkv, dkv, kvin)
        dkvin = ops.gemm(dkv, wkv, b_ks=True)                                   # [G*S, D]
        dxm = dgm = dbm = None
        if _need(ctx, 0) or _need(ctx, 2) or _need(ctx, 3):
            dxm, dgm, dbm = _ln_bwd(dkvin, x2, nm_w, ctx.nm_b_ref, mean_m, rstd_m, _need(ctx, 2), _need(ctx, 3),
                                    grp=n1, grp_stride=S, grp_off=0)
            dxm = dxm.view(G, n1, D) if _need(ctx, 0) else None
        dl, dgl, dbl = _ln_bwd(dkvin, l2, nl_w, ctx.nl_b_ref, mean_l, rstd_l, _need(ctx, 4), _need(ctx, 5), dres=dy2, dy2=dhl,
                               grp=n2, grp_stride=S, grp_off=n1)
        return dxm, dl.view(G, n2, D), dgm, dbm, dgl, dbl, dwq, dwkv, dwo, None, None


def perceiver_attn(x, lat, nm_w, nm_b, nl_w, nl_b, wq, wkv, wo, heads, eps=1e-5):
    return PerceiverAttnFn.apply(x, lat, nm_w, nm_b, nl_w, nl_b, wq, wkv, wo, heads, eps)


class BcastRowsFn(Function):
    """latents "n d -> (G n) d" repeat and its adjoint."""

    @staticmethod
    def forward(ctx, lat, G):
        ctx.n = lat.shape[0]
        return ops.bcast_rows(lat, G * lat.shape[0])

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        return ops.reduce_rows_periodic(dy.contiguous(), ctx.n), None


# ----------------------------------------------------------------------------------------------- embedding
class EmbeddingFn(Function):
    @staticmethod
    def forward(ctx, ids, w, pos, pw):
        ctx.save_for_backward(ids, pos)
        ctx.vocab, ctx.npos = w.shape[0], (pw.shape[0] if pw is not None else 0)
        out = ops.embedding_fwd(ids.reshape(-1), w, pos.reshape(-1) if pos is not None else None, pw)
        return out.view(*ids.shape, w.shape[1])

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dy):
        ids, pos = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dw = ops.embedding_bwd(ids.reshape(-1), dy2, ctx.vocab) if _need(ctx, 1) else None
        dp = ops.embedding_bwd(pos.reshape(-1), dy2, ctx.npos) if (pos is not None and _need(ctx, 3)) else None
        return None, dw, None, dp


def embedding(ids, w, pos=None, pw=None):
    return EmbeddingFn.apply(ids, w, pos, pw)


# ----------------------------------------------------------------------------------------------- weighted focal CE
class FocalCEFn(Function):
    """loss = sum_rows w_b * ce * (1 - p_y)^gamma / #labeled   (UniMP/mmrec.py:190-213; focal term NOT detached).
    Also yields the HF-style unweighted mean CE (logged only, mmrec.py:182)."""

    @staticmethod
    def forward(ctx, logits, labels, weights, gamma, use_reweight):
        B, L, V = logits.shape
        assert logits.stride(2) == 1 and logits.stride(0) == L * logits.stride(1)
        lse, zy, out3 = ops.focal_ce_fwd(logits, V, labels, weights, gamma, use_reweight)
        ctx.save_for_backward(logits, labels, weights, lse, zy, out3)
        ctx.cfg = (gamma, use_reweight)
        loss = out3[0] / out3[1]
        ctx.mark_non_differentiable(out3)
        return loss, out3

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dloss, _):
        logits, labels, weights, lse, zy, out3 = ctx.saved_tensors
        gamma, rw = ctx.cfg
        B, L, V = logits.shape
        ldv = logits.stride(1)
        buf = torch.empty((B, L, ldv), dtype=bf16, device=logits.device)
        dl = buf[..., :V]
        ops.focal_ce_bwd(logits, V, labels, weights, gamma, rw, lse, zy, out3, dloss.float().reshape(1), dl)
        return dl, None, None, None, None


class SparseHeadLossFn(Function):
    """Head + weighted focal CE on the supervised rows only: ``h_rows`` [n, H] are the hidden states of the n positions
    whose next token carries a label, ``targets`` [n] those labels, ``row_w`` [n] the per-sample weights.  The same loss,
    dX and dW as LinearFn + FocalCEFn over all B*L rows (rows with label -100 contribute nothing to either), without the
    (B*L) x V logits: the rows are laid out as n two-token sequences so the unchanged focal kernels see
    logits[:, :-1] against labels[:, 1:]."""

    @staticmethod
    def forward(ctx, h_rows, w, targets, row_w, gamma, use_reweight):
        n, V = h_rows.shape[0], w.shape[0]
        ldv = (V + 7) // 8 * 8
        buf = torch.empty((n, 2, ldv), dtype=bf16, device=h_rows.device)
        ops.gemm(h_rows, w, out=buf.view(n, 2 * ldv)[:, :V])
        logits = buf[..., :V]
        labels = torch.stack([torch.full_like(targets, -100), targets], 1)
        lse, zy, out3 = ops.focal_ce_fwd(logits, V, labels, row_w, gamma, use_reweight)
        ctx.save_for_backward(h_rows, w, logits, labels, row_w, lse, zy, out3)
        ctx.cfg = (gamma, use_reweight)
        ctx.mark_non_differentiable(out3)
        return out3[0] / out3[1], out3

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dloss, _):
        h_rows, w, logits, labels, row_w, lse, zy, out3 = ctx.saved_tensors
        gamma, rw = ctx.cfg
        n, _, V = logits.shape
        ldv = logits.stride(1)
        buf = torch.empty((n, 2, ldv), dtype=bf16, device=logits.device)
        ops.focal_ce_bwd(logits, V, labels, row_w, gamma, rw, lse, zy, out3, dloss.float().reshape(1), buf[..., :V])
        dl = buf.view(n, 2 * ldv)[:, :V]                          # row i of the first position, leading dimension 2*ldv
        dh = ops.gemm(dl, w, b_ks=True) if _need(ctx, 0) else None
        dw = ops.gemm(dl, h_rows, a_ks=True, b_ks=True) if _need(ctx, 1) else None
        return dh, dw, None, None, None, None


class DenseHeadLossFn(Function):
    """LM head + weighted focal CE in one node: the FORWARD is the reference's -- dense logits for all B*L positions (returned,
    non-differentiable, as the model's ``output["logits"]``: mmrec.py:190) and the loss over them (mmrec.py:190-213); the
    BACKWARD touches the labeled positions only.  d loss / d logits is exactly zero on every row whose next token carries no
    label (~98 % of the rows: 10 answers in 512 tokens), so the dense [B*L, V] gradient the reference materialises, and the
    zero rows of its dX = dlogits W and dW = dlogits^T h products, are never formed: ``rows`` (b*L + j of the scored
    positions, from the label mask) selects the n rows whose gradient is written compactly [n, V]; dX is scattered back
    into a zero [B*L, H] tensor and dW contracts over the n rows.  Same gradients as LinearFn + FocalCEFn
    (tests/test_model_gpu.py::test_compact_head_backward_equals_dense)."""

    @staticmethod
    def forward(ctx, h, w, labels, weights, rows, gamma, use_reweight):
        B, L, H = h.shape
        V = w.shape[0]
        ldv = (V + 7) // 8 * 8
        h2 = h.reshape(B * L, H)
        y = ops.gemm(h2, w, ldc=ldv)                                                    # [B*L, V] view, leading dimension ldv
        logits = y.as_strided((B, L, V), (L * ldv, ldv, 1), y.storage_offset())
        lse, zy, out3 = ops.focal_ce_fwd(logits, V, labels, weights, gamma, use_reweight)
        ctx.save_for_backward(h2, w, logits, labels, weights, lse, zy, out3, rows)
        ctx.cfg = (gamma, use_reweight, B, L, H)
        ctx.mark_non_differentiable(out3, logits)
        return out3[0] / out3[1], out3, logits

    @staticmethod
    @ops.backward_scope
    def backward(ctx, dloss, _a, _b):
        h2, w, logits, labels, weights, lse, zy, out3, rows = ctx.saved_tensors
        gamma, rw, B, L, H = ctx.cfg
        V = w.shape[0]
        dh = torch.zeros((B * L, H), dtype=bf16, device=h2.device) if _need(ctx, 0) else None
        dw = None
        if rows.numel() > 0:
            dl = ops.focal_ce_bwd_rows(logits, V, labels, weights, gamma, rw, lse, zy, out3, dloss.float().reshape(1), rows)
            if dh is not None:
                dh.index_copy_(0, rows, ops.gemm(dl, w, b_ks=True))                       # rows are distinct positions
            if _need(ctx, 1):
                dw = ops.gemm(dl, h2.index_select(0, rows), a_ks=True, b_ks=True)
        # no labeled row: the head's gradient is zero -- None, not a [V, H] tensor of zeros
        return (dh.view(B, L, H) if dh is not None else None), dw, None, None, None, None, None


def dense_head_loss(h, w, labels, weights, rows, gamma, use_reweight=True):
    """returns (loss, stats, logits [B, L, V]); see DenseHeadLossFn."""
    return DenseHeadLossFn.apply(h, w, labels, weights, rows, float(gamma), bool(use_reweight))


def sparse_head_loss(h_rows, w, targets, row_w, gamma, use_reweight=True):
    return SparseHeadLossFn.apply(h_rows, w, targets, row_w, float(gamma), bool(use_reweight))


def focal_ce(logits, labels, weights, gamma, use_reweight=True):
    """returns (loss, stats) with stats = [loss_sum, n_labeled, ce_sum] (fp32 device tensor)."""
    return FocalCEFn.apply(logits, labels, weights, float(gamma), bool(use_reweight))
