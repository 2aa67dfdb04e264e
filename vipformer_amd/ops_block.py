"""Operators of a transformer block over long token sequences (image patches, point groups, video patches), beside the attention,
LayerNorm and residual pieces of ops.py:

  rotary_axes           rotary positions with several axes (height / width, x / y / z, time / height / width) on queries and keys
  window_attention      attention inside a sliding window with first tokens that stay visible; training, prompts, single tokens over a cache
  gated_norm_residual   h = alpha x + beta gate * post(y), n = pre(h): the norms around a block with its gate and residual scale

Heads are a dimension of their own ([B, L, heads, head_dim], any strides whose last dimension is contiguous: slices of one projection's
output go in as they are).  fp16 and bf16 are chosen by the tensors, per call; the library's build-time operand type does not matter here.
Every operator is asynchronous on torch's current stream of the tensors' device, differentiable once (in backward mode; a forward-mode tangent
raises), and may be captured into a HIP graph once it has run there (a RotaryAxes makes its tables at its first use on a device).  As everywhere
in torch, a backward pass is captured only while no eager graph of the same leaves is alive (train.GraphedStep).  Saved tensors may travel
through hooks (offload, recomputation); what comes back with another type, shape or device is refused.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L
from . import ops

F32 = torch.float32
_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}                   # VPF_T_*
_POS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}       # VPF_POS_*
_pack_rotary, _pack_norm, _pack_attn = (L.packer(c).pack for c in (L.Rotary, L.GatedNorm, L.WindowAttn))


def _same_device(what: str, first: torch.Tensor, *rest) -> None:
    dev = first.device
    if dev.type != "cuda":
        L.need_cuda(first)
    for t in rest:
        if t is not None and t.device != dev:
            L.need_cuda(t)
            raise L.VpfError(f"{what}: tensors on {dev} and {t.device}")


def _wants_grad(*ts) -> bool:
    """Does the call go through its autograd Function?  A tensor with a tangent need not require a gradient: while a forward-mode level is open the
    Function decides (it has no forward-mode rule, so torch raises where one is needed)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _once(what: str) -> None:
    """The kernels' gradients carry no graph of their own."""
    if torch.is_grad_enabled():
        raise L.VpfError(f"{what} is differentiable once (backward was called with create_graph=True)")


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


_top_hooks = torch._C._autograd._top_saved_tensors_default_hooks


def _keep(ctx, *ts) -> None:
    ctx.save_for_backward(*ts)
    ctx.at = None if _top_hooks(False) is not None else [_ptr(t) for t in ts]      # None: hooks take them from here


def _kept(ctx, what: str, want):
    """(the saved tensors, are they where they were?).  The kernels take addresses: tensors that lie elsewhere (a saved-tensor hook brought them back,
    or their storage was filled anew) are looked at before they go there.  want(): (shape, type, device) of each, None to leave one out."""
    ts = ctx.saved_tensors
    if [_ptr(t) for t in ts] == ctx.at:
        return ts, True
    for t, w in zip(ts, want()):
        if t is not None and (t.shape, t.dtype, t.device) != w:
            raise L.VpfError(f"{what}: a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}, it was {w[1]} {tuple(w[0])} on {w[2]}")
    return ts, False


def _dense(t):
    """A saved tensor that was contiguous.  (What a saved-tensor hook brings back has its values and shape; strides and address are its own.)"""
    return None if t is None else t.contiguous()


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    """Batch, token and head stride; 0 where the size is 1 (torch leaves any number there)."""
    sb, sl, sh, _ = t.stride()
    nb, nl, nh, _ = t.shape
    return (sb if nb > 1 else 0, sl if nl > 1 else 0, sh if nh > 1 else 0)


# --------------------------------------------------------------------------- rotary positions with several axes
class RotaryAxes:
    """How the channel pairs of a head turn: ``sections[a]`` pairs belong to axis ``a`` of the positions, the channels behind the
    ``2 * sum(sections)`` rotated ones stay as they are.

    ladder "axis":  pair j of the n pairs of an axis turns by  position * base ** (-j / n)   (every axis sees all wavelengths)
    ladder "joint": pair p of all P pairs turns by             position[its axis] * base ** (-p / P)
    layout "half":  pair p is the channels (p, p + P);  "pair": the channels (2 p, 2 p + 1)

    Build it once per model; its tables (fp64 frequencies, axis numbers) are made once per device."""

    def __init__(self, sections: Sequence[int], head_dim: int, base: float = 10000.0, layout: str = "half", ladder: str = "axis"):
        self.sections, self.head_dim, self.base = tuple(int(n) for n in sections), int(head_dim), float(base)
        P = sum(self.sections)
        if not 1 <= len(self.sections) <= 8 or min(self.sections) < 0 or P < 1:
            raise L.VpfError(f"RotaryAxes: sections {tuple(sections)}: 1 to 8 axes with at least one pair in all")
        if self.head_dim % 2 or not 2 * P <= self.head_dim <= 1024:
            raise L.VpfError(f"RotaryAxes: {P} pairs do not fit an even head_dim of at most 1024 (got {head_dim})")
        if not (math.isfinite(self.base) and self.base > 0.0):
            raise L.VpfError(f"RotaryAxes: base must be positive and finite (got {base})")
        if layout not in ("half", "pair") or ladder not in ("axis", "joint"):
            raise L.VpfError(f"RotaryAxes: layout is 'half' or 'pair', ladder 'axis' or 'joint' (got {layout!r}, {ladder!r})")
        self.layout, self.ladder, self.pairs, self.layout_code = layout, ladder, P, int(layout == "pair")
        self._tables = {}

    def frequencies(self) -> torch.Tensor:
        """Radians per unit of position of every pair, fp64 on the host."""
        if self.ladder == "joint":
            return self.base ** (-torch.arange(self.pairs, dtype=torch.float64) / self.pairs)
        return torch.cat([self.base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in self.sections])

    def tables(self, device: torch.device):
        t = self._tables.get(device)
        if t is None:
            axis = torch.repeat_interleave(torch.arange(len(self.sections), dtype=torch.int32), torch.tensor(self.sections))
            t = self._tables[device] = ((self.frequencies() / (2.0 * math.pi)).to(device), axis.to(device))
        return t


_NONE3 = (0, 0, 0)


def _rotary_ready(t):
    """(tensor, strides).  The kernel takes any strides with a contiguous, pair-aligned last dimension; everything else is copied."""
    st = sb, sl, sh = _strides(t)
    if (sb | sl | sh) & 1 or t.stride(3) != 1 or t.data_ptr() % (2 * t.element_size()):
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides(t)
    return t, st


def _rotary_run(plan, pos, q, k, inverse):
    q, sq = _rotary_ready(q)
    B, Lt, Hq, dh = shape = q.shape
    dt, dev = q.dtype, q.device
    oq = torch.empty(shape, dtype=dt, device=dev)
    ok, Hk, kp, okp, sk, sok = None, 0, 0, 0, _NONE3, _NONE3
    if k is not None:
        k, sk = _rotary_ready(k)
        ok = torch.empty(k.shape, dtype=dt, device=dev)
        Hk, kp, okp, sok = k.shape[2], k.data_ptr(), ok.data_ptr(), _strides(ok)
    freq, axis = plan.tables(dev)
    L.launch("vpf_rotary_axes", _pack_rotary(
        B, Lt, Hq, Hk, dh, plan.pairs, len(plan.sections), plan.layout_code, _TYPE[dt], _POS[pos.dtype], inverse, 0, q.data_ptr(), kp, oq.data_ptr(), okp,
        *sq, *sk, *_strides(oq), *sok, pos.data_ptr(), pos.stride(0) if pos.dim() == 3 and pos.shape[0] > 1 else 0, freq.data_ptr(), axis.data_ptr()), dev)
    return oq, ok


class RotaryAxesFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, pos, q, k):
        ctx.plan, ctx.pos = plan, (pos.shape, pos.dtype, pos.device)
        _keep(ctx, pos)
        oq, ok = _rotary_run(plan, pos, q, k, 0)
        return oq if k is None else (oq, ok)

    @staticmethod
    def backward(ctx, gq, gk=None):
        _once("rotary_axes")
        ((pos,), _) = _kept(ctx, "rotary_axes", lambda: (ctx.pos,))
        return (None, None) + _rotary_run(ctx.plan, pos.contiguous(), gq, gk, 1)


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, plan: RotaryAxes):
    """Turn the channel pairs of q [B, L, heads, head_dim] and k [B, L, key heads, head_dim] (or None) by their tokens' positions.

    positions: [L, axes] or [B, L, axes] (or [1, L, axes]), integers or fp32 / fp64 coordinates; no gradient reaches them.  Angles are
    formed in fp64, so positions far into a stream keep their fraction of a turn.  fp32, fp16 and bf16, rounded once.
    Returns new contiguous tensors (q, k), or q alone where k is None."""
    qs = q.shape
    ks = qs if k is None else k.shape
    if len(qs) != 4 or len(ks) != 4 or ks[0] != qs[0] or ks[1] != qs[1] or ks[3] != qs[3]:
        raise L.VpfError(f"rotary_axes: q [B, L, heads, head_dim] and k of the same B, L and head_dim (got {tuple(q.shape)}, "
                         f"{None if k is None else tuple(k.shape)})")
    if qs[3] != plan.head_dim:
        raise L.VpfError(f"rotary_axes: head_dim {qs[3]}, the plan was built for {plan.head_dim}")
    if q.dtype not in _TYPE or (k is not None and k.dtype != q.dtype):
        raise L.VpfError(f"rotary_axes: q and k of one type out of fp32, fp16, bf16 (got {q.dtype}, {None if k is None else k.dtype})")
    ps = positions.shape
    if len(ps) not in (2, 3) or ps[-1] != len(plan.sections) or ps[-2] != qs[1] or (len(ps) == 3 and ps[0] != 1 and ps[0] != qs[0]):
        raise L.VpfError(f"rotary_axes: positions [L, axes] or [B, L, axes] = [({q.shape[0]},) {q.shape[1]}, {len(plan.sections)}] "
                         f"(got {tuple(positions.shape)})")
    if positions.dtype not in _POS:
        raise L.VpfError(f"rotary_axes: positions are int32, int64, fp32 or fp64 (got {positions.dtype})")
    if positions.requires_grad:
        raise L.VpfError("rotary_axes: no gradient with respect to the positions (detach them)")
    _same_device("rotary_axes", q, k, positions)
    pos = positions.contiguous()
    if _wants_grad(q, k):
        return RotaryAxesFn.apply(plan, pos, q, k)
    outs = _rotary_run(plan, pos, q, k, 0)
    return outs[0] if k is None else outs


# --------------------------------------------------------------------------- norms around a block, its gate and residual scale
def _norm_forward(cfg, x, y, gate, params, keep):
    """cfg: (kind, gate_mode, gate_rows, has_post, has_pre, alpha, beta, eps_post, eps_pre)."""
    kind, mode, gate_rows, has_post, has_pre, alpha, beta, eps_post, eps_pre = cfg
    D = x.shape[-1]
    rows = x.numel() // D
    h = torch.empty_like(x)
    n = torch.empty_like(y) if has_pre else None
    stats = torch.empty(4 * rows, dtype=F32, device=x.device) if keep else None
    L.launch("vpf_gated_norm_fwd", _pack_norm(
        rows, gate_rows, D, kind, _TYPE[x.dtype], _TYPE[y.dtype], mode, has_post, has_pre, 0, alpha, beta, eps_post, eps_pre, x.data_ptr(), y.data_ptr(),
        _ptr(gate), *map(_ptr, params), h.data_ptr(), _ptr(n), _ptr(stats), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), x.device)
    return h, n, stats


class GatedNormFn(torch.autograd.Function):
    """Gradients of parameters go back through autograd, divided by the internal gradient scale the forward ran under (ops.py)."""

    @staticmethod
    def forward(ctx, cfg, gate_is_param, x, y, gate, *params):
        h, n, stats = _norm_forward(cfg, x, y, gate, params, True)
        ctx.cfg, ctx.iscale, ctx.gate_is_param = cfg, ops._current_iscale(), gate_is_param
        ctx.y_type, ctx.gate_shape = y.dtype, None if gate is None else gate.shape
        _keep(ctx, x, y, gate, stats, *params)
        return (h, n) if n is not None else h

    @staticmethod
    def backward(ctx, dh, dn=None):
        _once("gated_norm_residual")
        kind, mode, gate_rows, has_post, has_pre, alpha, beta, eps_post, eps_pre = ctx.cfg
        shape, dev = dh.shape, dh.device
        D = shape[-1]
        ts, same = _kept(ctx, "gated_norm_residual", lambda: (
            (shape, dh.dtype, dev), (shape, ctx.y_type, dev), (ctx.gate_shape, ctx.y_type if mode == 2 else F32, dev),
            ((4 * (dh.numel() // D),), F32, dev)) + 4 * (((D,), F32, dev),))
        x, y, gate, stats, *params = ts if same else map(_dense, ts)
        need = ctx.needs_input_grad[1:]
        if x.numel() == 0:
            return (None, None, *(torch.zeros_like(t) if t is not None and n else None for t, n in zip((x, y, gate, *params), need[1:])))
        dh = dh.contiguous()
        dn = None if dn is None else dn.contiguous()
        dx = torch.empty_like(x) if need[1] else None
        dy = torch.empty_like(y) if need[2] else None
        dgate = torch.empty_like(gate) if need[3] else None
        flat = grads = None
        if True in need[4:]:
            flat = torch.empty(4, D, dtype=F32, device=dev)
            grads = [g if n else None for g, n in zip(flat.unbind(0), need[4:])]
        else:
            grads = [None] * 4
        args = [x.numel() // D, gate_rows, D, kind, _TYPE[x.dtype], _TYPE[y.dtype], mode, has_post, has_pre, 0, alpha, beta, eps_post, eps_pre,
                x.data_ptr(), y.data_ptr(), _ptr(gate), *map(_ptr, params), 0, 0, stats.data_ptr(), dh.data_ptr(), _ptr(dn), _ptr(dx), _ptr(dy), _ptr(dgate),
                *map(_ptr, grads), 0, 0]
        floats = L.scratch_floats("vpf_gated_norm_ws", _pack_norm(*args))
        ws = torch.empty(max(floats, 4), dtype=F32, device=dev)
        args[-2:] = ws.data_ptr(), ws.numel()
        L.launch("vpf_gated_norm_bwd", _pack_norm(*args), dev)
        inv = ctx.iscale.inv if ctx.iscale is not None else None
        if inv is not None:
            if flat is not None:
                flat.mul_(inv)
            if dgate is not None and ctx.gate_is_param:
                dgate.mul_(inv)
        return (None, None, dx, dy, dgate, *grads)


_NO_PARAMS = (None, None)


def _norm_params(what, wb, kind, eps, x):
    """(weight, bias) of one norm, each fp32 [D] or None, and its epsilon."""
    if isinstance(wb, torch.nn.Module):
        want = {"layer": torch.nn.LayerNorm, "rms": torch.nn.RMSNorm}[kind]
        if not isinstance(wb, want) or tuple(wb.normalized_shape) != (x.shape[-1],):
            raise L.VpfError(f"gated_norm_residual: {what}: a {want.__name__} over {x.shape[-1]} channels for kind {kind!r} (got {wb})")
        eps = torch.finfo(F32).eps if wb.eps is None else wb.eps        # (what torch's module uses for fp32, fp16 and bf16 inputs alike)
        wb = (wb.weight, getattr(wb, "bias", None))
    if len(wb) != 2:
        raise L.VpfError(f"gated_norm_residual: {what} is a norm module or (weight, bias)")
    for p in wb:
        if p is not None and (p.dtype is not F32 or p.dim() != 1 or p.shape[0] != x.shape[-1]):
            raise L.VpfError(f"gated_norm_residual: {what}: fp32 parameters of shape ({x.shape[-1]},) (got {p.dtype}, {tuple(p.shape)})")
    return tuple(None if p is None else p.contiguous() for p in wb), eps


def gated_norm_residual(x: torch.Tensor, y: torch.Tensor, gate: Optional[torch.Tensor] = None, *, post=None, pre=None, kind: str = "layer",
                        alpha: float = 1.0, beta: float = 1.0, eps: float = 1e-5):
    """h = alpha * x + beta * gate * post(y);  n = pre(h).  Returns (h, n); n is None where ``pre`` is None.

    x: the residual stream, y: the block's output, both [..., D] with D <= 8192; x is fp32, or x and y are of one type (fp16, bf16).  h has
    x's type, n has y's; n is taken from h before h is rounded.
    post / pre: (weight, bias) with fp32 [D] tensors or None entries, a LayerNorm / RMSNorm module, or None for no norm there.
    kind: "layer" or "rms" (biased variance, ``eps`` inside the root) for both norms; a module brings its own eps (None: that of fp32).
    gate: None, fp32 [D], one fp32 row of D per sample (x [B, ..., D]: gate [B, 1, .., D]), or one of x's shape and y's type."""
    shape = x.shape
    if len(shape) < 1 or shape != y.shape or not 1 <= shape[-1] <= 8192:
        raise L.VpfError(f"gated_norm_residual: x and y of one shape [..., D], 1 <= D <= 8192 (got {tuple(x.shape)}, {tuple(y.shape)})")
    if x.dtype not in _TYPE or y.dtype not in _TYPE or (x.dtype != F32 and x.dtype != y.dtype):
        raise L.VpfError(f"gated_norm_residual: x is fp32, or x and y are both fp16 or both bf16 (got {x.dtype}, {y.dtype})")
    if kind not in ("layer", "rms"):
        raise L.VpfError(f"gated_norm_residual: kind is 'layer' or 'rms' (got {kind!r})")
    D = shape[-1]
    rows = x.numel() // D
    if rows >= 1 << 31:
        raise L.VpfError(f"gated_norm_residual: {rows} rows; at most 2^31 - 1")
    mode, gate_rows = 0, 1
    if gate is not None:
        gs = gate.shape
        if gs == shape and gate.dtype == y.dtype:
            mode = 2
        elif len(gs) == 1 and gs[0] == D:
            mode, gate_rows = 1, max(rows, 1)
        elif len(shape) >= 2 and tuple(gs) == (shape[0],) + (1,) * (len(shape) - 2) + (D,):
            mode, gate_rows = 1, max(rows // max(shape[0], 1), 1)
        else:
            raise L.VpfError(f"gated_norm_residual: gate [D], one row per sample or x's shape in y's type (got {tuple(gate.shape)}, {gate.dtype})")
        if mode == 1 and gate.dtype != F32:
            raise L.VpfError(f"gated_norm_residual: a gate that is shared by rows is fp32 (got {gate.dtype})")
    wb_post, eps_post = (_NO_PARAMS, eps) if post is None else _norm_params("post", post, kind, eps, x)
    wb_pre, eps_pre = (_NO_PARAMS, eps) if pre is None else _norm_params("pre", pre, kind, eps, x)
    params = wb_post + wb_pre
    _same_device("gated_norm_residual", x, y, gate, *params)
    cfg = (int(kind == "rms"), mode, gate_rows, int(post is not None), int(pre is not None), float(alpha), float(beta), float(eps_post),
           float(eps_pre))
    gate_is_param = isinstance(gate, torch.nn.Parameter)         # (before a copy of it takes its place)
    x, y, gate = x.contiguous(), y.contiguous(), None if gate is None else gate.contiguous()
    if not _wants_grad(x, y, gate, *params):
        return _norm_forward(cfg, x, y, gate, params, False)[:2]
    out = GatedNormFn.apply(cfg, gate_is_param, x, y, gate, *params)
    return out if pre is not None else (out, None)


# --------------------------------------------------------------------------- attention inside a sliding window
def _attn_ready(t: torch.Tensor, shared: int = 0):
    """(tensor, its batch, token and head stride).  16-byte rows: a contiguous last dimension, an aligned base, strides that are multiples of 8
    elements, those of tokens below 2^23 and, for a backward pass over ``shared`` heads of a key head, those heads together below 2^29;
    everything else is copied."""
    st = sb, sl, sh = _strides(t)
    if (sb | sl | sh) & 7 or sl >= 1 << 23 or shared * sh >= 1 << 29 or t.stride(3) != 1 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides(t)
    return t, st


def _attn_launch(name, cfg, q, k, v, out, pad, lens, lse, lo, grads, strides, backward):
    """cfg: (left, right, sinks, scale); grads: (dout, dq, dk, dv); strides: of q, k, v, out, dout, dq, dk, dv in one tuple.  Scratch is asked for,
    allocated and handed over; it stays alive until the launch is issued (the allocator orders its reuse by stream)."""
    left, right, sinks, scale = cfg
    B, Lq, Hq, dh = q.shape
    _, Lkv, Hk, _ = k.shape
    dev = q.device
    head = (B, Lq, Lkv, Hq, Hk, dh, left, right, sinks, _TYPE[q.dtype], scale, int(lens is not None and lens.dtype is torch.int64),
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(pad), _ptr(lens), out.data_ptr(), _ptr(lse), _ptr(lo), *grads)
    packed = _pack_attn(*head, 0, 0, *strides)
    n = L.scratch_floats("vpf_window_attn_ws", packed, backward)
    if n:
        ws = torch.empty(n, dtype=F32, device=dev)
        packed = _pack_attn(*head, ws.data_ptr(), n, *strides)
    L.launch(name, packed, dev)


_NO_GRADS, _NO_STRIDES = (0,) * 4, (0,) * 12


def _attn_forward(cfg, q, k, v, pad, lens, strides, keep):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = lo = None
    if keep:
        lse = torch.empty(q.numel() // q.shape[3], dtype=F32, device=q.device)
        lo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _attn_launch("vpf_window_attn_fwd", cfg, q, k, v, out, pad, lens, lse, lo, _NO_GRADS, strides + _strides(out) + _NO_STRIDES, 0)
    return out, lse, lo


class WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, q, k, v, pad, lens):
        (q, sq), (k, sk), (v, sv) = _attn_ready(q, q.shape[2] // k.shape[2]), _attn_ready(k), _attn_ready(v)
        ctx.cfg, ctx.strides, ctx.keys = cfg, sq + sk + sv, k.shape
        out, lse, lo = _attn_forward(cfg, q, k, v, pad, lens, ctx.strides, True)
        _keep(ctx, q, k, v, out, lse, lo, pad, lens)
        ctx.qkv, ctx.lens64 = (q.stride(), k.stride(), v.stride()), lens is not None and lens.dtype is torch.int64
        return out

    @staticmethod
    def backward(ctx, dout):
        _once("window_attention")
        B, Lq, Hq, dh = rows = dout.shape
        keys, dt, dev = ctx.keys, dout.dtype, dout.device
        ts, same = _kept(ctx, "window_attention", lambda: (
            (rows, dt, dev), (keys, dt, dev), (keys, dt, dev), (rows, dt, dev), ((B * Lq * Hq,), F32, dev), (rows, dt, dev),
            ((B, keys[1]), torch.uint8, dev), ((B,), torch.int64 if ctx.lens64 else torch.int32, dev)))
        q, k, v, out, lse, lo, pad, lens = ts
        g = Hq // keys[2]
        if same and ctx.qkv == (q.stride(), k.stride(), v.stride()):
            strides, so = ctx.strides, _strides(out)
        else:
            lse, lo, pad, lens = map(_dense, (lse, lo, pad, lens))
            lo = lo.clone() if lo.data_ptr() & 15 else lo
            (q, sq), (k, sk), (v, sv), (out, so) = _attn_ready(q, g), _attn_ready(k), _attn_ready(v), _attn_ready(out)
            strides = sq + sk + sv
        dout, sd = _attn_ready(dout, g)
        dq, dk, dv = (torch.empty(shape, dtype=dt, device=dev) for shape in (rows, keys, keys))
        sdq, sdk = _strides(dq), _strides(dk)
        _attn_launch("vpf_window_attn_bwd", ctx.cfg, q, k, v, out, pad, lens, lse, lo, (dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()),
                     strides + so + sd + sdq + sdk + sdk, 1)
        return None, dq, dk, dv, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Tuple[Optional[int], Optional[int]] = (None, None), *,
                     sinks: int = 0, scale: Optional[float] = None, pad_mask: Optional[torch.Tensor] = None,
                     kv_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T over the visible keys) v for q [B, Lq, heads, head_dim] and k, v [B, Lkv, key heads, head_dim]; fp16 or bf16.

    window = (left, right): query at position p sees keys p - left .. p + right (None: open on that side; (n, 0) is causal), and of the first
    ``sinks`` keys those up to p + right, however far behind they are.
    With n keys in use the last query stands at the last of them: query i at position n - Lq + i.  n is Lkv, or kv_lens[b] (int32 / int64 [B],
    on the device, read by the kernels: a captured graph follows it; clamped to 0 .. Lkv): a preallocated cache that is filled to different
    lengths.
    pad_mask: bool [B, Lkv], True = this key is padding (as the ``pad_mask`` of the framework's encoders); it moves no positions.
    Keys that no query sees may hold anything, also NaN; a value that is not finite in a key that some query sees reaches the queries around it, as
    0 * NaN does in the product of weights and values.  A query that sees nothing gets zeros; it and its gradient may hold anything and reach
    nothing.  (In the gradients of keys and values, what is not finite in a query that sees some key, or in its gradient, reaches the keys around.)
    Key heads are shared by heads / key heads consecutive query heads.  head_dim: a multiple of 8 up to 128; scale defaults to head_dim ** -0.5.
    Returns a new contiguous [B, Lq, heads, head_dim]; gradients for q, k and v (until then a call keeps the result twice: what its rounding took
    away, and 4 bytes a query and head).  There is no dropout on the weights here."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or ks[0] != qs[0] or ks[3] != qs[3] or ks[2] < 1 or qs[2] < 1 or qs[2] % ks[2]:
        raise L.VpfError(f"window_attention: q [B, Lq, heads, head_dim], k and v [B, Lkv, key heads, head_dim], key heads dividing heads (got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    dt = q.dtype
    if (dt is not torch.bfloat16 and dt is not torch.float16) or k.dtype is not dt or v.dtype is not dt:
        raise L.VpfError(f"window_attention: q, k and v all fp16 or all bf16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    B, Lq, Hq, dh = qs
    Lkv, g = ks[1], Hq // ks[2]
    if dh % 8 or not 8 <= dh <= 128:
        raise L.VpfError(f"window_attention: head_dim is a multiple of 8 up to 128 (got {dh})")
    if Lq + Lkv >= 1 << 30 or Lq * g * g >= 1 << 31:
        raise L.VpfError(f"window_attention: Lq {Lq}, Lkv {Lkv}, {g} heads per key head: beyond the kernels' index range")
    left, right = window
    for side in (left, right):
        if side is not None and (isinstance(side, bool) or not isinstance(side, int) or side < 0):
            raise L.VpfError(f"window_attention: a side of the window is None or a whole number >= 0 (got {window})")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise L.VpfError(f"window_attention: sinks is a whole number >= 0 (got {sinks})")
    scale = dh ** -0.5 if scale is None else float(scale)
    if not (0.0 < scale < math.inf):
        raise L.VpfError(f"window_attention: scale must be positive and finite (got {scale})")
    if pad_mask is not None and (pad_mask.dtype != torch.bool or tuple(pad_mask.shape) != (B, Lkv)):
        raise L.VpfError(f"window_attention: pad_mask is bool [B, Lkv] = {(B, Lkv)} (got {pad_mask.dtype}, {tuple(pad_mask.shape)})")
    if kv_lens is not None and (kv_lens.dtype not in (torch.int32, torch.int64) or tuple(kv_lens.shape) != (B,)):
        raise L.VpfError(f"window_attention: kv_lens is int32 or int64 [B] = {(B,)} (got {kv_lens.dtype}, {tuple(kv_lens.shape)})")
    _same_device("window_attention", q, k, v, pad_mask, kv_lens)
    top = (1 << 30) - 1
    cfg = (-1 if left is None else min(left, top), -1 if right is None else min(right, top), min(sinks, top), scale)
    pad = None if pad_mask is None else pad_mask.contiguous().view(torch.uint8)
    lens = None if kv_lens is None else kv_lens.contiguous()
    if not _wants_grad(q, k, v):
        (q, sq), (k, sk), (v, sv) = _attn_ready(q), _attn_ready(k), _attn_ready(v)
        return _attn_forward(cfg, q, k, v, pad, lens, sq + sk + sv, False)[0]
    if lens is not None and lens.dtype is torch.int64:           # (64-bit counters go on counting behind the call: backward has its own)
        lens = lens.clone()
    return WindowAttentionFn.apply(cfg, q, k, v, pad, lens)
