"""GPU parity of the transformer-block operators (vipformer_amd/ops_block.py) against plain 64-bit implementations.

Tolerances are elementwise: half a step of the output's type (finfo.eps / 2 relative: the one rounding at the end) plus a counted number of
fp32 roundings, each at most 2^-24 of the sum of the magnitudes that meet in the element."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U24 = 2.0 ** -24
TYPES = {"f32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, ref, slack, what):
    """|got - ref| <= half a step of got's type at ref (and of its smallest number) + slack."""
    fi = torch.finfo(got.dtype)
    assert got.shape == ref.shape, what
    tol = (fi.eps / 2) * (ref.abs() + slack) + fi.smallest_normal * fi.eps / 2 + slack
    bad = (got.double() - ref).abs() - tol
    assert torch.isfinite(got.double()).all() and float(bad.max()) <= 0.0, \
        f"{what}: {int((bad > 0).sum())} of {bad.numel()} outside, worst {float((got.double() - ref).abs().max()):.3e} against {float(tol.flatten()[bad.flatten().argmax()]):.3e}"


# ------------------------------------------------------------------------------------------ rotary positions with several axes
def rotary_ref(x, pos, plan, sign=1.0):
    """(rotated, sum of the magnitudes that meet) in 64 bits."""
    f = plan.frequencies().cuda()
    axis = torch.repeat_interleave(torch.arange(len(plan.sections), device="cuda"), torch.tensor(plan.sections, device="cuda"))
    t = (pos if pos.dim() == 3 else pos[None]).double()[..., axis] * f * sign
    c, s = t.cos()[:, :, None], t.sin()[:, :, None]
    d, P = x.detach().double(), plan.pairs
    if plan.layout == "half":
        a, b, rest = d[..., :P], d[..., P:2 * P], d[..., 2 * P:]
        join = lambda u, v: torch.cat([u, v, rest], -1)
    else:
        a, b, rest = d[..., 0:2 * P:2], d[..., 1:2 * P:2], d[..., 2 * P:]
        join = lambda u, v: torch.cat([torch.stack([u, v], -1).flatten(-2), rest], -1)
    mag = a.abs() + b.abs()
    out = join(a * c - b * s, b * c + a * s)
    size = join(mag, mag)
    size[..., 2 * P:] = 0.0
    return out, size


# fp32 roundings of one element: the fraction of a turn (2^-25 turns are 3.2 units of 2^-24 rad), sincospi within 2 of its last places (4
# units at most), two products, one sum: 10
ROT = 10 * U24


@pytest.mark.parametrize("layout", ["half", "pair"])
@pytest.mark.parametrize("dtype", ["f32", "fp16", "bf16"])
@pytest.mark.parametrize("B,L,Hq,Hk,dh,sections,ladder", [
    (1, 1, 1, 1, 2, (1,), "axis"), (2, 96, 4, 4, 64, (16, 16), "axis"), (3, 145, 6, 2, 64, (8, 12, 12), "axis"),
    (1, 1025, 16, 4, 128, (22, 21, 21), "joint"), (5, 33, 3, 1, 40, (7, 7, 6), "axis"), (2, 17, 2, 2, 80, (5, 0, 3), "joint"),
    (1, 7, 70, 1, 1024, (512,), "axis"), (2, 0, 2, 2, 64, (32,), "axis"), (40, 3, 2, 1, 96, (1, 2, 3, 4, 5, 6, 7, 8), "axis")])
def test_rotary_forward_and_gradient(B, L, Hq, Hk, dh, sections, ladder, dtype, layout):
    from vipformer_amd.ops_block import RotaryAxes, rotary_axes
    g, dt = gen(L + dh), TYPES[dtype]
    plan = RotaryAxes(sections, dh, layout=layout, ladder=ladder)
    q, k = randn(g, B, L, Hq, dh, dtype=dt).requires_grad_(), randn(g, B, L, Hk, dh, dtype=dt).requires_grad_()
    pos = torch.rand(B, L, len(sections), generator=g, device="cuda") * 100 - 20
    oq, ok = rotary_axes(q, k, pos, plan)
    gq, gk = randn(g, *q.shape, dtype=dt), randn(g, *k.shape, dtype=dt)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    for got, x, sign, what in ((oq, q, 1.0, "q"), (ok, k, 1.0, "k"), (dq, gq, -1.0, "dq"), (dk, gk, -1.0, "dk")):
        if L == 0:
            assert got.shape == x.shape
            continue
        ref, size = rotary_ref(x, pos, plan, sign)
        close(got.detach(), ref, ROT * size, what)


@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_rotary_positions_types_sharing_and_far_positions(pdtype):
    from vipformer_amd.ops_block import RotaryAxes, rotary_axes
    g = gen(3)
    plan = RotaryAxes((10, 11, 11), 64)
    q, k = randn(g, 2, 50, 4, 64), randn(g, 2, 50, 2, 64)
    pos = torch.randint(0, 64, (50, 3), generator=g, device="cuda")
    pos[:, 0] += 2 ** 24 - 30 if pdtype == torch.float32 else 10 ** 9          # fp32 holds whole numbers up to 2^24
    pos = pos.to(pdtype)
    for p in (pos, pos[None], pos[None].expand(2, 50, 3)):
        oq, ok = rotary_axes(q, k, p, plan)
        for got, x in ((oq, q), (ok, k)):
            ref, size = rotary_ref(x, p, plan)
            # the reference's own angle in 64 bits: 10^9 rad at 2^-53 is 1e-7 rad, two more units
            close(got, ref, (ROT + 2 * U24) * size, "far")


@pytest.mark.parametrize("dtype", ["f32", "fp16"])
@pytest.mark.parametrize("layout", ["half", "pair"])
def test_rotary_strides_slices_and_single_tensor(dtype, layout):
    """Slices of one projection's output, head-first tensors, odd base offsets, a transposed last dimension, q alone."""
    from vipformer_amd.ops_block import RotaryAxes, rotary_axes
    g, dt = gen(9), TYPES[dtype]
    B, L, H, dh = 2, 37, 3, 48
    plan = RotaryAxes((12, 12), dh, layout=layout)
    pos = torch.randint(0, 9, (L, 2), generator=g, device="cuda")
    qkv = randn(g, B, L, 3 * H * dh, dtype=dt)
    q, k = qkv.view(B, L, 3, H, dh)[:, :, 0], qkv.view(B, L, 3, H, dh)[:, :, 1]
    heads_first = randn(g, B, H, L, dh, dtype=dt).transpose(1, 2)
    flat = randn(g, B * L * H * dh + 1, dtype=dt)[1:].view(B, L, H, dh)
    turned = randn(g, B, L, dh, H, dtype=dt).transpose(2, 3)
    rows = randn(g, B, L, H, dh + 1, dtype=dt)[..., :dh]                        # an odd row stride
    before = qkv.clone()
    for a, b in ((q, k), (heads_first, flat), (turned, rows), (rows, None)):
        out = rotary_axes(a, b, pos, plan)
        outs = (out,) if b is None else out
        for got, x in zip(outs, (a, b)):
            ref, size = rotary_ref(x, pos, plan)
            close(got, ref, ROT * size, "strided")
    assert torch.equal(qkv, before)


# ------------------------------------------------------------------------------------------ norms around a block, gate and residual scale
def norm_ref(x, y, gate, post, pre, kind, alpha, beta, eps, dh, dn):
    """Outputs and gradients in 64 bits with, for each, the sum of the magnitudes that meet in it."""
    d = lambda t: None if t is None else t.detach().double()
    x, y, gate, dh, dn = d(x), d(y), d(gate), d(dh), d(dn)
    layer = kind == "layer"
    D = x.shape[-1]

    def stats(z):
        m = z.mean(-1, keepdim=True) if layer else torch.zeros_like(z[..., :1])
        r = 1.0 / torch.sqrt(((z - m) ** 2).mean(-1, keepdim=True) + eps)
        return m, r

    def affine(wb):
        w, b = (d(wb[0]), d(wb[1])) if wb is not None else (None, None)
        return (torch.ones(D, device="cuda", dtype=torch.float64) if w is None else w), (torch.zeros(D, device="cuda", dtype=torch.float64) if b is None else b)

    def back(e, zh, r):
        out = e - zh * (e * zh).mean(-1, keepdim=True) - (e.mean(-1, keepdim=True) if layer else 0.0)
        size = e.abs() + zh.abs() * (e * zh).abs().mean(-1, keepdim=True) + (e.abs().mean(-1, keepdim=True) if layer else 0.0)
        return out * r, size * r

    gt = torch.ones_like(x) if gate is None else gate.expand_as(x)
    wp, bp = affine(post)
    yh, ry = y, torch.ones_like(y[..., :1])
    ysize = y.abs()
    if post is not None:
        my, ry = stats(y)
        yh = (y - my) * ry
        ysize = (y.abs() + y.abs().mean(-1, keepdim=True)) * ry
    u, usize = yh * wp + bp, ysize * wp.abs() + bp.abs()
    h = alpha * x + beta * gt * u
    hsize = abs(alpha) * x.abs() + abs(beta) * gt.abs() * usize
    out = {"h": (h, hsize)}
    dH, dHsize = dh, dh.abs()
    if pre is not None:
        wn, bn = affine(pre)
        mh, rh = stats(h)
        hh = (h - mh) * rh
        # an error of h reaches every channel of its row through the statistics
        rel = hsize + hsize.mean(-1, keepdim=True) + hh.abs() * (hsize * hh.abs()).mean(-1, keepdim=True)
        hhsize = rel * rh
        out["n"] = (hh * wn + bn, hhsize * wn.abs() + bn.abs())
        e = dn * wn
        part, psize = back(e, hh, rh)
        # hh enters the gradient twice and rh once: their errors on top
        grown = rh * (hhsize * (e * hh).abs().mean(-1, keepdim=True) + hh.abs() * (e.abs() * hhsize).mean(-1, keepdim=True))
        grown = grown + psize * (hhsize * hh.abs()).mean(-1, keepdim=True)
        dH, dHsize = dh + part, dh.abs() + psize + grown
        out["dw_pre"] = ((dn * hh).flatten(0, -2).sum(0), (dn.abs() * (hh.abs() + hhsize)).flatten(0, -2).sum(0))
        out["db_pre"] = (dn.flatten(0, -2).sum(0), dn.abs().flatten(0, -2).sum(0))
    out["dx"] = (alpha * dH, abs(alpha) * dHsize)
    if gate is not None:
        full, fsize = beta * dH * u, abs(beta) * (dHsize * u.abs() + dH.abs() * usize)
        shape = gate.shape
        if gate.shape == x.shape:
            out["dgate"] = (full, fsize)
        elif gate.dim() == 1:
            out["dgate"] = (full.flatten(0, -2).sum(0), fsize.flatten(0, -2).sum(0))
        else:
            out["dgate"] = (full.reshape(shape[0], -1, D).sum(1).view(shape), fsize.reshape(shape[0], -1, D).sum(1).view(shape))
    f, fs = beta * gt * dH, abs(beta) * gt.abs() * dHsize
    if post is not None:
        out["dw_post"] = ((f * yh).flatten(0, -2).sum(0), (fs * yh.abs() + f.abs() * ysize).flatten(0, -2).sum(0))
        out["db_post"] = (f.flatten(0, -2).sum(0), fs.flatten(0, -2).sum(0))
        dy, dysize = back(f * wp, yh, ry)
        _, more = back(fs * wp.abs(), yh, ry)
        fw = (f * wp).abs()
        grown = ry * (ysize * (fw * yh.abs()).mean(-1, keepdim=True) + yh.abs() * (fw * ysize).mean(-1, keepdim=True))
        grown = grown + dysize * (ysize * yh.abs()).mean(-1, keepdim=True)
        out["dy"] = (dy, dysize + more + grown)
    else:
        out["dy"] = (f, fs)
    return out


# fp32 roundings on the longest path of one element: 8 products and sums in a thread, 10 levels of the joining tree, twice (mean, variance),
# for two norms, root, scale, gate and residual: under 64; forward values enter the gradient once more: under 128
FWD_N, BWD_N = 64 * U24, 128 * U24


def norm_case(shape, kind, gate, x, y, post, pre, alpha=0.9, beta=0.75, eps=1e-5, seed=0, bias=None):
    from vipformer_amd.ops_block import gated_norm_residual
    g, tx, ty = gen(seed + shape[-1]), TYPES[x], TYPES[y]
    D = shape[-1]
    X, Y = randn(g, *shape, dtype=tx, scale=2.0).requires_grad_(), (randn(g, *shape, scale=0.7) + 0.3).to(ty).requires_grad_()
    aff = lambda: (1.0 + randn(g, D, scale=0.2)).requires_grad_()
    bias = (kind == "layer") if bias is None else bias
    P = (aff(), aff() if bias else None) if post else None
    N = (aff(), aff() if bias else None) if pre else None
    gshape = {"none": None, "channel": (D,), "sample": (shape[0],) + (1,) * (len(shape) - 2) + (D,), "token": shape}[gate]
    G = None if gshape is None else randn(g, *gshape, dtype=ty if gate == "token" else torch.float32, scale=0.5).requires_grad_()
    h, n = gated_norm_residual(X, Y, gate=G, post=P, pre=N, kind=kind, alpha=alpha, beta=beta, eps=eps)
    dh, dn = randn(g, *shape, dtype=tx), (randn(g, *shape, dtype=ty) if pre else None)
    names = {"dx": X, "dy": Y, "dgate": G, "dw_post": P and P[0], "db_post": P and P[1], "dw_pre": N and N[0], "db_pre": N and N[1]}
    names = {k: v for k, v in names.items() if v is not None}
    outs, douts = ([h], [dh]) if n is None else ([h, n], [dh, dn])
    grads = torch.autograd.grad(outs, list(names.values()), douts)
    ref = norm_ref(X, Y, G, P, N, kind, alpha, beta, eps, dh, dn)
    assert h.dtype == tx and (n is None or n.dtype == ty)
    close(h.detach(), *(ref["h"][0], FWD_N * ref["h"][1]), "h")
    if n is not None:
        close(n.detach(), ref["n"][0], FWD_N * ref["n"][1], "n")
    for name, got in zip(names, grads):
        assert got.dtype == names[name].dtype
        close(got, ref[name][0], BWD_N * ref[name][1], name)
    with torch.no_grad():
        h2, n2 = gated_norm_residual(X, Y, gate=G, post=P, pre=N, kind=kind, alpha=alpha, beta=beta, eps=eps)
    assert torch.equal(h2, h) and (n is None or torch.equal(n2, n))


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("x,y", [("f32", "fp16"), ("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("shape", [(2, 70, 256), (3, 37, 1001), (1, 1, 40)])
def test_gated_norm_forward_and_gradients(shape, x, y, gate, kind):
    norm_case(shape, kind, gate, x, y, True, True)


@pytest.mark.parametrize("x,y", [("f32", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("D", [8, 13, 128, 136, 384, 520, 1024, 1032, 2048, 2055, 4096, 4104, 8185, 8192])
def test_gated_norm_widths(D, x, y):
    norm_case((2, 9, D), "layer", "sample", x, y, True, True)


@pytest.mark.parametrize("post,pre", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_gated_norm_with_one_norm_or_none(post, pre, gate):
    norm_case((4, 65, 264), "layer", gate, "f32", "fp16", post, pre)
    norm_case((4, 65, 264), "rms", gate, "fp16", "fp16", post, pre, bias=True)


@pytest.mark.parametrize("shape", [(5, 1, 64), (700, 2, 64), (257, 96), (2, 3, 4, 5, 72), (4096, 3, 16), (33, 1000, 256)])
def test_gated_norm_many_samples_and_ranks(shape):
    norm_case(shape, "layer", "sample", "f32", "fp16", True, True)


@pytest.mark.parametrize("L", [1, 2, 7, 31, 33])
def test_gated_norm_gates_of_few_rows(L):
    """Gate rows that serve fewer rows than a workgroup holds (their gradient goes through scratch row by row), in both paths of the row kernels."""
    norm_case((301, L, 64), "layer", "sample", "f32", "fp16", True, True)
    norm_case((40, L, 257), "rms", "sample", "bf16", "bf16", True, True)
    norm_case((5, L, 2048), "layer", "sample", "f32", "f32", False, True)


def test_gated_norm_more_samples_than_a_grid():
    """300 000 gate rows of 1 000 channels: the fold of their gradients walks over more items than a launch has workgroups."""
    from vipformer_amd.ops_block import gated_norm_residual
    g = gen(14)
    B, D = 300000, 1000
    x, y = randn(g, B, 1, D).requires_grad_(), randn(g, B, 1, D, dtype=torch.float16)
    gate = randn(g, B, 1, D).requires_grad_()
    h, _ = gated_norm_residual(x, y, gate=gate, post=(None, None), kind="rms")
    dh = randn(g, B, 1, D)
    (dg,) = torch.autograd.grad(h, gate, dh)
    rows = torch.randint(0, B, (500,), generator=g, device="cuda")
    rows[0], rows[1] = 0, B - 1
    ref = norm_ref(x[rows], y[rows], gate[rows], (None, None), None, "rms", 1.0, 1.0, 1e-5, dh[rows], None)
    close(dg[rows], ref["dgate"][0], BWD_N * ref["dgate"][1], "dgate")


def test_gated_norm_modules_identity_and_unused_outputs():
    from vipformer_amd.ops_block import gated_norm_residual
    g = gen(11)
    x, y = randn(g, 2, 50, 256).requires_grad_(), randn(g, 2, 50, 256, dtype=torch.float16)
    ln, rms = torch.nn.LayerNorm(256, eps=1e-3).cuda(), torch.nn.RMSNorm(256).cuda()
    h, n = gated_norm_residual(x, y, post=ln, pre=torch.nn.LayerNorm(256, elementwise_affine=False).cuda())
    ref = norm_ref(x, y, None, (ln.weight, ln.bias), (None, None), "layer", 1.0, 1.0, 1e-3, h, y)
    close(h.detach(), ref["h"][0], FWD_N * ref["h"][1], "module eps")
    gated_norm_residual(x, y, post=rms, pre=rms, kind="rms")
    # the same parameters in both places: their gradient is the sum of the two
    w = (1.0 + randn(g, 256, scale=0.1)).requires_grad_()
    h, n = gated_norm_residual(x, y, post=(w, None), pre=(w, None), kind="rms", eps=1e-5)
    dh, dn = randn(g, *h.shape), randn(g, *n.shape, dtype=torch.float16)
    (dw,) = torch.autograd.grad((h, n), (w,), (dh, dn))
    ref = norm_ref(x, y, None, (w, None), (w, None), "rms", 1.0, 1.0, 1e-5, dh, dn)
    close(dw, ref["dw_post"][0] + ref["dw_pre"][0], BWD_N * (ref["dw_post"][1] + ref["dw_pre"][1]), "shared weight")
    # a loss that uses one output only
    h, n = gated_norm_residual(x, y, post=(w, None), pre=(w, None), kind="rms", eps=1e-5)
    (dx,) = torch.autograd.grad(h, (x,), dh)
    assert torch.equal(dx, dh)


def test_gated_norm_is_bitwise_reproducible():
    from vipformer_amd.ops_block import gated_norm_residual
    g = gen(12)
    x, y = randn(g, 64, 128, 256).requires_grad_(), randn(g, 64, 128, 256, dtype=torch.float16).requires_grad_()
    gate, w, b = randn(g, 256).requires_grad_(), randn(g, 256).requires_grad_(), randn(g, 256).requires_grad_()
    dh, dn = randn(g, 64, 128, 256), randn(g, 64, 128, 256, dtype=torch.float16)
    runs = []
    for _ in range(3):
        h, n = gated_norm_residual(x, y, gate=gate, post=(w, b), pre=(w, b))
        runs.append([h.detach(), n.detach(), *torch.autograd.grad((h, n), (x, y, gate, w, b), (dh, dn))])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_gated_norm_under_internal_grad_scale():
    """Parameters get their gradient in the loss's own units; the gradient that flows on keeps the scale."""
    from vipformer_amd import ops
    from vipformer_amd.ops_block import gated_norm_residual
    g = gen(13)
    x, y = randn(g, 4, 16, 64).requires_grad_(), randn(g, 4, 16, 64, dtype=torch.float16).requires_grad_()
    gate, w = torch.nn.Parameter(randn(g, 64)), torch.nn.Parameter(1.0 + randn(g, 64, scale=0.1))
    dh = randn(g, 4, 16, 64, scale=1e-4)

    def grads(on):
        with ops.internal_grad_scale(on) as holder:
            h, _ = gated_norm_residual(x, y, gate=gate, post=(w, None))
            out = ops.ScaleGradFn.apply(h, holder) if on else h
        return torch.autograd.grad(out, (x, gate, w), dh)

    plain, scaled = grads(False), grads(True)
    s = float(scaled[0].abs().max() / plain[0].abs().max())
    assert s > 1024 and math.log2(s) == int(math.log2(s))
    assert torch.equal(scaled[1], plain[1]) and torch.equal(scaled[2], plain[2])


# ------------------------------------------------------------------------------------------ attention inside a sliding window
def seen_mask(B, Lq, Lkv, window, sinks, pad, lens):
    """[B, Lq, Lkv] True = visible, straight from the definition."""
    left, right = ((1 << 40) if s is None else s for s in window)
    n = torch.full((B,), Lkv) if lens is None else lens.cpu().long().clamp(0, Lkv)
    p = (n[:, None] - Lq + torch.arange(Lq))[:, :, None]
    j = torch.arange(Lkv)[None, None, :]
    m = (j < n[:, None, None]) & (j <= p + right) & ((j >= p - left) | (j < sinks))
    return m.cuda() if pad is None else m.cuda() & ~pad[:, None, :]


def attention_ref(q, k, v, mask, scale, dout=None):
    """out (and dq, dk, dv) in 64 bits, with the magnitudes their roundings scale with (root of the sums of squares)."""
    B, Lq, Hq, dh = q.shape
    Hk = k.shape[2]
    g = Hq // Hk
    Q, K, V = (t.detach().double().transpose(1, 2) for t in (q, k, v))                 # [B, H, L, dh]
    K, V = K.repeat_interleave(g, 1), V.repeat_interleave(g, 1)
    M = mask[:, None]
    K, V = (torch.where(mask.any(1)[:, None, :, None], t, 0.0) for t in (K, V))        # keys nobody sees hold anything
    S = (Q @ K.transpose(-1, -2) * scale).masked_fill(~M, -math.inf)
    P = torch.nan_to_num(torch.softmax(S, -1), nan=0.0) * M
    res = {"out": (P @ V, ((P ** 2) @ (V ** 2)).sqrt())}
    if dout is not None:
        G = dout.double().transpose(1, 2)
        dP = G @ V.transpose(-1, -2)
        delta = (G * res["out"][0]).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        # an element of dS carries: its own rounding, P's error through dP - delta, and delta's (out is rounded: half a step of every G out)
        ddelta = ((G * res["out"][0]) ** 2).sum(-1, keepdim=True).sqrt()
        e = dS.abs() + P * ddelta
        group = lambda t: t.reshape(B, Hk, g, *t.shape[2:]).sum(2)
        res["dq"] = (scale * dS @ K, scale * (e ** 2 @ K ** 2).sqrt())
        res["dk"] = (group(scale * dS.transpose(-1, -2) @ Q), scale * group((e ** 2).transpose(-1, -2) @ Q ** 2).sqrt())
        res["dv"] = (group(P.transpose(-1, -2) @ G), group((P ** 2).transpose(-1, -2) @ G ** 2).sqrt())
    return {n: (a.transpose(1, 2), b.transpose(1, 2)) for n, (a, b) in res.items()}


def attention_close(got, ref, size, what):
    """Elementwise: half a step for the output's rounding, and for the rounding of the weights (P, dS) to the same type, independent from element
    to element and at most half a step each: the root of the sum of squares times half a step is their standard deviation's bound, 8 of
    them the limit for any of up to 10^7 elements; fp32 sums of up to 2^15 terms add less than 2^-12 of it.  fp16 weights below 2^-14 are
    spaced 2^-24: half of that for each of the terms, relative to operands of size 1."""
    fi = torch.finfo(got.dtype)
    half = fi.eps / 2
    tol = half * ref.abs() + 8 * half * size + 1e-6
    if got.dtype == torch.float16:
        tol = tol + 8 * 2.0 ** -25 * math.sqrt(ref.shape[1]) * 4
    d = (got.double() - ref).abs()
    assert got.shape == ref.shape and torch.isfinite(got.double()).all(), what
    bad = d - tol
    assert d.numel() == 0 or float(bad.max()) <= 0.0, f"{what}: {int((bad > 0).sum())} of {d.numel()} outside, worst {float(d.max()):.3e}"


def attention_case(B, Lq, Lkv, Hq, Hk, dh, window, sinks, dtype, pad=None, lens=None, train=True, scale=None, seed=0, garbage=True, views=False):
    from vipformer_amd.ops_block import window_attention
    g, dt = gen(seed + Lq + 7 * Lkv + dh), TYPES[dtype]
    if views:
        buf = randn(g, B, Lq, 3, Hq, dh, dtype=dt)
        q, k, v = (buf[:, :, i].detach() for i in range(3))
    else:
        q, k, v = randn(g, B, Lq, Hq, dh, dtype=dt), randn(g, B, Lkv, Hk, dh, dtype=dt), randn(g, B, Lkv, Hk, dh, dtype=dt)
    mask = seen_mask(B, Lq, Lkv, window, sinks, pad, lens)
    if garbage:                                                                        # what no query sees holds NaN and infinities
        hidden = ~mask.any(1)
        for t in (k, v):
            t[hidden] = float("nan")
            t[:, ::3][hidden[:, ::3]] = float("inf")
    if train:
        for t in (q, k, v):
            t.requires_grad_()
    out = window_attention(q, k, v, window, sinks=sinks, pad_mask=pad, kv_lens=lens, scale=scale)
    sc = dh ** -0.5 if scale is None else scale
    dout = randn(g, B, Lq, Hq, dh, dtype=dt) if train else None
    ref = attention_ref(q, k, v, mask, sc, dout)
    attention_close(out.detach(), *ref["out"], "out")
    empty = ~mask.any(-1)
    assert float(out.detach()[empty].abs().sum()) == 0.0
    if not train:
        return
    grads = torch.autograd.grad(out, (q, k, v), dout)
    for got, name in zip(grads, ("dq", "dk", "dv")):
        attention_close(got, *ref[name], name)
    assert float(grads[0][empty].abs().sum()) == 0.0
    hidden = ~mask.any(1)
    assert float(grads[1][hidden].abs().sum()) == 0.0 and float(grads[2][hidden].abs().sum()) == 0.0
    with torch.no_grad():
        assert torch.equal(window_attention(q, k, v, window, sinks=sinks, pad_mask=pad, kv_lens=lens, scale=scale), out)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,L,Hq,Hk,dh,window,sinks", [
    (1, 1, 1, 1, 8, (None, None), 0), (1, 1, 4, 2, 64, (0, 0), 1), (2, 31, 2, 2, 32, (5, 5), 0), (2, 32, 2, 1, 40, (None, 0), 0),
    (1, 96, 4, 4, 64, (24, 24), 1), (2, 97, 6, 2, 64, (16, 0), 4), (3, 130, 3, 3, 96, (40, 7), 3), (1, 257, 8, 1, 128, (None, None), 0),
    (2, 333, 4, 2, 80, (100, 60), 70), (1, 700, 2, 2, 64, (0, 0), 0), (1, 1025, 6, 6, 64, (128, 128), 1), (1, 1500, 4, 1, 128, (200, 0), 130),
    (1, 900, 2, 1, 24, (0, 0), 5), (1, 640, 5, 1, 64, (3, None), 2), (2, 300, 3, 1, 48, (None, 9), 4)])
def test_window_attention_forward_and_gradients(B, L, Hq, Hk, dh, window, sinks, dtype):
    attention_case(B, L, L, Hq, Hk, dh, window, sinks, dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh", [32, 56, 96, 120, 128])
def test_window_attention_every_workgroup_shape(dh, dtype):
    """Enough rows for workgroups of 128, 64 and 32 of them, with and without shared key heads and padding."""
    g = gen(dh)
    for B, L, Hq, Hk in ((32, 190, 8, 8), (64, 65, 8, 2), (64, 100, 2, 2), (3, 60, 2, 2)):
        pad = torch.arange(L, device="cuda")[None, :] >= torch.randint(1, L + 1, (B, 1), generator=g, device="cuda")
        attention_case(B, L, L, Hq, Hk, dh, (33, 21), 2, dtype)
        attention_case(B, L, L, Hq, Hk, dh, (40, 0), 3, dtype, pad=pad)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,L,Hq,Hk,dh", [(64, 130, 8, 2, 128), (43, 140, 9, 3, 128), (64, 160, 16, 2, 120), (1, 4100, 32, 8, 128)])
def test_window_attention_wide_key_tiles_of_shared_heads(B, L, Hq, Hk, dh, dtype):
    """Gradients over 128-key tiles where the query heads of a key head divide a row block and where they do not."""
    attention_case(B, L, L, Hq, Hk, dh, (33, 21), 2, dtype)


@pytest.mark.parametrize("L,Hq,Hk,dh,window,sinks", [(3000, 2, 1, 64, (0, 0), 600), (2500, 1, 1, 32, (3, 0), 100), (3000, 4, 1, 128, (10, 10), 130)])
def test_window_attention_many_first_tokens(L, Hq, Hk, dh, window, sinks):
    """First tokens over several key tiles: with pieces of their far rows, and (more than 8 tiles) without."""
    attention_case(1, L, L, Hq, Hk, dh, window, sinks, "bf16")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Lq,Lkv,window,sinks", [(5, 200, (30, 0), 2), (200, 5, (30, 0), 2), (64, 64, (10, 10), 0), (1, 1000, (100, 0), 4), (130, 300, (None, 0), 0),
                                                 (3, 0, (4, 4), 1), (0, 3, (4, 4), 1)])
def test_window_attention_padding_lengths_and_other_query_counts(Lq, Lkv, window, sinks, dtype):
    g = gen(Lq + Lkv)
    pad = torch.rand(3, Lkv, generator=g, device="cuda") < 0.4
    pad[1] = True                                                                      # a sample without any key
    attention_case(3, Lq, Lkv, 4, 2, 64, window, sinks, dtype, pad=pad)
    lens = torch.tensor([Lkv, Lkv // 3, 0], device="cuda", dtype=torch.int64 if Lq % 2 else torch.int32)
    attention_case(3, Lq, Lkv, 4, 4, 64, window, sinks, dtype, lens=lens)
    attention_case(3, Lq, Lkv, 6, 2, 72, window, sinks, dtype, lens=lens, pad=pad)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lkv,Hq,Hk,dh,left,sinks", [(8, 1, 4096, 16, 4, 128, 1023, 4), (1, 1, 30000, 8, 8, 64, None, 0), (2, 1, 77, 4, 1, 40, 20, 3),
                                                        (3, 2, 9000, 32, 8, 128, 4000, 1), (16, 1, 5000, 6, 6, 64, 300, 64), (1, 40, 6000, 8, 2, 128, 2000, 4),
                                                        (1, 1, 1, 64, 1, 128, 0, 0), (5, 3, 2500, 96, 2, 96, 1000, 200)])
def test_window_attention_single_tokens_over_a_cache(B, Lq, Lkv, Hq, Hk, dh, left, sinks, dtype):
    """Few queries over a long cache: the keys are split over workgroups; slots outside the window and behind the length hold NaN."""
    lens = torch.tensor([max(1, Lkv - b * Lkv // B) for b in range(B)], device="cuda", dtype=torch.int32)
    attention_case(B, Lq, Lkv, Hq, Hk, dh, (left, 0), sinks, dtype, lens=lens, train=False)


def test_window_attention_strides_views_scale_and_alignment():
    from vipformer_amd.ops_block import window_attention
    attention_case(2, 150, 150, 6, 6, 64, (30, 30), 1, "fp16", views=True, garbage=False)
    attention_case(1, 200, 200, 4, 4, 128, (64, 0), 2, "bf16", views=True, garbage=False, scale=0.31)
    g = gen(5)
    q = randn(g, 2, 4, 60, 64, dtype=torch.float16).transpose(1, 2)                    # heads first
    odd = randn(g, 2 * 60 * 4 * 64 + 3, dtype=torch.float16)[3:].view(2, 60, 4, 64)    # a base that is not 16-byte aligned
    rows = randn(g, 2, 60, 4, 68, dtype=torch.float16)[..., :64]                       # a head stride that is no multiple of 8
    wide = randn(g, 1, 60, 1, 64, dtype=torch.float16).expand(2, 60, 4, 64)            # one tensor for every sample and head
    for a, b, c in ((q, odd, rows), (odd, wide, q), (rows, q, wide)):
        a, b, c = (t.detach().requires_grad_() for t in (a, b, c))
        out = window_attention(a, b, c, (9, 3), sinks=2)
        dout = randn(g, 2, 4, 60, 64, dtype=torch.float16).transpose(1, 2)
        ref = attention_ref(a, b, c, seen_mask(2, 60, 60, (9, 3), 2, None, None), 0.125, dout)
        attention_close(out.detach(), *ref["out"], "out")
        for got, name in zip(torch.autograd.grad(out, (a, b, c), dout), ("dq", "dk", "dv")):
            attention_close(got, *ref[name], name)


def test_window_attention_query_heads_far_apart():
    """512 heads of one key head over 4 GiB: the gradient's kernels have 32-bit offsets inside a stage."""
    from vipformer_amd.ops_block import window_attention
    g = gen(11)
    near, (k, v) = randn(g, 1, 3, 512, 8, dtype=torch.bfloat16), (randn(g, 1, 70, 1, 8, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    far, dout = (torch.empty(512 << 22, dtype=torch.bfloat16, device="cuda").as_strided((1, 3, 512, 8), (1 << 31, 8, 1 << 22, 1)) for _ in range(2))
    far.copy_(near)
    dout.copy_(randn(g, 1, 3, 512, 8, dtype=torch.bfloat16))
    runs = []
    for q, d in ((near, dout.contiguous()), (far.detach(), dout)):
        q.requires_grad_()
        out = window_attention(q, k, v, (20, 0))
        runs.append((out.detach(), *torch.autograd.grad(out, (q, k, v), d)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_window_attention_large_scores_and_growing_maxima():
    """Scores from -300 to 300 whose maximum rises along the keys (the running maximum moves many times) and falls."""
    from vipformer_amd.ops_block import window_attention
    g = gen(6)
    for sign in (1.0, -1.0):
        q, k, v = randn(g, 1, 100, 2, 64), randn(g, 1, 400, 2, 64), randn(g, 1, 400, 2, 64)
        q[..., 0], k[..., 0] = 20.0, sign * torch.linspace(-12, 12, 400, device="cuda")[None, :, None]
        q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
        out = window_attention(q, k, v, scale=1.0)
        ref = attention_ref(q, k, v, torch.ones(1, 100, 400, dtype=torch.bool, device="cuda"), 1.0)
        # fp32 scores of 300 carry 2^-24 * 300 * log2(e) / 2 + 64 sums: 1e-4 relative in the weights, below half a step of bf16
        attention_close(out, *ref["out"], "out")


def test_window_attention_is_bitwise_reproducible():
    from vipformer_amd.ops_block import window_attention
    g = gen(8)
    q, k, v = (randn(g, 2, 900, h, 64, dtype=torch.bfloat16).requires_grad_() for h in (8, 2, 2))
    dout = randn(g, 2, 900, 8, 64, dtype=torch.bfloat16)
    runs = []
    for _ in range(3):
        out = window_attention(q, k, v, (60, 0), sinks=4)
        runs.append([out.detach(), *torch.autograd.grad(out, (q, k, v), dout)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ------------------------------------------------------------------------------------------ edges that the three share
def test_empty_calls_and_zero_gradients():
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    w, gate = torch.ones(16, device="cuda", requires_grad=True), torch.ones(2, 1, 16, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 16, device="cuda", requires_grad=True)
    h, n = gated_norm_residual(x, x.detach().half(), gate=gate, post=(w, None), pre=(w, None), kind="rms")
    assert h.shape == n.shape == x.shape
    dx, dw, dg = torch.autograd.grad((h, n), (x, w, gate), (h.detach(), n.detach()))
    assert dx.shape == x.shape and float(dw.abs().sum()) == 0.0 and float(dg.abs().sum()) == 0.0
    q = torch.zeros(0, 5, 2, 16, device="cuda", dtype=torch.float16)
    assert rotary_axes(q, q, torch.zeros(5, 1, device="cuda"), RotaryAxes((8,), 16))[1].shape == q.shape
    assert window_attention(q, q, q, (3, 3)).shape == q.shape


def test_block_ops_refuse_a_second_derivative():
    from vipformer_amd import _lib
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    g = gen(1)
    q = randn(g, 1, 8, 1, 16, dtype=torch.float16).requires_grad_()
    x = randn(g, 1, 8, 16).requires_grad_()
    for out, leaf in ((rotary_axes(q, None, torch.zeros(8, 1, device="cuda"), RotaryAxes((8,), 16)), q), (window_attention(q, q, q), q),
                      (gated_norm_residual(x, x)[0], x)):
        with pytest.raises(_lib.VpfError, match="differentiable once"):
            torch.autograd.grad(out.float().sum(), leaf, create_graph=True)


def test_block_ops_mixed_devices_and_cpu_tensors_are_refused():
    from vipformer_amd import _lib
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    q, cpu = torch.zeros(1, 4, 1, 16, device="cuda", dtype=torch.float16), torch.zeros(1, 4, 1, 16, dtype=torch.float16)
    for call in (lambda: rotary_axes(q, None, torch.zeros(4, 1), RotaryAxes((8,), 16)), lambda: window_attention(q, cpu, cpu),
                 lambda: window_attention(q, q, q, kv_lens=torch.ones(1, dtype=torch.int32)), lambda: gated_norm_residual(q, q, post=(torch.ones(16), None))):
        with pytest.raises(_lib.VpfError):
            call()


def block_inputs(g, B=2, L=145, D=256, H=4):
    c = lambda *s, scale=1.0, dt=torch.float32: randn(g, *s, scale=scale, dtype=dt)
    P = dict(x=c(B, L, D), a=c(B, L, D, dt=torch.float16), wqkv=c(3 * D, D, scale=D ** -0.5, dt=torch.float16), wo=c(D, D, scale=D ** -0.5, dt=torch.float16),
             gate=c(D, scale=0.5), w1=1.0 + c(D, scale=0.1), b1=c(D, scale=0.1), w2=1.0 + c(D, scale=0.1), b2=c(D, scale=0.1))
    grid = torch.stack(torch.meshgrid(torch.arange(12.0), torch.arange(12.0), indexing="ij"), -1).reshape(-1, 2)
    pos = torch.cat([torch.zeros(1, 2), grid]).cuda()
    return P, pos


def block(P, pos, plan, pad=None):
    """Projection -> rotary positions -> windowed attention -> projection -> gated norms: the operators as one encoder block uses them."""
    from vipformer_amd.ops_block import gated_norm_residual, rotary_axes, window_attention
    B, L, D = P["x"].shape
    qkv = torch.nn.functional.linear(P["a"], P["wqkv"]).view(B, L, 3, plan.heads, plan.head_dim)
    q, k = rotary_axes(qkv[:, :, 0], qkv[:, :, 1], pos, plan)
    o = window_attention(q, k, qkv[:, :, 2], (32, 32), sinks=1, pad_mask=pad)
    y = torch.nn.functional.linear(o.flatten(2), P["wo"])
    return gated_norm_residual(P["x"], y, gate=P["gate"], post=(P["w1"], P["b1"]), pre=(P["w2"], P["b2"]), alpha=0.9)


def block_plan(H=4, dh=64):
    from vipformer_amd.ops_block import RotaryAxes
    plan = RotaryAxes((16, 16), dh, base=100.0)
    plan.heads = H
    return plan


def test_a_block_of_them_against_64_bits():
    """The run as it is used, forward and every gradient.  16 roundings to fp16 on the way (6 forward, 10 back), each 2^-11 of its tensor, at most
    doubled by softmax and norms: 2^-6 of the result's norm."""
    g = gen(21)
    P, pos = block_inputs(g)
    plan = block_plan()
    pad = torch.zeros(2, 145, dtype=torch.bool, device="cuda")
    pad[1, 100:] = True
    for t in P.values():
        t.requires_grad_()
    h, n = block(P, pos, plan, pad)
    dh, dn = randn(g, *h.shape), randn(g, *n.shape, dtype=torch.float16)
    grads = torch.autograd.grad((h, n), list(P.values()), (dh, dn))

    R = {k: v.detach().double().requires_grad_() for k, v in P.items()}
    B, L, D = R["x"].shape
    qkv = (R["a"] @ R["wqkv"].t()).view(B, L, 3, 4, 64)
    f = plan.frequencies().cuda()
    ang = torch.cat([pos[:, :1].double() * f[:16], pos[:, 1:].double() * f[16:]], -1)[None, :, None]
    turn = lambda t: torch.cat([t[..., :32] * ang.cos() - t[..., 32:] * ang.sin(), t[..., 32:] * ang.cos() + t[..., :32] * ang.sin()], -1)
    q, k, v = (t.transpose(1, 2) for t in (turn(qkv[:, :, 0]), turn(qkv[:, :, 1]), qkv[:, :, 2]))
    m = seen_mask(B, L, L, (32, 32), 1, pad, None)[:, None]
    s = (q @ k.transpose(-1, -2) / 8.0).masked_fill(~m, -math.inf)
    dead = ~m.any(-1, keepdim=True)
    o = (torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0) @ v).transpose(1, 2).reshape(B, L, D)
    y = o @ R["wo"].t()
    ln = lambda z, w, b: torch.nn.functional.layer_norm(z, (D,), w, b, 1e-5)
    hr = 0.9 * R["x"] + R["gate"] * ln(y, R["w1"], R["b1"])
    nr = ln(hr, R["w2"], R["b2"])
    ref = torch.autograd.grad((hr, nr), list(R.values()), (dh.double(), dn.double()))
    for name, a, b in [("h", h, hr), ("n", n, nr)] + list(zip(P, grads, ref)):
        a, b = a.detach().double(), b.detach()
        rel = float((a - b).norm() / b.norm())
        assert rel < 2.0 ** -6, (name, rel)


def test_gradients_against_differences():
    """<gradient, d> against (f(x + e d) - f(x - e d)) / 2 e of the operators themselves.  fp32: e = 2^-6, the difference carries e^2 / 6 of the third
    derivative and 2^-24 / e of each of the summed outputs, below 2^-9 of the sum of their magnitudes."""
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes
    g = gen(22)
    plan = RotaryAxes((4, 4), 20)
    q, dq, pos = randn(g, 2, 9, 3, 20), randn(g, 2, 9, 3, 20), torch.rand(9, 2, generator=g, device="cuda") * 50
    cq = randn(g, 2, 9, 3, 20)
    f = lambda t: float((rotary_axes(t, None, pos, plan).double() * cq).sum())
    q.requires_grad_()
    (grad,) = torch.autograd.grad(rotary_axes(q, None, pos, plan), q, cq)
    e = 2.0 ** -6
    with torch.no_grad():
        diff = (f(q + e * dq) - f(q - e * dq)) / (2 * e)
    assert abs(diff - float((grad.double() * dq).sum())) < 2.0 ** -9 * float((cq * dq).abs().sum())
    for kind in ("layer", "rms"):
        t = {n: randn(g, *s) for n, s in dict(x=(3, 7, 48), y=(3, 7, 48), gate=(3, 1, 48), w1=(48,), b1=(48,), w2=(48,), b2=(48,)).items()}
        ch, cn = randn(g, 3, 7, 48), randn(g, 3, 7, 48)
        run = lambda t: gated_norm_residual(t["x"], t["y"], gate=t["gate"], post=(t["w1"], t["b1"]), pre=(t["w2"], t["b2"]), kind=kind, alpha=0.9, beta=0.75)
        f = lambda t: sum(float((a.double() * c).sum()) for a, c in zip(run(t), (ch, cn)))
        leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
        grads = dict(zip(t, torch.autograd.grad(run(leaves), list(leaves.values()), (ch, cn))))
        for name in t:
            d = randn(g, *t[name].shape)
            e = 2.0 ** -8
            diff = (f({**t, name: t[name] + e * d}) - f({**t, name: t[name] - e * d})) / (2 * e)
            assert abs(diff - float((grads[name].double() * d).sum())) < 2.0 ** -9 * float((grads[name] * d).abs().sum() + ch.abs().sum()), (kind, name)


def test_captured_block_follows_its_inputs_over_replays():
    """Forward and backward of the block in one captured graph: replays with new inputs, eager work and synchronisations in between, bit for bit."""
    g = gen(23)
    P, pos = block_inputs(g)
    plan = block_plan()
    for t in P.values():
        t.requires_grad_()
    dh, dn = randn(g, 2, 145, 256), randn(g, 2, 145, 256, dtype=torch.float16)

    def step():
        h, n = block(P, pos, plan)
        return [h.detach(), n.detach(), *torch.autograd.grad((h, n), list(P.values()), (dh, dn))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            P["a"].copy_(randn(g, *P["a"].shape, dtype=torch.float16))
            P["x"].copy_(randn(g, *P["x"].shape))
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i


def test_captured_decode_follows_lengths_and_cache():
    """Single tokens over a preallocated cache in a captured graph: lengths and cache advance on the device between replays."""
    from vipformer_amd.ops_block import window_attention
    g = gen(24)
    B, cap, Hq, Hk, dh = 3, 9000, 8, 2, 128
    q = randn(g, B, 1, Hq, dh, dtype=torch.bfloat16)
    kc, vc = (torch.full((B, cap, Hk, dh), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    lens = torch.tensor([5000, 4097, 100], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens.tolist()):
        kc[b, :n], vc[b, :n] = randn(g, n, Hk, dh, dtype=torch.bfloat16), randn(g, n, Hk, dh, dtype=torch.bfloat16)
    run = lambda: window_attention(q, kc, vc, (4095, 0), sinks=4, kv_lens=lens)
    run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):
        at = lens.long()
        for b in range(B):
            kc[b, at[b]], vc[b, at[b]] = randn(g, Hk, dh, dtype=torch.bfloat16), randn(g, Hk, dh, dtype=torch.bfloat16)
        q.copy_(randn(g, B, 1, Hq, dh, dtype=torch.bfloat16))
        lens += 1
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, run())
        m = seen_mask(B, 1, cap, (4095, 0), 4, None, lens)
        attention_close(got, *attention_ref(q, kc, vc, m, dh ** -0.5)["out"], "decode")


def test_calls_on_two_streams_at_once():
    """Two streams, each with its own inputs, many calls in flight: every result is the one a lone call gives."""
    from vipformer_amd.ops_block import gated_norm_residual, window_attention
    g = gen(25)
    sets = []
    for _ in range(2):
        q, k, v = (randn(g, 1, 2000, h, 64, dtype=torch.bfloat16).requires_grad_() for h in (4, 2, 2))
        x, w = randn(g, 1, 2000, 256).requires_grad_(), randn(g, 256).requires_grad_()
        sets.append((q, k, v, x, w, randn(g, 1, 2000, 256), randn(g, 1, 1, 4, 64, dtype=torch.bfloat16), randn(g, 1, 20000, 2, 64, dtype=torch.bfloat16)))

    def work(s):
        q, k, v, x, w, dh, qs, kv = s
        out = window_attention(q, k, v, (50, 0), sinks=3)
        h, _ = gated_norm_residual(x, out.flatten(2), gate=w, post=(w, None), kind="rms")
        return [out.detach(), h.detach(), *torch.autograd.grad(h, (q, k, v, x, w), dh), window_attention(qs, kv, kv, (9999, 0))]

    alone = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))


def test_expanded_gradients_and_sums():
    """Gradients that arrive with strides of 0 (a plain .sum()) and through views."""
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    g = gen(26)
    q = randn(g, 2, 40, 4, 64, dtype=torch.float16).requires_grad_()
    out = window_attention(q, q, q, (9, 9))
    (a,) = torch.autograd.grad(out.sum(), q)
    m = seen_mask(2, 40, 40, (9, 9), 0, None, None)
    ref = attention_ref(q, q, q, m, 0.125, torch.ones_like(q))
    # three gradients of one tensor, added in fp16: two more roundings, each half a step of a partial sum
    extra = sum(ref[n][0].abs() for n in ("dq", "dk", "dv"))
    d = (a.double() - sum(ref[n][0] for n in ("dq", "dk", "dv"))).abs()
    assert float((d - 2.0 ** -11 * (3 * extra + 8 * sum(ref[n][1] for n in ("dq", "dk", "dv"))) - 1e-5).max()) <= 0.0
    plan, pos = RotaryAxes((32,), 64), torch.arange(40, device="cuda")[:, None]
    (b,) = torch.autograd.grad(rotary_axes(q, None, pos, plan).sum(), q)
    r, size = rotary_ref(torch.ones_like(q), pos, plan, -1.0)
    close(b, r, ROT * size, "rotary")
    x = randn(g, 2, 40, 64).requires_grad_()
    h, n = gated_norm_residual(x, x.detach(), pre=(None, None))
    (c,) = torch.autograd.grad(h.sum() + n.transpose(0, 1).sum(), x)
    one = torch.ones_like(x)
    ref = norm_ref(x, x.detach(), None, None, (None, None), "layer", 1.0, 1.0, 1e-5, one, one)
    close(c, ref["dx"][0], BWD_N * ref["dx"][1], "norm")


def test_rotary_in_place_through_the_c_abi():
    """oq = q, ok = k: the same bits as with outputs of their own."""
    from vipformer_amd import _lib as L, ops_block as O
    g = gen(27)
    for layout in ("half", "pair"):
        plan = O.RotaryAxes((10, 10), 48, layout=layout)
        q, k, pos = randn(g, 2, 300, 6, 48, dtype=torch.bfloat16), randn(g, 2, 300, 2, 48, dtype=torch.bfloat16), torch.rand(300, 2, generator=g, device="cuda") * 9
        oq, ok = O.rotary_axes(q, k, pos, plan)
        freq, axis = plan.tables(q.device)
        s = O._strides(q) + O._strides(k)
        L.launch("vpf_rotary_axes", O._pack_rotary(2, 300, 6, 2, 48, 20, 2, plan.layout_code, 2, 0, 0, 0, q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(),
                                                   *s, *s, pos.data_ptr(), 0, freq.data_ptr(), axis.data_ptr()), q.device)
        assert torch.equal(q, oq) and torch.equal(k, ok)


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^32 bytes (and elements): a cache of 2.1 million tokens, as many tokens to rotate and to norm."""
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    g = gen(28)
    n, dt = (1 << 21) + 5, torch.bfloat16
    k, v = (torch.empty(1, n, 8, 128, dtype=dt, device="cuda") for _ in range(2))
    tail = slice(n - 3100, n)
    for t in (k, v):
        t.fill_(float("nan"))
        t[:, tail], t[:, :4] = randn(g, 1, 3100, 8, 128, dtype=dt), randn(g, 1, 4, 8, 128, dtype=dt)
    q = randn(g, 1, 2, 16, 128, dtype=dt)
    out = window_attention(q, k, v, (3000, 0), sinks=4)
    cat = lambda t: torch.cat([t[:, :4], t[:, tail]], 1)
    p = torch.arange(2)[:, None] + 3102
    j = torch.arange(3104)[None]
    m = ((j <= p) & ((j >= p - 3000) | (j < 4)))[None].cuda()
    attention_close(out, *attention_ref(q, cat(k), cat(v), m, 128 ** -0.5)["out"], "cache")
    k[:, :-16] = 0.5
    plan, pos = RotaryAxes((64,), 128), torch.arange(n, device="cuda", dtype=torch.int32)[:, None]
    r = rotary_axes(k, None, pos, plan)
    ref, size = rotary_ref(k[:, -16:], pos[-16:], plan)
    close(r[:, -16:], ref, ROT * size, "rotary")
    del r, v
    x = k.view(n, 1024)
    h, nn = gated_norm_residual(x, x, pre=(None, None), kind="rms")
    ref = norm_ref(x[-16:], x[-16:], None, None, (None, None), "rms", 1.0, 1.0, 1e-5, x[-16:], x[-16:])
    close(h[-16:], ref["h"][0], FWD_N * ref["h"][1], "h")
    close(nn[-16:], ref["n"][0], FWD_N * ref["n"][1], "n")


# ------------------------------------------------------------------------------------------ under torch's own machinery
@pytest.mark.parametrize("pinned", [False, True])
def test_gradients_of_tensors_that_were_offloaded(pinned):
    """Saved tensors that travel to the host and back: packed q / k / v slices return contiguous."""
    from vipformer_amd.ops_block import RotaryAxes, gated_norm_residual, rotary_axes, window_attention
    g = gen(21)
    plan, pos = RotaryAxes((16, 16), 64), torch.randint(0, 50, (90, 2), generator=g, device="cuda")
    qkv, w = randn(g, 2, 90, 3, 6, 64, dtype=torch.bfloat16).requires_grad_(), randn(g, 64).requires_grad_()
    dout = randn(g, 2, 90, 6, 64, dtype=torch.bfloat16)

    def grads():
        q, k, v = qkv.unbind(2)
        out = window_attention(q, k, v, (9, 0), sinks=1) + window_attention(*rotary_axes(q, k, pos, plan), v, (20, 4))
        h, n = gated_norm_residual(out, v, post=(w, None), pre=(w, None), kind="rms")
        return torch.autograd.grad((h, n), (qkv, w), (dout, dout))
    plain = grads()
    with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
        moved = grads()
    assert all(torch.equal(a, b) for a, b in zip(plain, moved))


@pytest.mark.parametrize("dtype", ["f32", "fp16", "bf16"])
@pytest.mark.parametrize("scale", [0.05, 0.003])
def test_gated_norm_default_epsilon_of_rms_modules(dtype, scale):
    """RMSNorm(D) without an epsilon, behind and in front of a block, on small activations: the module's own formula with fp32's epsilon, and
    the module's own output on the same inputs."""
    from vipformer_amd.ops_block import gated_norm_residual
    g, dt, eps = gen(22), TYPES[dtype], torch.finfo(torch.float32).eps
    z, zero = randn(g, 40, 256, dtype=dt, scale=scale), torch.zeros(40, 256, dtype=dt, device="cuda")
    rms = torch.nn.RMSNorm(256, device="cuda")
    with torch.no_grad():
        rms.weight.copy_(1.0 + randn(g, 256, scale=0.2))
        h, _ = gated_norm_residual(zero, z, post=rms, kind="rms")
        h2, n = gated_norm_residual(z, zero, pre=rms, kind="rms")
        own = rms(z.float())
    assert torch.equal(h2, z)
    for got, post, pre, (a, b), name in ((h, (rms.weight, None), None, (zero, z), "h"), (n, None, (rms.weight, None), (z, zero), "n")):
        ref = norm_ref(a, b, None, post, pre, "rms", 1.0, 1.0, eps, zero, zero)
        close(got, ref[name][0], FWD_N * ref[name][1], name)
        # torch's module in fp32 on the same values carries no more roundings than the kernel
        close(got, own.double(), 2 * FWD_N * ref[name][1], "module")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lkv,Hq,Hk,dh,window,sinks", [
    (3, 70, 70, 4, 2, 64, (0, 0), 0), (2, 200, 40, 6, 2, 72, (9, 0), 2), (64, 130, 130, 9, 3, 128, (0, 0), 1), (1, 900, 900, 2, 1, 32, (1, 1), 3),
    (3, 300, 300, 8, 1, 96, (None, 0), 0)])
def test_window_attention_queries_that_see_nothing_hold_anything(B, Lq, Lkv, Hq, Hk, dh, window, sinks, dtype):
    """Queries in front of the first key and queries whose every key is padding, with NaN and infinities in them and in their gradients."""
    from vipformer_amd.ops_block import window_attention
    g, dt = gen(23 + dh), TYPES[dtype]
    q, k, v = randn(g, B, Lq, Hq, dh, dtype=dt), randn(g, B, Lkv, Hk, dh, dtype=dt), randn(g, B, Lkv, Hk, dh, dtype=dt)
    dout = randn(g, B, Lq, Hq, dh, dtype=dt)
    pad = torch.rand(B, Lkv, generator=g, device="cuda") < 0.5
    lens = torch.randint(Lkv // 2, Lkv + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    mask = seen_mask(B, Lq, Lkv, window, sinks, pad, lens)
    blind = ~mask.any(-1)
    assert blind.any() and not blind.all()
    for t, what in ((q, (math.nan, math.inf)), (dout, (-math.inf, math.nan))):
        t[blind] = what[0]
        t[:, ::3][blind[:, ::3]] = what[1]
    for t in (q, k, v):
        t.requires_grad_()
    out = window_attention(q, k, v, window, sinks=sinks, pad_mask=pad, kv_lens=lens)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    zeroed = lambda t: torch.where(blind[..., None, None], 0.0, t.detach())
    ref = attention_ref(zeroed(q), k, v, mask, dh ** -0.5, zeroed(dout))
    attention_close(out.detach(), *ref["out"], "out")
    for got, name in zip(grads, ("dq", "dk", "dv")):
        attention_close(got, *ref[name], name)
    assert float(out.detach()[blind].abs().sum()) == 0.0 and float(grads[0][blind].abs().sum()) == 0.0


def small_steps_close(got, ref, size, flushed, what):
    """attention_close without its absolute terms: half a step of the result (and of fp16's smallest numbers, 2^-25), 8 standard deviations of the
    weights' roundings, and `flushed`: what weights below the smallest number of their scaled fp16 form can add up to."""
    half = torch.finfo(got.dtype).eps / 2
    tol = half * ref.abs() + 8 * half * size + 2.0 ** -25 + flushed
    bad = (got.double() - ref).abs() - tol
    assert got.shape == ref.shape and torch.isfinite(got.double()).all(), what
    assert float(bad.max()) <= 0.0, f"{what}: {int((bad > 0).sum())} of {bad.numel()} outside, worst {float((got.double() - ref).abs().max()):.3e}"


@pytest.mark.parametrize("B,Lq,Lkv,Hq,Hk,dh,window,gsize,vsize,ksize,rows", [
    (1, 2048, 2048, 1, 1, 64, (None, None), 1e-4, 1.0, 1.0, False), (1, 300, 8192, 2, 1, 128, (None, None), 1e-3, 1.0, 1.0, False),
    (1, 300, 8192, 4, 2, 96, (None, None), 1e-4, 1.0, 1.0, False), (64, 200, 200, 4, 4, 128, (None, 0), 1e-5, 1.0, 1.0, True),
    (16, 190, 190, 8, 8, 32, (40, 3), 1e-2, 1.0, 1.0, True), (2, 777, 777, 6, 2, 64, (100, 0), 1.0, 1.0, 1.0, True),
    (1, 70, 70, 2, 1, 64, (5, 0), 300.0, 100.0, 2e-4, False), (32, 190, 190, 8, 8, 64, (33, 21), 500.0, 200.0, 1e-4, True)])
def test_window_attention_fp16_gradients_of_any_size(B, Lq, Lkv, Hq, Hk, dh, window, gsize, vsize, ksize, rows):
    """dS is rounded to fp16 for its products: over many keys it lies far below fp16's smallest numbers, with large values and gradients far beyond
    its largest, while dq and dk are ordinary.  `rows`: gradients that differ by 10^4 from query to query."""
    from vipformer_amd.ops_block import window_attention
    g, dt = gen(24 + Lq), torch.float16
    q, k, v = randn(g, B, Lq, Hq, dh, dtype=dt), randn(g, B, Lkv, Hk, dh, scale=ksize, dtype=dt), randn(g, B, Lkv, Hk, dh, scale=vsize, dtype=dt)
    q = (q.float() * (1.0 if ksize == 1.0 else 0.1)).to(dt)
    dout = randn(g, B, Lq, Hq, dh, scale=gsize)
    if rows:
        dout = dout * 10.0 ** -(torch.arange(Lq, device="cuda") % 5)[:, None, None]
    dout = dout.to(dt)
    for t in (q, k, v):
        t.requires_grad_()
    mask, scale = seen_mask(B, Lq, Lkv, window, 0, None, None), dh ** -0.5
    ref = attention_ref(q, k, v, mask, scale, dout)
    out = window_attention(q, k, v, window)
    dq, dk, _ = torch.autograd.grad(out, (q, k, v), dout)
    # scaled weights of a row or a key: its largest at 2^10 or more, the smallest step 2^-24 -- half of that for each of n terms, 8 deviations
    most = 2.0 * float(dout.abs().double().sum(-1).max() * v.detach().abs().max())
    flushed = lambda n, t: 8 * 2.0 ** -35 * most * scale * math.sqrt(n) * float(t.detach().abs().max())
    small_steps_close(dq, *ref["dq"], flushed(Lkv, k), "dq")
    small_steps_close(dk, *ref["dk"], flushed(Lq * Hq // Hk, q), "dk")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lkv,Hq,Hk,dh", [(1, 1, 4100, 4, 1, 128), (1, 200, 4100, 1, 1, 64), (64, 65, 4100, 8, 2, 40), (16, 200, 4100, 16, 16, 96)])
def test_window_attention_weights_far_below_the_largest(B, Lq, Lkv, Hq, Hk, dh, dtype):
    """A first token that takes nearly all the weight and has no value (weights of the others: 2^-24.6 of it, 2^-25 .. 2^-24 with their own
    differences): the result is what the others hold."""
    from vipformer_amd.ops_block import window_attention
    g, dt = gen(25 + dh), TYPES[dtype]
    q, k, v = torch.zeros(B, Lq, Hq, dh, device="cuda"), torch.zeros(B, Lkv, Hk, dh, device="cuda"), randn(g, B, Lkv, Hk, dh, scale=3e3) + 2e4
    q[..., 0], q[..., 1] = 1.0, 0.25
    k[:, 0, :, 0], v[:, 0] = 17.05, 0.0
    k[:, 1:, :, 1] = torch.rand(B, Lkv - 1, Hk, generator=g, device="cuda") - 0.5
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out = window_attention(q, k, v, scale=1.0)
    ref = attention_ref(q, k, v, torch.ones(B, Lq, Lkv, dtype=torch.bool, device="cuda"), 1.0)["out"]
    # scores of 17 in fp32: 2^-24 * 17 * log2(e), the sum of 4100 weights: 2^-24 a term and 2^-12 at most -- below half a step of fp16 together
    small_steps_close(out, ref[0], ref[1], 2.0 ** -12 * ref[0].abs(), "out")


def test_window_attention_fp16_value_gradients_of_very_many_keys():
    """Weights of 2^-19.07 = 30.5 steps of 2^-24: dv is their sum over the queries times the gradients."""
    from vipformer_amd.ops_block import window_attention
    g, B, Lq, n, dh = gen(26), 1, 40, 550073, 32
    q, k, v = torch.zeros(B, Lq, 1, dh, device="cuda").half(), randn(g, B, n, 1, dh, dtype=torch.float16), randn(g, B, n, 1, dh, dtype=torch.float16).requires_grad_()
    dout = randn(g, B, Lq, 1, dh, dtype=torch.float16, scale=1000.0)
    (dv,) = torch.autograd.grad(window_attention(q, k, v), (v,), dout)
    ref = (dout.double().sum(1, keepdim=True) / n).expand(B, n, 1, dh)
    size = ((dout.double() ** 2).sum(1, keepdim=True).sqrt() / n).expand(B, n, 1, dh)
    # the sum of the weights in fp32, 550073 terms of one size in tiles: 2^-12 of it at most
    small_steps_close(dv, ref, size, 2.0 ** -12 * ref.abs(), "dv")


def kernels_of(call):
    """Names of the kernels that a call launches."""
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return [e.key for e in p.key_averages()]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh", [72, 96, 120, 128])
@pytest.mark.parametrize("B,L,Hq,Hk,window,sinks", [(8, 1030, 32, 8, (1023, 0), 3), (3, 4100, 16, 16, (4095, 0), 0), (2, 4200, 27, 9, (2000, 30), 70)])
def test_window_attention_two_row_blocks_a_wave(B, L, Hq, Hk, window, sinks, dh, dtype):
    """Long walks beside many rows: forward with two blocks of rows in a wave, rows that are no multiple of 256, first tokens, padding and lengths;
    some heads of every sample against 64 bits."""
    from vipformer_amd.ops_block import window_attention
    g, dt = gen(27 + dh), TYPES[dtype]
    q, k, v = randn(g, B, L, Hq, dh, dtype=dt), randn(g, B, L, Hk, dh, dtype=dt), randn(g, B, L, Hk, dh, dtype=dt)
    pad = torch.rand(B, L, generator=g, device="cuda") < 0.3
    lens = torch.tensor([L - 37 * b - (b > 0) * 300 for b in range(B)], device="cuda", dtype=torch.int32)
    plain = lambda: window_attention(q, k, v, window, sinks=sinks)
    names = kernels_of(plain)
    assert any("wa_fwd_kernel" in n and ("4, 2, 1, 64" in n or "Li4ELi2ELi1ELi64E" in n) for n in names), names
    pick = (0, Hk // 2, Hk - 1)
    for p, n in ((None, None), (pad, None), (None, lens), (pad, lens)):
        hidden = ~seen_mask(B, L, L, window, sinks, p, n).any(1)
        kk, vv = k.clone(), v.clone()
        kk[hidden], vv[hidden] = float("nan"), float("inf")
        out = window_attention(q, kk, vv, window, sinks=sinks, pad_mask=p, kv_lens=n)
        for b in range(B):
            mask = seen_mask(B, L, L, window, sinks, p, n)[b:b + 1]
            for h in pick:
                part = lambda t, m: t[b:b + 1, :, h * m:(h + 1) * m]
                ref = attention_ref(part(q, Hq // Hk), part(kk, 1), part(vv, 1), mask, dh ** -0.5)["out"]
                attention_close(part(out, Hq // Hk), *ref, f"sample {b} head {h}")
                if b and h:
                    break


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh", [80, 128])
def test_window_attention_two_row_blocks_a_wave_and_their_gradients(dh, dtype):
    from vipformer_amd.ops_block import window_attention
    B, L, Hq, Hk, window, sinks = 8, 1030, 32, 8, (1023, 0), 3
    g, dt = gen(28 + dh), TYPES[dtype]
    q, k, v = (randn(g, B, L, h, dh, dtype=dt).requires_grad_() for h in (Hq, Hk, Hk))
    dout = randn(g, B, L, Hq, dh, dtype=dt)
    pad = torch.rand(B, L, generator=g, device="cuda") < 0.3
    lens = torch.tensor([L - 61 * b for b in range(B)], device="cuda", dtype=torch.int32)
    for p, n in ((None, None), (pad, lens)):
        out = window_attention(q, k, v, window, sinks=sinks, pad_mask=p, kv_lens=n)
        grads = torch.autograd.grad(out, (q, k, v), dout)
        for b, h in ((0, 0), (3, 5), (7, 7)):
            part = lambda t, m: t.detach()[b:b + 1, :, h * m:(h + 1) * m]
            wide = Hq // Hk
            ref = attention_ref(part(q, wide), part(k, 1), part(v, 1), seen_mask(B, L, L, window, sinks, p, n)[b:b + 1], dh ** -0.5, part(dout, wide))
            for got, name, m in zip((out, *grads), ("out", "dq", "dk", "dv"), (wide, wide, 1, 1)):
                attention_close(part(got, m), *ref[name], f"{name}, sample {b}, key head {h}")


@pytest.mark.parametrize("far", [2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_window_attention_lengths_are_clamped_in_64_bits(far):
    from vipformer_amd.ops_block import window_attention
    g = gen(29)
    q, k, v = randn(g, 4, 3, 4, 64, dtype=torch.float16), *(randn(g, 4, 200, 2, 64, dtype=torch.float16) for _ in range(2))
    lens = torch.tensor([far, -far, 17, 200], device="cuda")
    clamped = lens.clamp(0, 200)
    a, b, c = (window_attention(q, k, v, (50, 0), sinks=1, kv_lens=n) for n in (lens, clamped, clamped.int()))
    strided = window_attention(q, k, v, (50, 0), sinks=1, kv_lens=torch.stack([lens, lens + 1], 1)[:, 0])
    assert torch.equal(a, b) and torch.equal(b, c) and torch.equal(c, strided)
    assert float(a[1].abs().sum()) == 0.0 and float(a[0].abs().sum()) > 0.0


@pytest.mark.parametrize("train", [False, True])
def test_window_attention_heads_first_caches_beyond_32_bits(train):
    """Heads that lie 70000 x 128 elements apart, the last of 250 beyond 2^31 elements: single tokens, and (3 heads) a prompt with its gradients, as
    over a copy with the tokens first."""
    from vipformer_amd.ops_block import window_attention
    g = gen(30)
    B, heads = (2, 3) if train else (1, 250)
    cache = torch.empty(B, heads, 70000, 128, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    k, v = (t.transpose(1, 2) for t in ((cache, cache.flip(1)) if train else (cache, cache)))
    lens = torch.tensor([70000, 65537][:B], device="cuda")
    Lq = 40 if train else 1
    q = randn(g, B, Lq, heads, 128, dtype=torch.bfloat16)
    runs = []
    for a, b in ((k, v), (k.contiguous(), v.contiguous())):
        leaves = [t.detach().requires_grad_(train) for t in (q, a, b)]
        out = window_attention(*leaves, (69000, 0), sinks=2, kv_lens=lens)
        grads = torch.autograd.grad(out, leaves, q) if train else ()
        runs.append([out.detach(), *grads])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    m = seen_mask(B, Lq, 70000, (69000, 0), 2, None, lens)
    last = slice(heads - 1, heads)
    attention_close(runs[0][0][:, :, last], *attention_ref(q[:, :, last], k[:, :, last], v[:, :, last], m, 128 ** -0.5)["out"], "last head")
