"""Measured cases of the transformer-block operators in ``vipformer_amd.ops_block``.

Three operators that one encoder block over a long token sequence (image patches, point groups, video patches) uses together:

  rotary    rotary positions with several axes on the queries and keys               ops_block.rotary_axes
  attention attention inside a sliding window with first tokens that stay visible    ops_block.window_attention
  norm      norm behind a block, its gate and residual scale, norm before the next   ops_block.gated_norm_residual

``own = False`` computes the plain form with elementary torch operations in 32 bits (64 for the rotary angles); ``own = True`` calls the
framework.  A case with ``train`` returns the outputs and every gradient.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, B, Lq, Lkv, Hq, Hk, dh, left, right, sinks, dtype, train=False, pad=False, lens=False, packed=False):
    return dict(name=name, op="attention", B=B, Lq=Lq, Lkv=Lkv, Hq=Hq, Hk=Hk, dh=dh, left=left, right=right, sinks=sinks, dtype=dtype,
                train=train, pad=pad, lens=lens, packed=packed)


def _rotary(name, B, L, Hq, Hk, dh, axes, layout, dtype, train=False, per_sample=False, far=0, packed=False):
    return dict(name=name, op="rotary", B=B, L=L, Hq=Hq, Hk=Hk, dh=dh, axes=axes, layout=layout, dtype=dtype, train=train,
                per_sample=per_sample, far=far, packed=packed)


def _norm(name, B, L, D, kind, gate, x, y, post=True, pre=True, train=False):
    return dict(name=name, op="norm", B=B, L=L, D=D, kind=kind, gate=gate, x=x, y=y, post=post, pre=pre, train=train)


def listed():
    return [
        # One point cloud's 96 group tokens through the small encoder (4 heads of 64): what a single sample waits for.
        _attention("attention_small", 1, 96, 96, 4, 4, 64, 24, 24, 1, "fp16"),
        # One new token for each of 8 sequences over a preallocated cache that is full to different lengths; shared key heads.
        _attention("attention_step", 8, 1, 16384, 16, 4, 128, 4095, 0, 4, "bf16", lens=True),
        # Training on 16 images of 32 x 32 patches and one class token that everything sees; q, k, v are slices of one projection.
        _attention("attention_image_train", 16, 1025, 1025, 6, 6, 64, 128, 128, 1, "fp16", train=True, packed=True),
        # Training on point sequences of different lengths (padded batch), shared key heads, a head width that fills no tile.
        _attention("attention_points_train", 5, 777, 777, 6, 2, 80, 100, 60, 5, "bf16", train=True, pad=True),
        # A long causal sequence of video patches, forward only.
        _attention("attention_video", 1, 32768, 32768, 16, 4, 128, 4095, 0, 4, "bf16"),
        # Training on a long causal sequence.
        _attention("attention_video_train", 1, 8192, 8192, 16, 4, 128, 2047, 0, 4, "bf16", train=True),
        # Training on 64 clouds of 1024 point tokens with their coordinates as three axes of positions.
        _rotary("rotary_points_train", 64, 1024, 6, 6, 64, 3, "half", "fp16", train=True, per_sample=True, packed=True),
        # A video of time x height x width patches far into a stream, an odd token count.
        _rotary("rotary_video", 1, 32769, 16, 4, 128, 3, "pair", "bf16", far=1000000),
        # One sample's 96 tokens between two blocks of the small encoder.
        _norm("norm_small", 1, 96, 256, "layer", "channel", "f32", "fp16"),
        # The pre-training batch: 128 clouds of 128 tokens, fp32 residual stream, half-precision branch, one gate per channel.
        _norm("norm_points_train", 128, 128, 256, "layer", "channel", "f32", "fp16", train=True),
        # A wide model on long sequences, everything in bf16, one gate vector per sample.
        _norm("norm_wide_train", 16, 2048, 2048, "rms", "sample", "bf16", "bf16", train=True),
        # Odd rows and width in fp32 with a gate for every token.
        _norm("norm_odd_train", 3, 333, 1001, "layer", "token", "f32", "f32", train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_attention(rng):
    g = rng.choice([1, 1, 2, 3, 4])
    Hk = rng.choice([1, 2, 4, 6])
    dh = rng.choice([32, 40, 64, 64, 80, 96, 128])
    dtype = rng.choice(["fp16", "bf16"])
    kind = rng.choice(["step", "forward", "train", "train"])
    sinks = rng.choice([0, 1, 4, 5, 70])
    if kind == "step":
        Lkv = _log(rng, 64, 65536)
        return _attention("", _log(rng, 1, 16), rng.choice([1, 1, 2, 5]), Lkv, Hk * g, Hk, dh, _log(rng, 16, Lkv), 0, sinks, dtype, lens=True)
    L = _log(rng, 1, 32768 if kind == "forward" else 8192)
    left = _log(rng, 1, 4095)
    right = rng.choice([0, left])
    pad = rng.random() < 0.3
    return _attention("", _log(rng, 1, 32), L, L, Hk * g, Hk, dh, left, right, sinks, dtype, train=kind == "train", pad=pad,
                      packed=g == 1 and rng.random() < 0.5)


def _draw_rotary(rng):
    g = rng.choice([1, 2, 4])
    Hk = rng.choice([1, 2, 4, 6])
    return _rotary("", _log(rng, 1, 64), _log(rng, 1, 32769), Hk * g, Hk, rng.choice([32, 40, 64, 80, 128]), rng.choice([1, 2, 3]),
                   rng.choice(["half", "pair"]), rng.choice(["fp16", "bf16", "f32"]), train=rng.random() < 0.5, per_sample=rng.random() < 0.5,
                   far=rng.choice([0, 0, 1000000]), packed=g == 1 and rng.random() < 0.5)


def _draw_norm(rng):
    x, y = rng.choice([("f32", "fp16"), ("f32", "fp16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("fp16", "fp16")])
    D = rng.choice([_log(rng, 8, 8192), 8 * _log(rng, 1, 1024), 256 * rng.randint(1, 4)])
    post, pre = rng.choice([(True, True), (True, True), (True, False), (False, True)])
    return _norm("", _log(rng, 1, 128), _log(rng, 1, 4096), D, rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "sample", "token"]),
                 x, y, post, pre, train=rng.random() < 0.6)


_TOP = {}


def draw(rng):
    """One more case of the ranges that the listed ones stand for: lengths from one token to the longest, whole and odd sizes."""
    if not _TOP:
        for c in listed():
            w = work(c)
            t = _TOP.setdefault(c["op"], {"bytes": 0, "flops": 0, "dense": 0})
            t["bytes"], t["flops"] = max(t["bytes"], w["bytes"]), max(t["flops"], w["flops"])
            t["dense"] = max(t["dense"], _dense(c))
    while True:
        op = rng.choice(["attention", "attention", "rotary", "norm"])
        case = {"attention": _draw_attention, "rotary": _draw_rotary, "norm": _draw_norm}[op](rng)
        w, top = work(case), _TOP[op]
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and _dense(case) <= top["dense"]:
            del case["name"]
            return case


def _dense(case):
    """Scores that the plain form of an attention case computes."""
    if case["op"] != "attention":
        return 0
    keys = min(case["Lkv"], case["left"] + case["right"] + case["sinks"] + 1 + _rows(case))
    return case["B"] * case["Hq"] * case["Lq"] * keys * (3 if case["train"] else 1)


# ------------------------------------------------------------------------------------------------ what a case cannot do without
def _case_lens(case):
    """Keys in use of every sample: a spread of fills of the cache, or of lengths of a padded batch."""
    B, Lkv = case["B"], case["Lkv"]
    if not (case["lens"] or case["pad"]):
        return [Lkv] * B
    return [max(1, Lkv - (b * 5 * Lkv) // (8 * B)) for b in range(B)]


def _visible(case):
    """(query, key) pairs inside the mask, and keys that at least one query of their sample sees, over the batch."""
    pairs = keys = 0
    for n in _case_lens(case):
        Lq, left, right, sinks = case["Lq"], case["left"], case["right"], case["sinks"]
        at = (n if case["lens"] else case["Lkv"]) - Lq
        i = torch.arange(at, at + Lq, dtype=torch.float64)
        hi = torch.clamp(i + right + 1, 0, n)
        lo = torch.clamp(i - left, 0, n)
        lo = torch.minimum(lo, hi)
        s = torch.clamp(torch.minimum(torch.full_like(i, float(min(sinks, n))), lo), min=0)
        s = torch.minimum(s, hi)
        pairs += int((hi - lo + s).sum())
        first = int(lo.min())
        keys += max(0, int(hi.max()) - first) + min(first, sinks, n)
    return pairs, keys


def work(case):
    if case["op"] == "attention":
        e, dh = 2, case["dh"]
        pairs, keys = _visible(case)
        q = case["B"] * case["Lq"] * case["Hq"] * dh
        kv = keys * case["Hk"] * dh
        all_kv = case["B"] * case["Lkv"] * case["Hk"] * dh
        flops = 4 * dh * pairs * case["Hq"]
        byts = e * (2 * q + 2 * kv)
        if case["train"]:                                   # + dout in; dq, dk, dv out (dk, dv whole)
            flops += 10 * dh * pairs * case["Hq"]
            byts += e * (2 * q + 2 * all_kv)
        return {"bytes": byts, "flops": flops}
    if case["op"] == "rotary":
        e = 4 if case["dtype"] == "f32" else 2
        n = case["B"] * case["L"] * (case["Hq"] + case["Hk"]) * case["dh"]
        k = 2 if case["train"] else 1                       # the gradient is the same pass over the outputs' gradients
        pos = case["L"] * case["axes"] * 4 * (case["B"] if case["per_sample"] else 1)
        return {"bytes": 2 * e * n * k + pos, "flops": 3 * n * k}
    ex, ey = (4 if case[t] == "f32" else 2 for t in ("x", "y"))
    n = case["B"] * case["L"] * case["D"]
    gate = {"none": 0, "channel": 4 * case["D"], "sample": 4 * case["B"] * case["D"], "token": ey * n}[case["gate"]]
    byts = n * (ex + ey + ex + (ey if case["pre"] else 0)) + gate
    flops = n * 16
    if case["train"]:                                       # dh, dn in; dx, dy out (and the gate's gradient)
        byts += n * (ex + (ey if case["pre"] else 0) + ex + ey) + gate
        flops += n * 30
    return {"bytes": byts, "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _heads(g, case, L, heads, dtype):
    """[B, L, heads, dh] for every entry of ``heads``: slices of one projection's output, or tensors of their own."""
    B, dh = case["B"], case["dh"]
    if not case["packed"]:
        return [_randn(g, (B, n, h, dh), dtype) for n, h in zip(L, heads)]
    buf = _randn(g, (B, L[0], sum(heads), dh), dtype)
    return [t.detach() for t in buf.split(heads, dim=2)]


def _sections(case):
    """Pairs of channels of each axis: even shares of half the head, what is left goes to the first axes."""
    P, A = case["dh"] // 2, case["axes"]
    return tuple(P // A + (1 if a < P % A else 0) for a in range(A))


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "attention":
        dt = DTYPES[case["dtype"]]
        q, k, v = _heads(g, case, (case["Lq"], case["Lkv"], case["Lkv"]), (case["Hq"], case["Hk"], case["Hk"]), dt)
        lens = _case_lens(case)
        s = dict(case=case, q=q, k=k, v=v, host_lens=lens, pad=None, lens=None)
        ends = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if case["pad"]:
            s["pad"] = torch.arange(case["Lkv"], device="cuda")[None, :] >= ends[:, None]
        if case["lens"]:
            s["lens"] = ends
        if case["train"]:
            for t in ("q", "k", "v"):
                s[t].requires_grad_()
            s["dout"] = _randn(g, (case["B"], case["Lq"], case["Hq"], case["dh"]), dt)
        return s
    if case["op"] == "rotary":
        dt = DTYPES[case["dtype"]]
        q, k = _heads(g, case, (case["L"],) * 2, (case["Hq"], case["Hk"]), dt)
        lead = (case["B"], case["L"]) if case["per_sample"] else (case["L"],)
        if case["far"]:                                     # patch indices, the first axis far into a stream
            top = torch.tensor([64] * case["axes"], device="cuda")
            pos = (torch.rand(lead + (case["axes"],), generator=g, device="cuda") * top).long()
            pos[..., 0] += case["far"]
            pos = pos.int()
        else:                                               # coordinates
            pos = torch.rand(lead + (case["axes"],), generator=g, device="cuda") * 64.0
        s = dict(case=case, q=q, k=k, pos=pos)
        if own:
            from vipformer_amd.ops_block import RotaryAxes
            s["plan"] = RotaryAxes(_sections(case), case["dh"], layout=case["layout"])
        if case["train"]:
            q.requires_grad_()
            k.requires_grad_()
            s["dq"], s["dk"] = _randn(g, q.shape, dt), _randn(g, k.shape, dt)
        return s
    tx, ty = DTYPES[case["x"]], DTYPES[case["y"]]
    B, L, D = case["B"], case["L"], case["D"]
    s = dict(case=case, x=_randn(g, (B, L, D), tx, 2.0), y=_randn(g, (B, L, D), ty, 0.7))
    affine = lambda: (1.0 + _randn(g, (D,), torch.float32, 0.2), _randn(g, (D,), torch.float32, 0.2))
    wp, bp = affine()
    wn, bn = affine()
    rms = case["kind"] == "rms"
    s["post"] = (wp, None if rms else bp) if case["post"] else None
    s["pre"] = (wn, None if rms else bn) if case["pre"] else None
    shape = {"none": None, "channel": (D,), "sample": (B, 1, D), "token": (B, L, D)}[case["gate"]]
    s["gate"] = None if shape is None else _randn(g, shape, ty if case["gate"] == "token" else torch.float32, 0.5)
    s["leaves"] = [t for t in (s["x"], s["y"], s["gate"]) + (s["post"] or ()) + (s["pre"] or ()) if t is not None]
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_()
        s["dh"] = _randn(g, (B, L, D), tx)
        s["dn"] = _randn(g, (B, L, D), ty) if case["pre"] else None
    return s


ALPHA, BETA, EPS = 0.9, 0.75, 1e-5          # scales of the residual stream and of the branch, the norms' epsilon


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else {"attention": _plain_attention, "rotary": _plain_rotary, "norm": _plain_norm}[state["case"]["op"]](state)


def _run_own(s):
    from vipformer_amd import ops_block
    c = s["case"]
    if c["op"] == "attention":
        out = ops_block.window_attention(s["q"], s["k"], s["v"], (c["left"], c["right"]), sinks=c["sinks"], pad_mask=s["pad"], kv_lens=s["lens"])
        if not c["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]
    if c["op"] == "rotary":
        q, k = ops_block.rotary_axes(s["q"], s["k"], s["pos"], s["plan"])
        if not c["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    h, n = ops_block.gated_norm_residual(s["x"], s["y"], gate=s["gate"], post=s["post"], pre=s["pre"], kind=c["kind"], alpha=ALPHA, beta=BETA,
                                         eps=EPS)
    outs = [h] if n is None else [h, n]
    if not c["train"]:
        return outs
    grads = torch.autograd.grad(outs, s["leaves"], [s["dh"]] if n is None else [s["dh"], s["dn"]])
    return [t.detach() for t in outs] + list(grads)


# ------------------------------------------------------------------------------------------------ the plain forms
def _rows(case):
    """Queries of one block of the plain form: its scores stay near 2^28 numbers."""
    per = case["B"] * case["Hq"] * min(case["Lkv"], case["left"] + case["right"] + case["sinks"] + 1025)
    return max(1, min(case["Lq"], (1 << 28) // per, 1024))


def _plain_blocks(s):
    """(rows, key index, hidden) of every block of queries: the keys that its window and the first tokens can reach."""
    c = s["case"]
    Lq, Lkv, left, right, sinks = (c[t] for t in ("Lq", "Lkv", "left", "right", "sinks"))
    at = [(n if c["lens"] else Lkv) - Lq for n in s["host_lens"]]
    end = s["lens"].long() if c["lens"] else torch.full((c["B"],), Lkv, device="cuda")
    step = _rows(c)
    for r0 in range(0, Lq, step):
        r1 = min(Lq, r0 + step)
        lo = min(max(0, min(at) + r0 - left), Lkv)
        hi = min(max(0, max(at) + r1 + right), Lkv)
        first = min(sinks, lo, hi)
        j = torch.cat([torch.arange(first, device="cuda"), torch.arange(lo, max(lo, hi), device="cuda")])
        pos = (end - Lq)[:, None, None] + torch.arange(r0, r1, device="cuda")[None, :, None]
        seen = (j <= pos + right) & ((j >= pos - left) | (j < sinks)) & (j < end[:, None, None])
        if s["pad"] is not None:
            seen = seen & ~s["pad"][:, j][:, None, :]
        yield r0, r1, j, ~seen


def _plain_attention(s):
    c = s["case"]
    B, Lq, Lkv, Hq, Hk, dh = (c[t] for t in ("B", "Lq", "Lkv", "Hq", "Hk", "dh"))
    g, scale, dt = Hq // Hk, 1.0 / math.sqrt(dh), s["q"].dtype
    with torch.no_grad():
        q = s["q"].float().view(B, Lq, Hk, g, dh).permute(0, 2, 1, 3, 4)              # [B, Hk, Lq, g, dh]
        k, v = (s[t].float().transpose(1, 2).contiguous() for t in ("k", "v"))        # [B, Hk, Lkv, dh]
        out = torch.empty(B, Lq, Hq, dh, dtype=dt, device="cuda")
        if c["train"]:
            dout = s["dout"].float().view(B, Lq, Hk, g, dh).permute(0, 2, 1, 3, 4)
            dq, dk, dv = torch.empty(B, Lq, Hq, dh, dtype=dt, device="cuda"), torch.zeros_like(k), torch.zeros_like(v)
        back = lambda t, n: t.view(B, Hk, n, g, dh).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, dh).to(dt)
        for r0, r1, j, hidden in _plain_blocks(s):
            n = r1 - r0
            if j.numel() == 0:
                out[:, r0:r1] = 0
                if c["train"]:
                    dq[:, r0:r1] = 0
                continue
            qb, kb, vb = q[:, :, r0:r1].reshape(B, Hk, n * g, dh), k[:, :, j], v[:, :, j]
            hide = hidden[:, None, :, None, :].expand(B, 1, n, g, j.numel()).reshape(B, 1, n * g, j.numel())
            p = torch.matmul(qb, kb.transpose(-1, -2)).mul_(scale).masked_fill_(hide, -math.inf)
            top = p.amax(-1, keepdim=True)
            p = p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
            p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
            ob = torch.matmul(p, vb)
            out[:, r0:r1] = back(ob, n)
            if c["train"]:
                db = dout[:, :, r0:r1].reshape(B, Hk, n * g, dh)
                dvb = torch.matmul(p.transpose(-1, -2), db)
                ds = torch.matmul(db, vb.transpose(-1, -2)).sub_((db * ob).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                dq[:, r0:r1] = back(torch.matmul(ds, kb), n)
                dk.index_add_(2, j, torch.matmul(ds.transpose(-1, -2), qb))
                dv.index_add_(2, j, dvb)
        if not c["train"]:
            return [out]
        return [out, dq, dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt)]


def _turns(s):
    """cos and sin of every (token, pair) in 64 bits: far positions times small frequencies lose their fraction in 32."""
    c = s["case"]
    angles = []
    for a, n in enumerate(_sections(c)):
        freq = 10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1))
        angles.append(s["pos"][..., a:a + 1].double() * freq)
    t = torch.cat(angles, -1)
    return (t if t.dim() == 3 else t[None])[:, :, None, :]                            # [B or 1, L, 1, P]


def _plain_rotary(s):
    c = s["case"]
    with torch.no_grad():
        t = _turns(s)
        cos, sin = t.cos().float(), t.sin().float()

        def turn(x, sin):
            f = x.float()
            if c["layout"] == "half":
                a, b = f.chunk(2, -1)
                return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
            a, b = f[..., 0::2], f[..., 1::2]
            return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)

        outs = [turn(s["q"], sin), turn(s["k"], sin)]
        if c["train"]:
            outs += [turn(s["dq"], -sin), turn(s["dk"], -sin)]
        return outs


def _plain_norm(s):
    c = s["case"]
    layer = c["kind"] == "layer"

    def norm(z, wb):
        if layer:
            z = z - z.mean(-1, keepdim=True)
        r = (z.square().mean(-1, keepdim=True) + EPS).rsqrt()
        zh = z * r
        n = zh * wb[0]
        return (n if wb[1] is None else n + wb[1]), zh, r

    def norm_back(dn, zh, r, w):
        d = dn * w
        out = d - zh * (d * zh).mean(-1, keepdim=True)
        if layer:
            out = out - d.mean(-1, keepdim=True)
        return out * r

    def affine_back(dn, zh, wb):
        out = [(dn * zh).sum((0, 1))]
        return out if wb[1] is None else out + [dn.sum((0, 1))]

    with torch.no_grad():
        x, y = s["x"].float(), s["y"].float()
        gate = None if s["gate"] is None else s["gate"].float()
        if c["post"]:
            u, yh, ry = norm(y, s["post"])
        else:
            u = y
        h = ALPHA * x + BETA * (u if gate is None else gate * u)
        outs = [h.to(s["x"].dtype)]
        if c["pre"]:
            n, hh, rh = norm(h, s["pre"])
            outs.append(n.to(s["y"].dtype))
        if not c["train"]:
            return outs
        d, pre_grads, post_grads = s["dh"].float(), [], []
        if c["pre"]:
            dn = s["dn"].float()
            d = d + norm_back(dn, hh, rh, s["pre"][0])
            pre_grads = affine_back(dn, hh, s["pre"])
        outs.append((ALPHA * d).to(s["x"].dtype))
        du = BETA * (d if gate is None else d * gate)
        dy = du
        if c["post"]:
            dy = norm_back(du, yh, ry, s["post"][0])
            post_grads = affine_back(du, yh, s["post"])
        outs.append(dy.to(s["y"].dtype))
        if gate is not None:
            dg = BETA * d * u
            dg = {"channel": lambda: dg.sum((0, 1)), "sample": lambda: dg.sum(1, keepdim=True), "token": lambda: dg}[c["gate"]]()
            outs.append(dg.to(s["gate"].dtype))
        return outs + post_grads + pre_grads


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions, in 64 bits, differentiated by autograd."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "rotary":
        t = _turns(s)
        turn = torch.polar(torch.ones_like(t), t)

        def rotate(x, w):
            d = x.detach().double()
            if case["layout"] == "half":
                P = case["dh"] // 2
                z = torch.complex(d[..., :P].contiguous(), d[..., P:].contiguous()) * w
                return torch.cat([z.real, z.imag], -1)
            return torch.view_as_real(torch.view_as_complex(d.reshape(d.shape[:-1] + (-1, 2)).contiguous()) * w).flatten(-2)

        outs = [rotate(s["q"], turn), rotate(s["k"], turn)]
        if case["train"]:
            outs += [rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())]
        return outs
    leaf = {id(t): t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]}
    of = lambda t: None if t is None else leaf[id(t)]

    def norm(z, wb):
        w, b = of(wb[0]), of(wb[1])
        if case["kind"] == "layer":
            var, mean = torch.var_mean(z, -1, unbiased=False, keepdim=True)
            n = (z - mean) / torch.sqrt(var + EPS) * w
        else:
            n = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * w
        return n if b is None else n + b

    u = of(s["y"])
    if case["post"]:
        u = norm(u, s["post"])
    if s["gate"] is not None:
        u = u * of(s["gate"])
    h = ALPHA * of(s["x"]) + BETA * u
    outs = [h] + ([norm(h, s["pre"])] if case["pre"] else [])
    if not case["train"]:
        return outs
    douts = [s["dh"].double()] + ([s["dn"].double()] if case["pre"] else [])
    grads = torch.autograd.grad(outs, [leaf[id(t)] for t in s["leaves"]], douts)
    return [t.detach() for t in outs] + list(grads)


def _exact_attention(s):
    c = s["case"]
    B, Lq, Lkv, Hq, Hk, dh = (c[t] for t in ("B", "Lq", "Lkv", "Hq", "Hk", "dh"))
    out = torch.zeros(B, Lq, Hq, dh, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(s[t].shape, dtype=torch.float64, device="cuda") for t in ("q", "k", "v")] if c["train"] else []
    j = torch.arange(Lkv, device="cuda")
    for b in range(B):
        end = s["host_lens"][b] if c["lens"] else Lkv
        for r0 in range(0, Lq, 1024):
            r1 = min(Lq, r0 + 1024)
            pos = (torch.arange(r0, r1, device="cuda") + (end - Lq))[:, None]
            seen = (j < end) & (j <= pos + c["right"]) & ((pos - j <= c["left"]) | (j < c["sinks"]))
            if s["pad"] is not None:
                seen = seen & torch.logical_not(s["pad"][b])
            idx = seen.any(0).nonzero()[:, 0]
            if idx.numel() == 0:
                continue
            m = seen[:, idx]
            alone = ~m.any(-1, keepdim=True)
            for h in range(Hq):
                kv = h // (Hq // Hk)
                q, k, v = (t.detach().double().requires_grad_(c["train"]) for t in (s["q"][b, r0:r1, h], s["k"][b, idx, kv], s["v"][b, idx, kv]))
                w = torch.softmax((q @ k.t() / math.sqrt(dh)).masked_fill(~m, -math.inf).masked_fill(alone, 0.0), -1).masked_fill(alone, 0.0)
                o = w @ v
                out[b, r0:r1, h] = o.detach()
                if c["train"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["dout"][b, r0:r1, h].double())
                    grads[0][b, r0:r1, h] = dq
                    grads[1][b, idx, kv] += dk
                    grads[2][b, idx, kv] += dv
    return [out] + grads
