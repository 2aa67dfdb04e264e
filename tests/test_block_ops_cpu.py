"""CPU: refusals of the transformer-block operators, of their Python entry points and of the C ABI (no launch happens)."""
import ctypes

import pytest
import torch

from vipformer_amd import _lib as L
from vipformer_amd import build
from vipformer_amd import ops_block as O


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build(verbose=False)


def refuses(match, fn, *a, **k):
    with pytest.raises(L.VpfError, match=match):
        fn(*a, **k)


def test_structs_match_the_library():
    for which, cls in ((8, L.Rotary), (9, L.GatedNorm)):
        assert L.lib().vpf_abi_sizeof(which) == ctypes.sizeof(cls), cls.__name__


def test_packed_argument_structs_have_the_c_layout():
    """L.packer builds what ctypes builds, field for field."""
    for cls in (L.Rotary, L.GatedNorm, L.WindowAttn):
        values = [float(i) / 8 if t is L.F else 3 + 7 * i for i, (_, t) in enumerate(cls._fields_)]
        raw = L.packer(cls).pack(*values)
        assert len(raw) == ctypes.sizeof(cls)
        back = cls.from_buffer_copy(raw)
        assert [getattr(back, n) for n, _ in cls._fields_] == values, cls.__name__


def test_rotary_refusals():
    plan = O.RotaryAxes((8, 8), 32)
    q, k, pos = torch.zeros(2, 5, 4, 32), torch.zeros(2, 5, 2, 32), torch.zeros(5, 2)
    refuses("no CPU fallback", O.rotary_axes, q, k, pos, plan)
    refuses("head_dim", O.rotary_axes, q[0], k, pos, plan)
    refuses("head_dim", O.rotary_axes, q, k[:, :4], pos, plan)
    refuses("built for 32", O.rotary_axes, q[..., :16], k[..., :16], pos, plan)
    refuses("one type", O.rotary_axes, q, k.half(), pos, plan)
    refuses("one type", O.rotary_axes, q.double(), k.double(), pos, plan)
    refuses("positions", O.rotary_axes, q, k, torch.zeros(5, 3), plan)
    refuses("positions", O.rotary_axes, q, k, torch.zeros(4, 2), plan)
    refuses("positions", O.rotary_axes, q, k, torch.zeros(3, 5, 2), plan)
    refuses("positions are", O.rotary_axes, q, k, pos.half(), plan)
    refuses("no gradient", O.rotary_axes, q, k, pos.clone().requires_grad_(), plan)
    for bad in (dict(sections=(20,), head_dim=32), dict(sections=(), head_dim=32), dict(sections=(0, 0), head_dim=32), dict(sections=(-1, 4), head_dim=32),
                dict(sections=(4,), head_dim=33), dict(sections=(4,), head_dim=2048), dict(sections=(1,) * 9, head_dim=32),
                dict(sections=(4,), head_dim=32, base=0.0), dict(sections=(4,), head_dim=32, base=float("inf")),
                dict(sections=(4,), head_dim=32, layout="odd"), dict(sections=(4,), head_dim=32, ladder="none")):
        refuses("RotaryAxes", O.RotaryAxes, **bad)


def test_rotary_frequencies():
    f = O.RotaryAxes((2, 1), 8, base=100.0).frequencies()
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 1.0], dtype=torch.float64), rtol=1e-15)
    f = O.RotaryAxes((2, 2), 8, base=10000.0, ladder="joint").frequencies()
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)


def test_rotary_c_abi_refusals():
    fn = L.lib().vpf_rotary_axes
    fn.argtypes, fn.restype = L.SIGS["vpf_rotary_axes"], L.I
    ok = dict(B=1, L=4, Hq=2, Hk=1, head_dim=32, P=16, axes=2, layout=0, dtype=1, pos_type=0)
    call = lambda **k: fn(ctypes.byref(L.Rotary(**{**ok, **k})), None)
    assert fn(None, None) == -5 and call() == -5                                  # null struct, null tensors
    for bad in (dict(B=-1), dict(head_dim=0), dict(P=17), dict(P=0), dict(axes=0), dict(axes=9), dict(head_dim=1026), dict(Hq=5000)):
        assert call(**bad) == -1, bad
    for bad in (dict(layout=2), dict(dtype=3), dict(dtype=-1), dict(pos_type=4)):
        assert call(**bad) == -3, bad
    assert call(L=0) == 0                                                         # nothing to do
    assert call(layout=1, q=2, k=4, oq=4, ok=4, pos=4, freq=8, axis=4) == -2      # pairs of 16-bit channels at an odd address


def test_gated_norm_refusals():
    x, y, w = torch.zeros(2, 5, 32), torch.zeros(2, 5, 32, dtype=torch.float16), torch.ones(32)
    f = O.gated_norm_residual
    refuses("no CPU fallback", f, x, y)
    refuses("one shape", f, x, y[:, :4])
    refuses("one shape", f, torch.zeros(2, 9000), torch.zeros(2, 9000))
    refuses("one shape", f, torch.zeros(2, 0), torch.zeros(2, 0))
    refuses("x is fp32", f, x.half(), y.float())
    refuses("x is fp32", f, x.half(), y.bfloat16())
    refuses("x is fp32", f, x.double(), y)
    refuses("kind", f, x, y, kind="batch")
    for gate in (torch.zeros(31), torch.zeros(2, 32), torch.zeros(3, 1, 32), torch.zeros(2, 5, 32), torch.zeros(5, 32)):
        refuses("gate", f, x, y, gate=gate)
    refuses("is fp32", f, x, y, gate=torch.zeros(32, dtype=torch.float16))
    refuses("fp32 parameters", f, x, y, post=(w.half(), None))
    refuses("fp32 parameters", f, x, y, pre=(w, w[:31]))
    refuses("norm module or", f, x, y, pre=(w,))
    refuses("LayerNorm", f, x, y, pre=torch.nn.LayerNorm(31))
    refuses("LayerNorm", f, x, y, pre=torch.nn.RMSNorm(32))
    refuses("RMSNorm", f, x, y, post=torch.nn.LayerNorm(32), kind="rms")


def test_gated_norm_c_abi_refusals():
    fwd, bwd, ws = L.lib().vpf_gated_norm_fwd, L.lib().vpf_gated_norm_bwd, L.lib().vpf_gated_norm_ws
    fwd.argtypes = bwd.argtypes = L.SIGS["vpf_gated_norm_fwd"]
    ws.restype = L.L_
    ok = dict(rows=6, gate_rows=3, D=32, kind=0, x_type=0, y_type=1, gate_mode=0, has_post=1, has_pre=1)
    make = lambda **k: L.GatedNorm(**{**ok, **k})
    for fn in (fwd, bwd):
        assert fn(None, None) == -5 and fn(ctypes.byref(make()), None) == -5
        for bad in (dict(rows=-1), dict(rows=1 << 31), dict(D=0), dict(D=8193), dict(kind=2), dict(gate_mode=1, gate_rows=4), dict(gate_mode=1, gate_rows=0)):
            assert fn(ctypes.byref(make(**bad)), None) == -1, bad
        for bad in (dict(gate_mode=3), dict(x_type=3), dict(y_type=-1), dict(x_type=1, y_type=0), dict(x_type=2, y_type=1)):
            assert fn(ctypes.byref(make(**bad)), None) == -3, bad
        assert fn(ctypes.byref(make(rows=0)), None) == 0
    assert ws(ctypes.byref(make(rows=0))) == 0 and ws(ctypes.byref(make(D=0))) == -1
    need = ws(ctypes.byref(make(gate_mode=1)))
    assert need >= (4 + 2) * 32
    # a workspace that is too small is refused before anything is launched
    small = make(gate_mode=1, x=16, y=16, gate=16, dh=16, dn=16, stats=16, ws=16, ws_floats=need - 1)
    assert bwd(ctypes.byref(small), None) == -1


def test_window_attention_refusals():
    assert L.lib().vpf_abi_sizeof(10) == ctypes.sizeof(L.WindowAttn)
    H = torch.float16
    q, k = torch.zeros(2, 5, 4, 32, dtype=H), torch.zeros(2, 9, 2, 32, dtype=H)
    f = O.window_attention
    refuses("no CPU fallback", f, q, k, k)
    for a, b, c in ((q[0], k, k), (q, k, k[:, :8]), (q[:1], k, k), (q[..., :16], k, k), (q[:, :, :3], k, k), (q, k[:, :, :0], k[:, :, :0])):
        refuses("key heads dividing heads", f, a, b, c)
    refuses("all fp16 or all bf16", f, q.float(), k.float(), k.float())
    refuses("all fp16 or all bf16", f, q, k.bfloat16(), k)
    for dh in (4, 20, 136):
        t = torch.zeros(1, 3, 1, dh, dtype=H)
        refuses("multiple of 8", f, t, t, t)
    for w in ((-1, 0), (0, -2), (1.5, 0), (True, 0)):
        refuses("side of the window", f, q, k, k, w)
    for s in (-1, 1.0, True):
        refuses("sinks", f, q, k, k, sinks=s)
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refuses("scale", f, q, k, k, scale=s)
    refuses("pad_mask", f, q, k, k, pad_mask=torch.zeros(2, 9))
    refuses("pad_mask", f, q, k, k, pad_mask=torch.zeros(2, 5, dtype=torch.bool))
    refuses("kv_lens", f, q, k, k, kv_lens=torch.zeros(2))
    refuses("kv_lens", f, q, k, k, kv_lens=torch.zeros(3, dtype=torch.int32))
    many = torch.zeros(1, 1, 1, 8, dtype=H).expand(1, 1 << 17, 128, 8)
    refuses("index range", f, many, torch.zeros(1, 9, 1, 8, dtype=H), torch.zeros(1, 9, 1, 8, dtype=H))


def test_window_attention_c_abi_refusals():
    fwd, bwd, ws = L.lib().vpf_window_attn_fwd, L.lib().vpf_window_attn_bwd, L.lib().vpf_window_attn_ws
    fwd.argtypes = bwd.argtypes = L.SIGS["vpf_window_attn_fwd"]
    ws.restype = L.L_
    ok = dict(B=2, Lq=5, Lkv=9, Hq=4, Hk=2, head_dim=32, left=3, right=0, sinks=1, dtype=1, scale=0.2)
    make = lambda **k: L.WindowAttn(**{**ok, **k})
    for fn in (fwd, bwd):
        assert fn(None, None) == -5 and fn(ctypes.byref(make()), None) == -5
        for bad in (dict(B=-1), dict(Lq=-1), dict(Lkv=1 << 30), dict(Hk=0), dict(Hk=3), dict(head_dim=4), dict(head_dim=36), dict(head_dim=136),
                    dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(Lq=1 << 29, Hq=8)):
            assert fn(ctypes.byref(make(**bad)), None) == -1, bad
        for bad in (dict(dtype=0), dict(dtype=3)):
            assert fn(ctypes.byref(make(**bad)), None) == -3, bad
        assert fn(ctypes.byref(make(B=0)), None) == 0
    full = dict(q=16, k=16, v=16, out=16, lse=16, out_lo=16, dout=16, dq=16, dk=16, dv=16, ws=16)
    assert fwd(ctypes.byref(make(**{**full, "q": 8})), None) == -2                # not 16-byte aligned
    assert fwd(ctypes.byref(make(**full, k_sl=12)), None) == -2                   # a row stride that is no multiple of 8
    assert bwd(ctypes.byref(make(**full, dv_sh=4)), None) == -2
    heads = dict(B=1, Hq=1024, Hk=1, ws_floats=1 << 30)                           # 1024 heads of one key head over 2^30 elements
    for far in (dict(q_sh=1 << 20), dict(do_sh=1 << 20)):
        assert bwd(ctypes.byref(make(**full, **heads, **far)), None) == -2
    need = ws(ctypes.byref(make()), 1)
    assert need >= 2 * 2 * 10 and ws(ctypes.byref(make(Hk=0)), 1) == -1
    assert bwd(ctypes.byref(make(**full, ws_floats=need - 1)), None) == -1        # refused before anything is launched
    step = dict(B=1, Lq=1, Lkv=65536, left=-1, sinks=0)
    need = ws(ctypes.byref(make(**step)), 0)
    assert need > 0 and fwd(ctypes.byref(make(**{**step, **full}, ws_floats=need - 1)), None) == -1
    assert fwd(ctypes.byref(make(**{**step, **full, "ws": 0})), None) == -5


def test_window_attention_copies_heads_that_lie_too_far_apart():
    t = torch.empty_strided((1, 3, 1024, 8), (1 << 30, 8, 1 << 20, 1), dtype=torch.float16, device="meta")
    assert O._attn_ready(t)[1] == (0, 8, 1 << 20) and O._attn_ready(t, 511)[1] == (0, 8, 1 << 20)
    assert O._attn_ready(t, 512)[1] == O._attn_ready(t, 1024)[1] == (0, 8 * 1024, 8)


class _Records:
    """Stands in for the library on the CPU: keeps every argument struct that would be launched; outputs stay unwritten."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(O, "_same_device", lambda *a: None)
        monkeypatch.setattr(L, "launch", lambda name, packed, dev: self.calls.append((name, packed)))
        monkeypatch.setattr(L, "scratch_floats", lambda *a: 4)

    def last(self, name, cls):
        assert self.calls[-1][0] == name
        return cls.from_buffer_copy(self.calls[-1][1])


def _packs_elsewhere(kept):
    """Saved-tensor hooks that bring every tensor back as a copy: contiguous ones (as an offload to the host does) at addresses that are not
    16-byte aligned, and dimensions in another order in memory."""
    def plain(t):
        out = torch.empty(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape).copy_(t)
        kept.append(out)
        return out

    def turned(t):
        order = list(range(t.dim()))[::-1]
        out = torch.empty([t.shape[i] for i in order], dtype=t.dtype).permute(order).copy_(t)
        kept.append(out)
        return out
    return [(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t), (lambda t: t, plain), (lambda t: t, turned)]


def test_window_attention_backward_takes_tensors_as_hooks_bring_them_back(monkeypatch):
    """Packed q / k / v slices under saved-tensor hooks: the gradient's launch gets strides of the tensors that it is handed."""
    rec, kept = _Records(monkeypatch), []
    B, Lq, H, dh = 2, 16, 6, 64
    for pack, unpack in _packs_elsewhere(kept):
        qkv = torch.zeros(B, Lq, 3, H, dh, dtype=torch.float16, requires_grad=True)
        pad, lens = torch.zeros(B, Lq, dtype=torch.bool), torch.full((B,), Lq, dtype=torch.int32)
        alive = []
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: alive.append(unpack(t)) or alive[-1]):
            out = O.window_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], (5, 0), sinks=1, pad_mask=pad, kv_lens=lens)
            out.backward(torch.zeros_like(out))
        a = rec.last("vpf_window_attn_bwd", L.WindowAttn)
        dense = (Lq * H * dh, H * dh, dh)
        for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
            assert tuple(getattr(a, f"{n}_{s}") for s in ("sb", "sl", "sh")) == dense, n
        for n in ("q", "k", "v", "out", "out_lo", "dout"):
            assert getattr(a, n) % 16 == 0, n
        assert qkv.grad.shape == qkv.shape


def test_rotary_and_gated_norm_backward_take_tensors_as_hooks_bring_them_back(monkeypatch):
    rec, kept = _Records(monkeypatch), []
    seen = {}
    run = O._rotary_run
    monkeypatch.setattr(O, "_rotary_run", lambda plan, pos, q, k, inverse: seen.update(pos=pos) or run(plan, pos, q, k, inverse))
    for pack, unpack in _packs_elsewhere(kept):
        hooks = torch.autograd.graph.saved_tensors_hooks(pack, unpack)
        q, plan, pos = torch.zeros(2, 5, 4, 32, requires_grad=True), O.RotaryAxes((8, 8), 32), torch.rand(2, 5, 2)
        with hooks:
            O.rotary_axes(q, None, pos, plan).sum().backward()
        assert rec.last("vpf_rotary_axes", L.Rotary).inverse == 1
        assert seen["pos"].is_contiguous() and torch.equal(seen["pos"], pos)
        x, w = torch.randn(3, 5, 32, requires_grad=True), torch.randn(32, requires_grad=True)
        gate = torch.randn(3, 1, 32, requires_grad=True)
        dense = []
        ready = O._dense
        monkeypatch.setattr(O, "_dense", lambda t: dense.append(ready(t)) or dense[-1])
        with hooks:
            h, n = O.gated_norm_residual(x, x.detach() + 1, gate=gate, post=(w, None), pre=(w, w))
            torch.autograd.grad((h, n), (x, gate, w), (h.detach(), n.detach()))
        monkeypatch.setattr(O, "_dense", ready)
        a = rec.last("vpf_gated_norm_bwd", L.GatedNorm)
        assert len(dense) == 8 and [a.x, a.y, a.gate, a.stats, a.w_post, a.b_post, a.w_pre, a.b_pre] == [t if t is None else t.data_ptr() for t in dense]
        assert all(t is None or t.is_contiguous() for t in dense)
        assert torch.equal(dense[0], x) and torch.equal(dense[2], gate)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A tangent that would be dropped raises as it does for every Function without a forward-mode rule, also where no gradient is recorded."""
    from torch.autograd import forward_ad
    rec = _Records(monkeypatch)
    q, x, w, pos = torch.zeros(1, 4, 2, 32, dtype=torch.float16), torch.ones(2, 3, 32), torch.ones(32), torch.zeros(4, 2)
    plan = O.RotaryAxes((8, 8), 32)
    calls = {
        "rotary q": lambda d: O.rotary_axes(d(q), q, pos, plan), "rotary k": lambda d: O.rotary_axes(q, d(q), pos, plan),
        "rotary positions": lambda d: O.rotary_axes(q, q, d(pos), plan),
        "attention q": lambda d: O.window_attention(d(q), q, q), "attention k": lambda d: O.window_attention(q, d(q), q),
        "attention v": lambda d: O.window_attention(q, q, d(q)),
        "norm x": lambda d: O.gated_norm_residual(d(x), x), "norm y": lambda d: O.gated_norm_residual(x, d(x), pre=(None, None)),
        "norm gate": lambda d: O.gated_norm_residual(x, x, gate=d(w)), "norm weight": lambda d: O.gated_norm_residual(x, x, post=(d(w), None)),
    }
    for name, call in calls.items():
        for context in (torch.enable_grad, torch.no_grad):
            with forward_ad.dual_level(), context():
                with pytest.raises(NotImplementedError, match="forward mode"):
                    call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
                n = len(rec.calls)
                call(lambda t: t)                                              # no tangent among the inputs: as ever
                assert len(rec.calls) == n + 1, name


@pytest.mark.parametrize("x,y", [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_modules_without_an_epsilon_get_the_one_of_fp32(monkeypatch, x, y):
    """torch.nn.RMSNorm's default; its own outputs in 16 bits bear out that it is fp32's."""
    rec, rms = _Records(monkeypatch), torch.nn.RMSNorm(32, elementwise_affine=False)
    O.gated_norm_residual(torch.zeros(2, 32, dtype=x), torch.zeros(2, 32, dtype=y), post=rms, pre=rms, kind="rms")
    a = rec.last("vpf_gated_norm_fwd", L.GatedNorm)
    eps = torch.finfo(torch.float32).eps
    assert a.eps_post == a.eps_pre == eps
    z = (torch.randn(8, 32) * 0.01).to(y)
    ref = z.double() * torch.rsqrt((z.double() ** 2).mean(-1, keepdim=True) + eps)
    # half a step of the output and 32 fp32 roundings of terms of one sign, each at most 2^-24
    assert ((rms(z).double() - ref).abs() <= ref.abs() * (torch.finfo(y).eps / 2 + 32 * 2.0 ** -24)).all()


def test_a_gate_parameter_that_is_not_contiguous_is_a_parameter(monkeypatch):
    """Its gradient leaves an internal gradient scale like any other parameter's, though the kernel works on a copy of it."""
    from vipformer_amd import ops
    _Records(monkeypatch)
    monkeypatch.setattr(torch, "empty_like", torch.ones_like)                   # (the kernels write nothing here: every gradient reads 1)
    x = torch.ones(4, 32, requires_grad=True)
    for make, want in ((lambda t: torch.nn.Parameter(t), 0.25), (lambda t: t.requires_grad_(), 1.0)):
        for gate in (make(torch.ones(32)), make(torch.ones(64)[::2]), make(torch.ones(32, 4).t()), make(torch.ones(4, 32))):
            with ops.internal_grad_scale() as holder:
                h, _ = O.gated_norm_residual(x, x.detach(), gate=gate)
            if holder.on:
                holder.inv = torch.tensor(0.25)
            (dgate,) = torch.autograd.grad(h, (gate,), torch.ones(4, 32))
            assert dgate.shape == gate.shape and torch.equal(dgate, torch.full_like(dgate, want if holder.on else 1.0)), gate.stride()


def test_saved_tensors_that_come_back_as_something_else_are_refused(monkeypatch):
    """Hooks that bring back another type, shape or device: the kernels would read something else, or behind its end."""
    rec = _Records(monkeypatch)
    q, x, w, plan = torch.zeros(1, 4, 2, 32, dtype=torch.float16), torch.ones(2, 3, 32), torch.ones(32), O.RotaryAxes((8, 8), 32)
    q.requires_grad_(), x.requires_grad_()
    calls = {"rotary_axes": (q, lambda: O.rotary_axes(q, None, torch.zeros(4, 2), plan)),
             "window_attention": (q, lambda: O.window_attention(q, q.detach(), q.detach(), kv_lens=torch.tensor([4]))),
             "gated_norm_residual": (x, lambda: O.gated_norm_residual(x, x.detach(), post=(w, None))[0])}
    for what, (leaf, call) in calls.items():
        for unpack in (lambda t: t.double(), lambda t: t[..., :-1], lambda t: t.flatten(), lambda t: t.to("meta")):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                out = call()
                n = len(rec.calls)
                refuses(f"{what}: a saved tensor came back", torch.autograd.grad, out, (leaf,), torch.zeros_like(out))
                assert len(rec.calls) == n, what


def test_window_attention_takes_long_caches_with_the_heads_first_as_they_are():
    """[B, heads, tokens, head_dim] caches of more than 65536 tokens: where a head begins is no offset inside a stage."""
    cache = torch.empty(2, 4, 70000, 128, dtype=torch.bfloat16, device="meta").transpose(1, 2)
    t, strides = O._attn_ready(cache)
    assert t is cache and strides == (4 * 70000 * 128, 128, 70000 * 128)
    rows = torch.empty_strided((1, 3, 2, 8), (0, 1 << 23, 8, 1), dtype=torch.float16, device="meta")
    assert O._attn_ready(rows)[1] == (0, 16, 8)                                 # tokens are
    fwd = L.lib().vpf_window_attn_fwd
    fwd.argtypes = L.SIGS["vpf_window_attn_fwd"]
    args = dict(B=1, Lq=1, Lkv=70000, Hq=4, Hk=4, head_dim=128, left=-1, right=0, dtype=2, scale=0.1, q=16, k=16, v=16, out=16, k_sl=128, v_sl=128)
    assert fwd(ctypes.byref(L.WindowAttn(**args, k_sh=1 << 40, v_sh=1 << 40)), None) == -5      # (no scratch: nothing is launched)
    assert fwd(ctypes.byref(L.WindowAttn(**{**args, "k_sl": 1 << 23})), None) == -2
