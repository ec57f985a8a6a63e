"""The sequence operators where no GPU is needed: argument validation of the C entry points, refusals of
the Python functions, module surfaces, and the 64-bit definitions that the GPU tests compare with."""
import ctypes

import pytest
import torch

import sequence_util as ref

FAKE = 0x1000  # never dereferenced: validation fails first


def rows(ptr=FAKE):
    from dwconv_b200 import _lib
    return _lib.Rows(ptr, 64, 8)


def test_c_entry_points_validate_before_any_launch():
    from dwconv_b200 import _lib
    L, F32 = _lib.lib, _lib.F32
    s = _lib.Sequence(2, 8, 8, None, 0)
    ws = L.dwconv_b200_conv1d_causal_workspace_bytes(F32, s, 4)
    assert ws >= 5 * 8 * 4 and ws % 16 == 0

    def conv(x=None, w=FAKE, y=FAKE, dtype=F32, seq=s, taps=4, act=0, bias=None, init=None):
        return L.dwconv_b200_conv1d_causal(x or rows(), w, bias, init, y, None, dtype, seq, taps, act, None)

    assert conv(w=None) == 1 and conv(y=None) == 1 and conv(x=rows(None)) == 1
    assert conv(dtype=_lib.F64) == 2 and conv(dtype=9) == 2
    assert conv(w=FAKE + 2) == 3 and conv(x=rows(FAKE + 1)) == 3 and conv(init=FAKE + 2) == 3
    assert conv(taps=0) == 1 and conv(taps=9) == 6 and conv(act=5) == 1 and conv(act=-1) == 1
    for bad in ((0, 8, 8, None, 0), (2, -1, 8, None, 0), (2, 8, 0, None, 0), (2, 8, 8, FAKE, 3), (1, 8, 8, FAKE, 0),
                (1, 8, 8, FAKE + 2, 3)):
        assert conv(seq=_lib.Sequence(*bad)) == 1, bad
    for big in ((1, (1 << 30) + 1, 8, None, 0), (1, 8, (1 << 26) + 1, None, 0), (1 << 26, 1 << 20, 1024, None, 0)):
        assert conv(seq=_lib.Sequence(*big)) == 7, big

    def conv_bwd(ws_ptr=FAKE, nbytes=ws, dx=FAKE, dw=FAKE, dy=None):
        return L.dwconv_b200_conv1d_causal_backward(rows(), FAKE, None, None, dy or rows(), None, dx, dw, None, None,
                                                    ws_ptr, nbytes, F32, s, 4, 0, None)

    assert conv_bwd(ws_ptr=None) == 1 and conv_bwd(ws_ptr=FAKE + 8) == 3 and conv_bwd(nbytes=ws - 1) == 4
    assert conv_bwd(dx=None) == 1 and conv_bwd(dw=None) == 1 and conv_bwd(dy=rows(None)) == 1
    assert L.dwconv_b200_conv1d_causal_workspace_bytes(_lib.F64, s, 4) == 0
    assert L.dwconv_b200_conv1d_causal_step(FAKE, 8, FAKE, None, None, FAKE, F32, 2, 8, 4, 0, None) == 1
    assert L.dwconv_b200_conv1d_causal_step(FAKE, 8, FAKE, None, FAKE + 1, FAKE, F32, 2, 8, 4, 0, None) == 3

    def rec(x=None, decay=FAKE, y=FAKE, scale=8.0, dtype=F32, seq=s, ckpt=None, fin=None):
        return L.dwconv_b200_recurrence(x or rows(), rows(), rows(), decay, None, y, fin, ckpt, dtype, seq, scale, None)

    assert rec(decay=None) == 1 and rec(y=None) == 1 and rec(x=rows(None)) == 1
    assert rec(scale=0.0) == 1 and rec(scale=-1.0) == 1 and rec(scale=float("nan")) == 1
    assert rec(dtype=_lib.F64) == 2 and rec(ckpt=FAKE + 4) == 3 and rec(fin=FAKE + 2) == 3 and rec(x=rows(FAKE + 2)) == 3
    assert rec(seq=_lib.Sequence(2, 8, 0, None, 0)) == 1
    need = L.dwconv_b200_recurrence_workspace_bytes(s)
    assert need >= 2 * 8 * 4 and L.dwconv_b200_recurrence_checkpoint_bytes(s) >= 2 * 8 * 4

    def rec_bwd(ckpt=FAKE, ws_ptr=FAKE, nbytes=need, dd=FAKE):
        return L.dwconv_b200_recurrence_backward(rows(), rows(), rows(), FAKE, None, ckpt, rows(), None, FAKE, FAKE,
                                                 FAKE, dd, None, ws_ptr, nbytes, F32, s, 8.0, None)

    assert rec_bwd(ckpt=None) == 1 and rec_bwd(ws_ptr=None) == 1 and rec_bwd(nbytes=need - 1) == 4
    assert rec_bwd(dd=None) == 1 and rec_bwd(dd=FAKE + 2) == 3 and rec_bwd(ws_ptr=FAKE + 8) == 3
    assert L.dwconv_b200_recurrence_step(FAKE, 8, FAKE, 8, FAKE, 8, FAKE, None, FAKE, F32, 2, 8, 8.0, None) == 1
    assert L.dwconv_b200_recurrence_step(FAKE, 8, FAKE, 8, FAKE, 8, FAKE, FAKE, FAKE, F32, 2, 8, 0.0, None) == 1

    def norm(x=FAKE, y=FAKE, stats=None, dtype=F32, n=4, C=8, eps=1e-5):
        return L.dwconv_b200_layer_norm(x, 8, None, None, y, stats, dtype, n, C, eps, None)

    assert norm(x=None) == 1 and norm(y=None) == 1 and norm(eps=-1.0) == 1 and norm(C=0) == 1 and norm(n=-1) == 1
    assert norm(dtype=_lib.F64) == 2 and norm(x=FAKE + 2) == 3 and norm(stats=FAKE + 4) == 3
    assert norm(C=(1 << 26) + 1) == 7 and norm(n=0) == 0
    nb = L.dwconv_b200_layer_norm_workspace_bytes(F32, 4, 8)

    def norm_bwd(stats=FAKE, dx=FAKE, dw=FAKE, ws_ptr=FAKE, nbytes=nb):
        return L.dwconv_b200_layer_norm_backward(FAKE, 8, None, stats, FAKE, 8, dx, dw, None, ws_ptr, nbytes, F32, 4, 8,
                                                 None)

    assert norm_bwd(stats=None) == 1 and norm_bwd(dx=None) == 1 and norm_bwd(ws_ptr=None) == 1
    assert norm_bwd(nbytes=nb - 1) == 4 and norm_bwd(ws_ptr=FAKE + 8) == 3 and norm_bwd(stats=FAKE + 4) == 3


def test_cpu_tensors_and_unknown_activations_are_refused():
    import dwconv_b200 as d
    from dwconv_b200 import sequence as S
    x, w, v = torch.zeros(1, 4, 8), torch.zeros(8, 1, 4), torch.zeros(8)
    for call in (lambda: d.depthwise_conv1d_causal(x, w), lambda: d.gated_linear_recurrence(x, x, x, v),
                 lambda: d.layer_norm(x, v, v), lambda: d.depthwise_conv1d_causal_step(x[0], w, torch.zeros(4, 3, 8)),
                 lambda: d.gated_linear_recurrence_step(x[0], x[0], x[0], v, torch.zeros(4, 8))):
        with pytest.raises(RuntimeError, match="input must be a CUDA tensor"):
            call()
    for name, args in (("conv1d_causal", (x, w, None, 0, None, None, False)), ("layer_norm", (x, v, v, 1e-5, False)),
                       ("recurrence", (x, x, x, v, None, None, 8.0, False, False))):
        with pytest.raises(RuntimeError, match="input must be a CUDA tensor"):
            S.CTYPES_FORMS[name](*args)
    with pytest.raises(ValueError, match="unknown activation"):
        d.depthwise_conv1d_causal(x, w, activation="tanh")
    with pytest.raises(ValueError, match="unknown activation"):
        d.CausalDepthwiseConv1d(8, 4, activation="tanh")
    with pytest.raises(ValueError, match="1 to 8 taps"):
        d.CausalDepthwiseConv1d(8, 9)
    with pytest.raises(ValueError, match="0 < low"):
        d.GatedLinearRecurrence(8, low=0.0)


def test_forward_mode_derivatives_are_refused():
    """A tangent would be lost without a word: every function refuses it, compiled or not."""
    import dwconv_b200 as d
    import dwconv_b200.sequence as seq
    x, w, vec = torch.ones(1, 4, 2), torch.ones(2, 1, 3), torch.ones(2)
    native = seq._nodes
    try:
        for seq._nodes in {native, None}:
            with torch.autograd.forward_ad.dual_level():
                t = torch.autograd.forward_ad.make_dual(x, x)
                row = torch.autograd.forward_ad.make_dual(x[:, 0], x[:, 0])
                for call in (lambda: d.depthwise_conv1d_causal(t, w), lambda: d.layer_norm(t),
                             lambda: d.gated_linear_recurrence(x, t, x, vec),
                             lambda: d.layer_norm(x[0], torch.autograd.forward_ad.make_dual(vec, vec)),
                             lambda: d.depthwise_conv1d_causal_step(row, w, torch.zeros(1, 2, 2)),
                             lambda: d.gated_linear_recurrence_step(row, row, row, vec, torch.zeros(1, 2))):
                    with pytest.raises(RuntimeError, match="forward-mode differentiation is not supported"):
                        call()
    finally:
        seq._nodes = native


def test_module_surfaces():
    import dwconv_b200 as d
    c = d.CausalDepthwiseConv1d(6, 4)
    c.load_state_dict(torch.nn.Conv1d(6, 6, 4, groups=6).state_dict())
    n = d.LayerNorm(6)
    n.load_state_dict(torch.nn.LayerNorm(6).state_dict())
    r = d.GatedLinearRecurrence(1000)
    a = torch.exp(-8.0 * torch.nn.functional.softplus(r.decay.double()))
    assert r.decay.dtype == torch.float32 and 0.8999 < float(a.min()) and float(a.max()) < 0.99901
    m = d.RecurrentMixer(6, width=8)
    before = m.recurrence.decay.detach().clone()
    m = m.to(torch.bfloat16)
    assert torch.equal(m.recurrence.decay, before)  # neither converted nor rounded
    assert m.recurrence.decay.dtype == torch.float32 and m.norm.weight.dtype == torch.bfloat16
    assert [tuple(t.shape) for t in m.initial_state(3)] == [(3, 3, 8), (3, 8)]
    assert [t.dtype for t in m.initial_state(3)] == [torch.bfloat16, torch.float32]


def differences(f, args, grads, gen, h=1e-5):
    """(f(x + h e) - f(x - h e)) / 2h along a random direction of each argument; the functions are smooth with
    values of order one, so the quotient is off by some h^2 and 2^-52 / h."""
    for i, name in enumerate(grads):
        e = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        ends = [f(*[a + s * h * e if j == i else a for j, a in enumerate(args)]) for s in (1, -1)]
        want = (grads[name] * e).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 1e-7 * (1 + abs(want)), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64])
def test_a_converted_recurrence_keeps_its_gradient_too(dtype):
    import dwconv_b200 as d
    r = d.GatedLinearRecurrence(5)
    value, grad = r.decay.detach().clone(), torch.randn(5)
    r.decay.grad = grad.clone()
    r.to(dtype)
    assert r.decay.dtype == r.decay.grad.dtype == torch.float32
    assert torch.equal(r.decay, value) and torch.equal(r.decay.grad, grad)
    torch.optim.SGD(r.parameters(), lr=1.).step()
    assert torch.equal(r.decay, value - grad)


def test_the_definitions_gradients_are_derivatives():
    gen = torch.Generator().manual_seed(21)

    def rand(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    for offsets, n in ((None, 2), ([0, 3, 3, 9], 3)):
        B, T, C = (2, 9, 3) if offsets is None else (1, 11, 3)
        args = [rand(B, T, C), rand(B, T, C), rand(B, T, C), rand(C), rand(n, C)]
        dy, ds = rand(B, T, C), rand(n, C)
        out, _ = ref.recurrence(*args[:4], 2.0, args[4], offsets, dy, ds)

        def f(x, u, v, decay, init):
            o, _ = ref.recurrence(x, u, v, decay, 2.0, init, offsets)
            return ((o["y"] * dy).sum() + (o["state"] * ds).sum()).item()

        differences(f, args, {k: out[k] for k in ("dx", "du", "dv", "ddecay", "dinitial")}, gen)
        args = [rand(B, T, C), rand(C, 1, 4), rand(C), rand(n, 3, C)]
        ds = rand(n, 3, C)
        out, _ = ref.conv(*args[:3], "silu", args[3], offsets, dy, ds)

        def f(x, w, b, init):
            o, _ = ref.conv(x, w, b, "silu", init, offsets)
            return ((o["y"] * dy).sum() + (o["state"] * ds).sum()).item()

        differences(f, args, {k: out[k] for k in ("dx", "dweight", "dbias", "dinitial")}, gen)
    args = [rand(4, 7), rand(7), rand(7)]
    dy = rand(4, 7)
    out, _ = ref.norm(*args, 1e-5, dy)
    differences(lambda *a: (ref.norm(*a, 1e-5)[0]["y"] * dy).sum().item(), args,
                {k: out[k] for k in ("dx", "dweight", "dbias")}, gen)


def test_the_definitions_agree_with_plain_formulas():
    gen = torch.Generator().manual_seed(22)
    x, w = torch.randn(2, 9, 3, generator=gen), torch.randn(3, 1, 4, generator=gen)
    b, h0 = torch.randn(3, generator=gen), torch.randn(2, 3, 3, generator=gen)
    out, _ = ref.conv(x, w, b, "silu", h0)
    full = torch.cat([h0, x], 1).double().transpose(1, 2)
    want = torch.nn.functional.silu(torch.nn.functional.conv1d(full, w.double(), b.double(), groups=3)).transpose(1, 2)
    assert torch.allclose(out["y"], want, rtol=0, atol=1e-12)
    n, _ = ref.norm(x, b, b, 1e-5)
    assert torch.allclose(n["y"], torch.nn.functional.layer_norm(x.double(), (3,), b.double(), b.double()), atol=1e-12)
    u, v, d = torch.randn(2, 9, 3, generator=gen), torch.randn(2, 9, 3, generator=gen), torch.randn(3, generator=gen)
    r, _ = ref.recurrence(x, u, v, d, 2.0)
    h = torch.zeros(2, 3, dtype=torch.float64)
    for t in range(9):
        a = torch.exp(-2.0 * torch.log1p(torch.exp(d.double())) * torch.sigmoid(u[:, t].double()))
        h = a * h + torch.sqrt(1 - a * a) * torch.sigmoid(v[:, t].double()) * x[:, t].double()
        assert torch.allclose(r["y"][:, t], h, rtol=0, atol=1e-12)
