"""The sequence operators on the GPU against their definitions in 64 bits (sequence_util.py, which also
derives the tolerances): types, sizes around the tiles' borders, strides, states, packed sequences with
empty ones among them, what is masked holding NaN, streams, graphs, and the three of them together."""
import pytest
import torch

import sequence_util as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
dtype_ids = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}.get
by_dtype = pytest.mark.parametrize("dtype", DTYPES, ids=dtype_ids)


def randn(gen, *shape, dtype=torch.float32, scale=1.0, grad=True):
    t = (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()
    return t.requires_grad_(grad)


def packed(lengths, tail=0):
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    return o, o[-1] + tail, torch.tensor(o, dtype=torch.int32, device="cuda")


LISTS = {
    "several": ([5, 0, 1, 64, 130, 0], 5),
    "aligned": ([64, 64, 8], 0),
    "empty_first": ([0, 0, 3], 0),
    "all_empty": ([0, 0], 9),
    "one": ([77], 0),
    "many_short": ([1, 2, 3] * 20, 7),
    "long": ([700, 1, 650], 3),
}


# ---- recurrence --------------------------------------------------------------------------------

def recurrence_inputs(B, T, C, n, dtype, seed, state, spread=True):
    g = torch.Generator().manual_seed(seed)
    x, u, v, dy = (randn(g, B, T, C, dtype=dtype) for _ in range(4))
    # decays from hardly any to next to everything per row; or long memories alone
    decay = (torch.rand(C, generator=g) * 14 - 9) if spread else (torch.rand(C, generator=g) * 4 - 8)
    decay = decay.cuda().requires_grad_()
    init = randn(g, n, C) if state else None
    dstate = randn(g, n, C, grad=False) if state else None
    return x, u, v, dy.detach(), decay, init, dstate


def run_recurrence(x, u, v, dy, decay, init, dstate, offsets_gpu, offsets, scale=8.0):
    import dwconv_b200 as d
    state = init is not None
    out = d.gated_linear_recurrence(x, u, v, decay, init, offsets_gpu, return_state=state, scale=scale)
    y = out[0] if state else out
    leaves = [x, u, v, decay] + ([init] if state else [])
    grads = torch.autograd.grad(list(out) if state else [y], leaves, [dy] + ([dstate] if state else []))
    want, tol = ref.recurrence(x, u, v, decay, scale, init, offsets, dy, dstate)
    dt = x.dtype
    ref.check(y, want["y"], tol["y"], dt, "y")
    for name, got in zip(("dx", "du", "dv"), grads):
        ref.check(got, want[name], tol[name], dt, name)
    ref.check(grads[3], want["ddecay"], tol["ddecay"], None, "ddecay")
    if state:
        ref.check(out[1], want["state"], tol["state"], None, "state")
        ref.check(grads[4], want["dinitial"], tol["dinitial"], None, "dinitial")
    with torch.no_grad():  # without a graph: the same bits
        again = d.gated_linear_recurrence(x, u, v, decay, init, offsets_gpu, return_state=state, scale=scale)
    assert torch.equal(again[0] if state else again, y)
    return y


SIZES = [(1, 1, 1), (2, 1, 2), (3, 7, 33), (1, 63, 64), (2, 64, 65), (1, 65, 130), (2, 129, 96), (1, 1029, 66),
         (5, 300, 31), (300, 130, 2), (2, 2100, 6)]


@by_dtype
@pytest.mark.parametrize("state", [False, True], ids=["zero", "state"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_recurrence_matches_its_definition(size, state, dtype):
    B, T, C = size
    run_recurrence(*recurrence_inputs(B, T, C, B, dtype, 1, state), None, None)


@by_dtype
@pytest.mark.parametrize("C", [1, 40, 66, 131])
@pytest.mark.parametrize("name", list(LISTS))
def test_recurrence_packed(name, C, dtype):
    offsets, T, on_gpu = packed(*LISTS[name])
    for state in (True, False):
        run_recurrence(*recurrence_inputs(1, T, C, len(offsets) - 1, dtype, 2, state), on_gpu, offsets)


@by_dtype
def test_recurrence_long_memories(dtype):
    run_recurrence(*recurrence_inputs(1, 3000, 64, 1, dtype, 3, True, spread=False), None, None)


def test_recurrence_scale_and_extreme_gates():
    x, u, v, dy, decay, init, dstate = recurrence_inputs(2, 40, 34, 2, torch.float32, 4, True)
    run_recurrence(x, u, v, dy, decay, init, dstate, None, None, scale=0.5)
    import dwconv_b200 as d
    big = torch.tensor([-200.0, -90.0, -30.0, 30.0, 90.0, 200.0], device="cuda")
    u2 = big.repeat(2, 40, 6)[:, :, :34].contiguous()
    y = d.gated_linear_recurrence(x, u2, u2, decay, init)
    want, tol = ref.recurrence(x, u2, u2, decay, 8.0, init)
    # sigmoid of -90 is 8e-40, below fp32's normal numbers: it counts as 0, and so does sqrt(1 - a^2)
    # below 1e-18
    ref.check(y, want["y"], tol["y"] + 1e-17, None, "y")
    inf = torch.full_like(u2, float("inf"))
    closed = d.gated_linear_recurrence(x, -inf, inf, decay, init)           # r = 0: the state stays
    assert torch.allclose(closed, init.detach()[:, None].expand_as(closed), rtol=0, atol=1e-16)
    grads = torch.autograd.grad(d.gated_linear_recurrence(x, -inf, inf, decay, init), [x, init], dy)
    assert bool(torch.isfinite(grads[0]).all()) and float(grads[0].abs().max()) < 1e-15


def test_recurrence_reads_strided_rows():
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(5)
    T, B, C = 70, 3, 34
    proj = randn(g, B, T, 3 * C, grad=False)
    x, u, v = proj.chunk(3, -1)
    decay = (torch.rand(C, generator=g) * 4 - 8).cuda()
    want = d.gated_linear_recurrence(x.contiguous(), u.contiguous(), v.contiguous(), decay)
    assert torch.equal(d.gated_linear_recurrence(x, u, v, decay), want)
    tb = proj.transpose(0, 1).contiguous().transpose(0, 1)                  # time-major storage
    assert torch.equal(d.gated_linear_recurrence(*tb.chunk(3, -1), decay), want)
    back = x.transpose(1, 2).contiguous().transpose(1, 2)                   # channels not side by side
    assert torch.equal(d.gated_linear_recurrence(back, u, v, decay), want)
    odd = torch.empty(B * T * C + 1, device="cuda")[1:].view(B, T, C).copy_(x)   # 4-byte aligned only
    assert torch.equal(d.gated_linear_recurrence(odd, u, v, decay), want)
    same = x[:, :1].expand(B, T, C)                                         # one row for all
    assert torch.equal(d.gated_linear_recurrence(same, u, v, decay),
                       d.gated_linear_recurrence(same.contiguous(), u, v, decay))
    leaf = proj.clone().requires_grad_()
    y = d.gated_linear_recurrence(*leaf.chunk(3, -1), decay)
    one, = torch.autograd.grad(y.sum(), leaf)                               # an expanded gradient
    leaf2 = proj.clone().requires_grad_()
    a, b, c = (t.contiguous() for t in leaf2.chunk(3, -1))
    two, = torch.autograd.grad(d.gated_linear_recurrence(a, b, c, decay), leaf2, torch.ones_like(y))
    assert torch.equal(one, two)


def test_recurrence_pieces_and_steps_equal_the_whole():
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(6)
    B, T, C = 2, 200, 66
    x, u, v = (randn(g, B, T, C, grad=False) for _ in range(3))
    decay = (torch.rand(C, generator=g) * 6 - 8).cuda()
    whole, end = d.gated_linear_recurrence(x, u, v, decay, return_state=True)
    want, tol = ref.recurrence(x, u, v, decay, 8.0)
    state, parts = None, []
    for lo, hi in ((0, 1), (1, 64), (64, 129), (129, 200)):
        y, state = d.gated_linear_recurrence(x[:, lo:hi], u[:, lo:hi], v[:, lo:hi], decay, state, return_state=True)
        parts.append(y)
    ref.check(torch.cat(parts, 1), want["y"], 2 * tol["y"], None, "pieces")
    st = torch.zeros(B, C, device="cuda")
    rows = []
    for t in range(T):
        rows.append(d.gated_linear_recurrence_step(x[:, t], u[:, t], v[:, t], decay, st))
    ref.check(torch.stack(rows, 1), want["y"], 2 * tol["y"], None, "steps")
    ref.check(st, want["state"], 2 * tol["state"], None, "state")


@by_dtype
@pytest.mark.parametrize("size", [(1, 1), (3, 33), (128, 64), (7, 130)], ids=lambda s: "x".join(map(str, s)))
def test_recurrence_step(size, dtype):
    import dwconv_b200 as d
    B, C = size
    x, u, v, _, decay, init, _ = recurrence_inputs(B, 1, C, B, dtype, 7, True)
    x, u, v, decay, init = (t.detach() for t in (x, u, v, decay, init))
    want, tol = ref.recurrence(x, u, v, decay, 8.0, init)
    st = init.clone()
    y = d.gated_linear_recurrence_step(x[:, 0], u[:, 0], v[:, 0], decay, st)
    ref.check(y, want["y"][:, 0], tol["y"][:, 0], dtype, "y")
    ref.check(st, want["state"], tol["state"], None, "state")


def test_recurrence_masked_rows_and_neighbours_stay_apart():
    """NaN and infinities behind the last sequence are not looked at; those of one sequence reach no
    other, forward or backward."""
    import dwconv_b200 as d
    offsets, T, on_gpu = packed([70, 3, 0, 90, 64], 6)
    C = 10
    x, u, v, dy, decay, init, dstate = recurrence_inputs(1, T, C, 5, torch.float32, 8, True)
    run_recurrence(x, u, v, dy, decay, init, dstate, on_gpu, offsets)

    def grads(x, u, v, dy, init, dstate):
        leaves = [t.detach().clone().requires_grad_() for t in (x, u, v, init)]
        out = d.gated_linear_recurrence(*leaves[:3], decay, leaves[3], on_gpu, return_state=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (dy, dstate)))

    clean = grads(x, u, v, dy, init, dstate)
    for t in (clean[0], *clean[2:5]):
        assert not t[:, offsets[-1]:].any()
    bad = [t.detach().clone() for t in (x, u, v, dy)]
    for t in bad:
        t[:, offsets[-1]:] = float("nan")
    for a, b in zip(grads(*bad, init, dstate), clean):
        assert torch.equal(a, b)
    for value in (float("nan"), float("inf")):
        bad = [t.detach().clone() for t in (x, u, v, dy, init, dstate)]
        for t in bad[:4]:
            t[:, offsets[3]:offsets[4]] = value
        for t in bad[4:]:
            t[3] = value
        got = grads(*bad)
        for a, b in zip((got[0], *got[2:5]), (clean[0], *clean[2:5])):
            assert torch.equal(a[:, :offsets[3]], b[:, :offsets[3]])
            assert torch.equal(a[:, offsets[4]:], b[:, offsets[4]:])
        for a, b in ((got[1], clean[1]), (got[5], clean[5])):
            keep = [0, 1, 2, 4]
            assert torch.equal(a[keep], b[keep])


def test_lists_that_are_not_ascending_stay_in_bounds():
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(9)
    T, C = 100, 36
    x, u, v = (randn(g, 1, T, C) for _ in range(3))
    w = randn(g, C, 1, 4)
    decay = torch.zeros(C, device="cuda", requires_grad=True)
    for values in ([50, 20, 90], [0, 300, -7, 40], [-5, -1, 1 << 30], [7, 7, 7]):
        offsets = torch.tensor(values, dtype=torch.int32, device="cuda")
        y = d.gated_linear_recurrence(x, u, v, decay, None, offsets)
        torch.autograd.grad(y, [x, u, v, decay], torch.ones_like(y))
        y = d.depthwise_conv1d_causal(x, w, None, "silu", None, offsets)
        torch.autograd.grad(y, [x, w], torch.ones_like(y))
    torch.cuda.synchronize()


def test_recurrence_needs_only_what_is_asked():
    import dwconv_b200 as d
    x, u, v, dy, decay, init, dstate = recurrence_inputs(2, 70, 34, 2, torch.float32, 10, True)
    want, tol = ref.recurrence(x, u, v, decay, 8.0, init, None, torch.zeros_like(dy), dstate)
    _, state = d.gated_linear_recurrence(x, u, v, decay, init, return_state=True)
    got = torch.autograd.grad(state, [x, init], dstate)                     # the state's gradient alone
    ref.check(got[0], want["dx"], tol["dx"], None, "dx")
    ref.check(got[1], want["dinitial"], tol["dinitial"], None, "dinitial")
    y, _ = d.gated_linear_recurrence(x, u.detach(), v.detach(), decay.detach(), return_state=True)
    assert torch.autograd.grad(y, [x], dy)[0].shape == x.shape


# ---- convolution -------------------------------------------------------------------------------

def conv_inputs(B, T, C, K, n, dtype, seed, state, bias):
    g = torch.Generator().manual_seed(seed)
    x, dy = randn(g, B, T, C, dtype=dtype), randn(g, B, T, C, dtype=dtype, grad=False)
    w = randn(g, C, 1, K, dtype=dtype, scale=K ** -0.5)
    b = randn(g, C, dtype=dtype) if bias else None
    init = randn(g, n, K - 1, C, dtype=dtype) if state else None
    dstate = randn(g, n, K - 1, C, dtype=dtype, grad=False) if state else None
    return x, dy, w, b, init, dstate


def run_conv(x, dy, w, b, init, dstate, act, offsets_gpu, offsets):
    import dwconv_b200 as d
    state = init is not None
    out = d.depthwise_conv1d_causal(x, w, b, act, init, offsets_gpu, return_state=state)
    y = out[0] if state else out
    leaves = {"dx": x, "dweight": w}
    if b is not None:
        leaves["dbias"] = b
    if state:
        leaves["dinitial"] = init
    grads = torch.autograd.grad(list(out) if state else [y], list(leaves.values()), [dy] + ([dstate] if state else []))
    want, tol = ref.conv(x, w, b, act, init, offsets, dy, dstate)
    ref.check(y, want["y"], tol["y"], x.dtype, "y")
    if state:
        ref.check(out[1], want["state"], tol["state"], x.dtype, "state")
    for name, got in zip(leaves, grads):
        ref.check(got, want[name], tol[name], x.dtype, name)


CONV_SIZES = [(1, 1, 1), (2, 2, 4), (3, 7, 33), (1, 64, 128), (2, 65, 132), (1, 257, 36), (5, 31, 6), (2, 600, 20)]


@by_dtype
@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("size", CONV_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_conv_matches_its_definition(size, K, dtype):
    B, T, C = size
    run_conv(*conv_inputs(B, T, C, K, B, dtype, 11, True, True), "silu", None, None)
    run_conv(*conv_inputs(B, T, C, K, B, dtype, 12, False, False), None, None, None)


@by_dtype
@pytest.mark.parametrize("act", list(ref.ACTS), ids=str)
def test_conv_activations(act, dtype):
    x, dy, w, b, init, dstate = conv_inputs(2, 50, 36, 4, 2, dtype, 13, True, True)
    if act in ("relu", "relu6", "hardswish"):
        # keep away from the kinks, where fp32 and 64 bits may take different sides
        p = ref.conv(x, w, b, None, init)[0]["y"]
        near = ((p.abs() < 1e-3) | ((p - 6).abs() < 1e-3) | ((p.abs() - 3).abs() < 1e-3)).cuda()
        dy = torch.where(near, torch.zeros_like(dy), dy)
    run_conv(x, dy, w, b, init, dstate, act, None, None)


@by_dtype
@pytest.mark.parametrize("C", [1, 36, 131])
@pytest.mark.parametrize("K", [1, 2, 4, 7])
@pytest.mark.parametrize("name", list(LISTS))
def test_conv_packed(name, K, C, dtype):
    offsets, T, on_gpu = packed(*LISTS[name])
    for state in (True, False):
        run_conv(*conv_inputs(1, T, C, K, len(offsets) - 1, dtype, 14, state, state), "silu", on_gpu, offsets)


def test_conv_masked_rows_and_neighbours_stay_apart():
    import dwconv_b200 as d
    offsets, T, on_gpu = packed([70, 3, 0, 90, 64], 6)
    x, dy, w, b, init, dstate = conv_inputs(1, T, 12, 4, 5, torch.float32, 15, True, True)

    def grads(x, dy, init, dstate):
        leaves = [t.detach().clone().requires_grad_() for t in (x, init)]
        out = d.depthwise_conv1d_causal(leaves[0], w, b, "silu", leaves[1], on_gpu, return_state=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (dy, dstate)))

    clean = grads(x, dy, init, dstate)
    assert not clean[0][:, offsets[-1]:].any() and not clean[2][:, offsets[-1]:].any()
    bad = [t.detach().clone() for t in (x, dy)]
    for t in bad:
        t[:, offsets[-1]:] = float("nan")
    for a, c in zip(grads(*bad, init, dstate), clean):
        assert torch.equal(a, c)
    # weight and bias gradients do not see them either
    leaves = [w, b]
    pair = [torch.autograd.grad(d.depthwise_conv1d_causal(t, w, b, "silu", init, on_gpu), leaves, g)
            for t, g in ((x, dy), bad)]
    for a, c in zip(*pair):
        assert torch.equal(a, c)
    bad = [t.detach().clone() for t in (x, dy, init, dstate)]
    for t in bad[:2]:
        t[:, offsets[3]:offsets[4]] = float("nan")
    for t in bad[2:]:
        t[3] = float("nan")
    got = grads(*bad)
    for a, c in ((got[0], clean[0]), (got[2], clean[2])):
        assert torch.equal(a[:, :offsets[3]], c[:, :offsets[3]])
        assert torch.equal(a[:, offsets[4]:], c[:, offsets[4]:])
    for a, c in ((got[1], clean[1]), (got[3], clean[3])):
        assert torch.equal(a[[0, 1, 2, 4]], c[[0, 1, 2, 4]])


def test_conv_strides_pieces_and_steps():
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(16)
    B, T, C, K = 3, 70, 36, 4
    wide = randn(g, B, T, 2 * C, grad=False)
    w, b = randn(g, C, 1, K, grad=False), randn(g, C, grad=False)
    x = wide[:, :, C:]
    want = d.depthwise_conv1d_causal(x.contiguous(), w, b, "silu")
    assert torch.equal(d.depthwise_conv1d_causal(x, w, b, "silu"), want)
    assert torch.equal(d.depthwise_conv1d_causal(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, "silu"), want)
    assert torch.equal(d.depthwise_conv1d_causal(x.transpose(1, 2).contiguous().transpose(1, 2), w, b, "silu"), want)
    odd = torch.empty(B * T * C + 1, device="cuda")[1:].view(B, T, C).copy_(x)
    assert torch.equal(d.depthwise_conv1d_causal(odd, w, b, "silu"), want)
    wt = torch.empty(K, C, device="cuda").t().unsqueeze(1).copy_(w)         # weights in another order
    assert torch.equal(d.depthwise_conv1d_causal(x, wt, b, "silu"), want)
    state, parts = None, []
    for lo, hi in ((0, 1), (1, 3), (3, 64), (64, 70)):
        y, state = d.depthwise_conv1d_causal(x[:, lo:hi], w, b, "silu", state, return_state=True)
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), want)
    assert torch.equal(state, x[:, T - K + 1:])
    st = torch.zeros(B, K - 1, C, device="cuda")
    rows = [d.depthwise_conv1d_causal_step(x[:, t], w, st, b, "silu") for t in range(T)]
    assert torch.equal(torch.stack(rows, 1), want)
    assert torch.equal(st, x[:, T - K + 1:])


@by_dtype
@pytest.mark.parametrize("K", [1, 2, 4, 8])
@pytest.mark.parametrize("size", [(1, 1), (3, 33), (128, 64)], ids=lambda s: "x".join(map(str, s)))
def test_conv_step(size, K, dtype):
    import dwconv_b200 as d
    B, C = size
    x, _, w, b, init, _ = conv_inputs(B, 1, C, K, B, dtype, 17, True, True)
    x, w, b, init = (t.detach() for t in (x, w, b, init))
    want, tol = ref.conv(x, w, b, "silu", init)
    st = init.clone()
    y = d.depthwise_conv1d_causal_step(x[:, 0], w, st, b, "silu")
    ref.check(y, want["y"][:, 0], tol["y"][:, 0], dtype, "y")
    ref.check(st, want["state"], tol["state"], dtype, "state")


# ---- layer norm --------------------------------------------------------------------------------

def run_norm(x, w, b, dy, eps=1e-5):
    import dwconv_b200 as d
    y = d.layer_norm(x, w, b, eps)
    leaves = {"dx": x}
    if w is not None:
        leaves["dweight"] = w
    if b is not None:
        leaves["dbias"] = b
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    want, tol = ref.norm(x, w, b, eps, dy)
    ref.check(y, want["y"], tol["y"], x.dtype, "y")
    for name, got in zip(leaves, grads):
        ref.check(got, want[name], tol[name], x.dtype, name)
    with torch.no_grad():
        assert torch.equal(d.layer_norm(x, w, b, eps), y)


NORM_SIZES = [(1, 1), (3, 2), (5, 8), (70, 24), (33, 96), (130, 33), (9, 256), (200, 257), (4, 1001), (7, 1024),
              (6, 4096), (3, 5001), (2, 8192), (2, 12288), (3, 16384), (2, 17000), (2, 40000), (1300, 40)]


@by_dtype
@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_norm_matches_its_definition(size, dtype):
    rows, C = size
    g = torch.Generator().manual_seed(18)
    x = (torch.randn(rows, C, generator=g) * 2 + 0.5).to(dtype).cuda().requires_grad_()
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dtype).cuda().requires_grad_()
    b = randn(g, C, dtype=dtype)
    dy = randn(g, rows, C, dtype=dtype, grad=False)
    run_norm(x, w, b, dy)
    run_norm(x, None, None, dy)


@by_dtype
@pytest.mark.parametrize("C", [520, 776, 1000, 2048, 3080, 4096])
def test_norm_of_many_rows(C, dtype):
    """CTAs that stay for many rows; widths with and without a tail."""
    g = torch.Generator().manual_seed(53)
    x = (torch.randn(4800, C, generator=g) * 2 + 0.5).to(dtype).cuda()
    w, b = (1 + 0.3 * torch.randn(C, generator=g)).to(dtype).cuda(), randn(g, C, dtype=dtype, grad=False)
    import dwconv_b200 as d
    for wt, bt in ((w, b), (None, b), (w, None)):
        y = d.layer_norm(x, wt, bt)
        want, tol = ref.norm(x, wt, bt, 1e-5)
        ref.check(y, want["y"], tol["y"], dtype, "y")
    # with a graph: the statistics that the backward reads
    rows = slice(0, 4800, 37)
    leaf = x.clone().requires_grad_()
    dy = randn(g, 4800, C, dtype=dtype, grad=False)
    dx, = torch.autograd.grad(d.layer_norm(leaf, w, b), leaf, dy)
    want, tol = ref.norm(x[rows], w, b, 1e-5, dy[rows])
    ref.check(dx[rows], want["dx"], tol["dx"], dtype, "dx")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 37, 9001])
@pytest.mark.parametrize("C", [24, 48, 88, 192, 376, 744, 768])
def test_norm_of_three_wide_vectors_per_thread(C, rows, dtype):
    """Rows within a warp whose threads hold three vectors, full ones and with places beyond the row; and
    the same rows off 16-byte boundaries, which go another way."""
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(54)
    x = (torch.randn(rows, C + 1, generator=g) * 2 - 0.5).to(dtype).cuda()
    w, b = (1 + 0.3 * torch.randn(C, generator=g)).to(dtype).cuda(), randn(g, C, dtype=dtype, grad=False)
    for rows_of_x in (x[:, :C].contiguous(), x[:, :C]):
        want, tol = ref.norm(rows_of_x, w, b, 1e-5)
        ref.check(d.layer_norm(rows_of_x, w, b), want["y"], tol["y"], dtype, "y")
        leaf = rows_of_x.clone().requires_grad_()
        dy = randn(g, rows, C, dtype=dtype, grad=False)
        y = d.layer_norm(leaf, w, b)
        want, tol = ref.norm(rows_of_x, w, b, 1e-5, dy)
        ref.check(y, want["y"], tol["y"], dtype, "y")
        ref.check(torch.autograd.grad(y, leaf, dy)[0], want["dx"], tol["dx"], dtype, "dx")


@pytest.mark.parametrize("C", [784, 1200, 1528, 1536])
def test_norm_of_six_wide_vectors_per_thread(C):
    """Many rows that one warp holds in six vectors per thread; a slice of them against the definition, and
    all of them against calls with few rows, which hold them otherwise."""
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(55)
    rows = 16384 + 5
    x = (torch.randn(rows, C, generator=g) * 2 - 0.5).to(torch.bfloat16).cuda()
    w, b = (1 + 0.3 * torch.randn(C, generator=g)).to(x.dtype).cuda(), randn(g, C, dtype=x.dtype, grad=False)
    y = d.layer_norm(x, w, b)
    want, tol = ref.norm(x[-700:], w, b, 1e-5)
    ref.check(y[-700:], want["y"], tol["y"], x.dtype, "y")
    few = torch.cat([d.layer_norm(part, w, b) for part in x.split(4096)])
    # each side is off by half a step of its value and the fp32 difference before it
    assert ((y.float() - few.float()).abs() <= 2 ** -7 * few.float().abs() + 1e-4).all()


def test_norm_far_from_zero_and_constant_rows():
    g = torch.Generator().manual_seed(19)
    for C in (40, 1000, 20000):
        x = (torch.randn(5, C, generator=g) + 1000).cuda()
        x[2] = 7.0
        x[3] = 0.0
        dy = randn(g, 5, C, grad=False)
        run_norm(x.requires_grad_(), None, None, dy)


def test_norm_layouts():
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(20)
    C = 48
    w, b = randn(g, C, grad=False), randn(g, C, grad=False)
    # the map behind a channels-last depthwise convolution, normalised over its channels in place
    m = torch.randn(2, C, 5, 6, generator=g).cuda().to(memory_format=torch.channels_last)
    k = torch.randn(C, 1, 3, 3, generator=g).cuda()
    y = d.depthwise_conv2d(m, k, padding=1)
    rows = y.permute(0, 2, 3, 1)
    got = d.layer_norm(rows, w, b)
    assert got.shape == rows.shape and torch.equal(got, d.layer_norm(rows.contiguous(), w, b))
    want, tol = ref.norm(rows, w, b, 1e-5)
    ref.check(got, want["y"], tol["y"], None, "maps")
    # slices, transposed rows, one vector
    big = randn(g, 4, 7, 3 * C, grad=False)
    for t in (big[..., C:2 * C], big[:, ::2, :C], big.transpose(0, 1)[..., :C], big[..., ::3], big[:1, :1, :C]):
        assert torch.equal(d.layer_norm(t, w, b), d.layer_norm(t.contiguous(), w, b))
    for t in (big[1, 2, 5:5 + C], big[:, :, 1:1 + C]):                      # not 16-byte aligned
        want, tol = ref.norm(t, w, b, 1e-5)
        ref.check(d.layer_norm(t, w, b), want["y"], tol["y"], None, "unaligned")
    leaf = big.clone().requires_grad_()
    one, = torch.autograd.grad(d.layer_norm(leaf[..., :C], w, b).sum(), leaf)
    leaf2 = big.clone().requires_grad_()
    z = d.layer_norm(leaf2[..., :C].contiguous(), w, b)
    two, = torch.autograd.grad(z, leaf2, torch.ones_like(z))
    assert torch.equal(one, two)


def test_norm_rows_keep_to_themselves():
    import dwconv_b200 as d
    x = torch.randn(9, 100, device="cuda")
    clean = d.layer_norm(x)
    x[4] = float("nan")
    got = d.layer_norm(x)
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(got[keep], clean[keep]) and bool(got[4].isnan().all())


# ---- streams, graphs, sizes ----------------------------------------------------------------------

def three(stream_input):
    import dwconv_b200 as d
    x, u, v, decay, w = stream_input
    y = d.layer_norm(d.depthwise_conv1d_causal(x, w, None, "silu"))
    return d.gated_linear_recurrence(y, u, v, decay)


def three_inputs(seed, T=300, C=66, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x, u, v = (randn(g, 2, T, C, dtype=dtype) for _ in range(3))
    return x, u, v, (torch.rand(C, generator=g) * 6 - 8).cuda().requires_grad_(), randn(g, C, 1, 4, dtype=dtype)


def test_two_streams_at_once():
    sets = [three_inputs(30 + i) for i in range(2)]
    want = []
    for s in sets:
        y = three(s)
        want.append((y, *torch.autograd.grad(y, list(s), torch.ones_like(y))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                y = three(s)
                got[i].append((y, *torch.autograd.grad(y, list(s), torch.ones_like(y))))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            for a, b in zip(run, want[i]):
                assert torch.equal(a, b)   # the same bits on every run, whatever else is running


def test_captured_training_step_and_decoding_step():
    """Forward and backward captured into one graph, replayed on other data; a second graph from the
    same memory pool beside it."""
    import dwconv_b200 as d
    static = three_inputs(40)
    seeds = torch.ones(2, 300, 66, device="cuda")

    def work():
        y = three(static)
        return (y, *torch.autograd.grad(y, list(static), seeds))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=graphs[0].pool() if graphs else None):
            outs.append([t.detach() for t in work()])
        graphs.append(gr)
    for seed in (41, 42):
        fresh = three_inputs(seed)
        with torch.no_grad():
            for a, b in zip(static, fresh):
                a.copy_(b)
        y = three(fresh)
        want = (y, *torch.autograd.grad(y, list(fresh), seeds))
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    # a decoder's step: state carried from replay to replay
    C = 66
    st_c, st_r = torch.zeros(2, 3, C, device="cuda"), torch.zeros(2, C, device="cuda")
    row = [torch.zeros(2, C, device="cuda") for _ in range(3)]
    x, u, v, decay, w = (t.detach() for t in three_inputs(43))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        z = d.layer_norm(d.depthwise_conv1d_causal_step(row[0], w, st_c, None, "silu"))
        h = d.gated_linear_recurrence_step(z, row[1], row[2], decay, st_r)
    st_c.zero_()
    st_r.zero_()
    rows = []
    for t in range(20):
        for r, full in zip(row, (x, u, v)):
            r.copy_(full[:, t])
        gr.replay()
        rows.append(h.clone())
    whole = three((x[:, :20], u[:, :20], v[:, :20], decay, w))
    assert torch.allclose(torch.stack(rows, 1), whole, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("op", ["conv", "recurrence", "norm"])
def test_capture_beside_a_live_eager_graph(op):
    """An eager graph on the default stream holds the leaves: a captured backward is refused before the
    engine can break the capture; once it is gone the same capture runs."""
    import gc
    import dwconv_b200 as d
    if not d.sequence._nodes:
        pytest.skip("the compiled nodes are not in use")
    x, u, v, decay, w = three_inputs(44)

    def work():
        if op == "conv":
            return d.depthwise_conv1d_causal(x, w, None, "silu"), [x, w]
        if op == "recurrence":
            return d.gated_linear_recurrence(x, u, v, decay), [x, u, v, decay]
        return d.layer_norm(x), [x]

    seeds = torch.ones_like(x)
    want = torch.autograd.grad(*work(), seeds)

    def captured():
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y, leaves = work()
            grads = torch.autograd.grad(y, leaves, seeds)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, want):
            assert torch.equal(a, b)

    alive = work()
    with pytest.raises(RuntimeError, match="still alive on the default stream"):
        captured()
    for a, b in zip(torch.autograd.grad(*alive, seeds), want):   # the eager graph itself goes on
        assert torch.equal(a, b)
    del alive
    gc.collect()   # frames of the refused call hold a graph of the leaves as well
    captured()


def test_offsets_into_tensors_pass_32_bits():
    """Tensors of more than 2^31 elements; the inputs are one row seen many times."""
    import dwconv_b200 as d
    C, T = 2048, (1 << 20) + 3 * 64 + 5
    g = torch.Generator().manual_seed(22)
    row = [randn(g, 1, 1, C, dtype=torch.bfloat16, grad=False).expand(1, T, C) for _ in range(3)]
    decay = torch.zeros(C, device="cuda")                                   # short memories: settles soon
    y, state = d.gated_linear_recurrence(*row, decay, return_state=True)
    assert torch.equal(y[0, T - 1], y[0, 500]) and torch.equal(y[0, 1 << 20], y[0, 500])
    assert torch.equal(state[0].bfloat16(), y[0, T - 1])
    del y
    w = randn(g, C, 1, 4, dtype=torch.bfloat16, grad=False)
    y = d.depthwise_conv1d_causal(row[0], w, None, "silu")
    assert torch.equal(y[0, T - 1], y[0, 3]) and torch.equal(y[0, 1 << 20], y[0, 3])
    del y
    y = d.layer_norm(row[0])
    assert torch.equal(y[0, T - 1], y[0, 0]) and torch.equal(y[0, 1 << 20], y[0, 0])


def test_saved_state_that_a_step_overwrites_is_noticed():
    import dwconv_b200 as d
    x, u, v, dy, decay, init, _ = recurrence_inputs(2, 4, 10, 2, torch.float32, 23, True)
    init = init.detach()
    y = d.gated_linear_recurrence(x, u, v, decay, init)
    with torch.no_grad():
        d.gated_linear_recurrence_step(x[:, 0], u[:, 0], v[:, 0], decay, init)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)
    xc, dyc, w, b, st, _ = conv_inputs(2, 4, 10, 4, 2, torch.float32, 24, True, True)
    st = st.detach()
    y = d.depthwise_conv1d_causal(xc, w, b, None, st)
    with torch.no_grad():
        d.depthwise_conv1d_causal_step(xc[:, 0], w, st, b)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [xc], dyc)


def test_nothing_to_do():
    """Batches, lengths and row counts of zero."""
    import dwconv_b200 as d
    C = 12
    decay = torch.zeros(C, device="cuda", requires_grad=True)
    w, b = torch.randn(C, 1, 4, device="cuda", requires_grad=True), torch.randn(C, device="cuda", requires_grad=True)
    for B, T in ((0, 5), (2, 0), (0, 0)):
        x = torch.randn(B, T, C, device="cuda", requires_grad=True)
        h0 = torch.randn(B, C, device="cuda", requires_grad=True)
        y, s = d.gated_linear_recurrence(x, x, x, decay, h0, return_state=True)
        assert y.shape == x.shape and torch.equal(s, h0)
        gx, gd, gh = torch.autograd.grad([y, s], [x, decay, h0], [y, torch.ones_like(s)])
        assert gx.shape == x.shape and not gd.any() and torch.equal(gh, torch.ones_like(h0))
        c0 = torch.randn(B, 3, C, device="cuda", requires_grad=True)
        y, s = d.depthwise_conv1d_causal(x, w, b, "silu", c0, return_state=True)
        assert y.shape == x.shape and torch.equal(s, c0)
        gx, gw, gb, gc = torch.autograd.grad([y, s], [x, w, b, c0], [y, torch.ones_like(s)])
        assert not gw.any() and not gb.any() and torch.equal(gc, torch.ones_like(c0))
        y = d.layer_norm(x, b.detach(), b)
        gx, gb = torch.autograd.grad(y, [x, b], y)
        assert gx.shape == x.shape and not gb.any()
    assert d.gated_linear_recurrence_step(*[torch.zeros(0, C, device="cuda")] * 3, decay.detach(),
                                          torch.zeros(0, C, device="cuda")).shape == (0, C)
    assert d.depthwise_conv1d_causal_step(torch.zeros(0, C, device="cuda"), w.detach(),
                                          torch.zeros(0, 3, C, device="cuda")).shape == (0, C)


# ---- together ----------------------------------------------------------------------------------

def mixer_in_64_bits(m, x, offsets=None):
    """The block from the definitions, in 64 bits."""
    p = {k: ref.wide(v) for k, v in m.state_dict().items()}
    n = ref.norm(x, p["norm.weight"], p["norm.bias"], m.norm.eps)[0]["y"]
    gate, z = (n @ p["project_in.weight"].t() + p["project_in.bias"]).chunk(2, -1)
    z = ref.conv(z, p["conv.weight"], p["conv.bias"], None, None, offsets)[0]["y"]
    u, v = (z @ p["project_gates.weight"].t() + p["project_gates.bias"]).chunk(2, -1)
    h = ref.recurrence(z, u, v, p["recurrence.decay"], m.recurrence.scale, None, offsets)[0]["y"]
    return ref.wide(x) + (h * torch.nn.functional.gelu(gate)) @ p["project_out.weight"].t() + p["project_out.bias"]


def test_recurrent_mixer_whole_pieces_steps_and_packed():
    import dwconv_b200 as d
    torch.manual_seed(25)
    torch.backends.cuda.matmul.allow_tf32 = False
    m = d.RecurrentMixer(48, width=64).cuda()
    x = torch.randn(2, 90, 48, device="cuda")
    want = mixer_in_64_bits(m, x)
    # products of 48 to 128 terms of order one in fp32, a memory of up to 90 rows: 1e-4 is some 1000 roundings
    with torch.no_grad():
        y, _ = m(x)
        assert (ref.wide(y) - want).abs().max() < 1e-4
        a, state = m(x[:, :50])
        b, state = m(x[:, 50:70], state)
        rows = [m.step(x[:, t], state) for t in range(70, 90)]
        got = torch.cat([a, b, torch.stack(rows, 1)], 1)
        assert (ref.wide(got) - want).abs().max() < 1e-4
        state = m.initial_state(2)
        rows = torch.stack([m.step(x[:, t], state) for t in range(90)], 1)
        assert (ref.wide(rows) - want).abs().max() < 1e-4
        offsets, T, on_gpu = packed([40, 0, 1, 85], 54)
        flat = x.reshape(1, 180, 48)
        y, _ = m(flat, None, on_gpu)
        want = mixer_in_64_bits(m, flat, offsets)
        assert (ref.wide(y) - want)[:, :offsets[-1]].abs().max() < 1e-4


def test_recurrent_mixer_gradients():
    """Every parameter's gradient against differences of the block's own loss in fp32."""
    import dwconv_b200 as d
    torch.manual_seed(26)
    m = d.RecurrentMixer(16, width=24).cuda()
    x = torch.randn(2, 40, 16, device="cuda", requires_grad=True)
    target = torch.randn(2, 40, 16, device="cuda")
    loss = (m(x)[0] * target).sum()
    loss.backward()
    for name, p in list(m.named_parameters()) + [("x", x)]:
        e = torch.randn_like(p)
        e /= e.norm()
        step = 1e-2
        with torch.no_grad():
            vals = []
            for sign in (1, -1):
                p += sign * step * e
                vals.append(ref.wide(m(x)[0] * target).sum().item())
                p -= sign * step * e
        got, want = (vals[0] - vals[1]) / (2 * step), (ref.wide(p.grad) * ref.wide(e)).sum().item()
        # fp32 outputs of order one summed over 1280 values: 2e-4 in the loss, 1e-2 in the quotient, and the
        # quotient's own third-order term, 1e-4 relative to curvatures of order 10
        assert abs(got - want) <= 2e-2 * (1 + abs(want)), (name, got, want)


def test_mixer_in_bf16_keeps_its_decay_in_fp32():
    import dwconv_b200 as d
    m = d.RecurrentMixer(32).cuda().bfloat16()
    assert m.recurrence.decay.dtype == torch.float32 and m.conv.weight.dtype == torch.bfloat16
    x = torch.randn(2, 10, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, state = m(x)
    y.sum().backward()
    assert x.grad.dtype == torch.bfloat16 and m.recurrence.decay.grad.dtype == torch.float32
    assert state[0].dtype == torch.bfloat16 and state[1].dtype == torch.float32


# ---- lists and sizes drawn at random ------------------------------------------------------------

@pytest.mark.parametrize("seed", range(24))
def test_random_problems(seed):
    """Sizes, types, states and packed lists drawn anew; lists may begin behind row 0 and hold more sequences
    than the kernels keep on chip."""
    import random
    r = random.Random(1000 + seed)
    dtype = r.choice(DTYPES)
    C = r.choice([1, 2, 7, 8, 24, 63, 64, 72, 130, 200])
    state = r.random() < 0.5
    offsets = on_gpu = None
    if r.random() < 0.6:
        B, count = 1, r.choice([1, 3, 20, 1500 if C <= 24 else 40])
        o = [r.choice([0, 0, 5])]
        for _ in range(count):
            o.append(o[-1] + (r.choice([0, 1, 2]) if count > 100 else r.choice([0, 1, 3, 31, 32, 65, r.randint(0, 300)])))
        offsets, T = o, max(1, o[-1] + r.choice([0, 4]))
        on_gpu = torch.tensor(o, dtype=torch.int32, device="cuda")
        n = count
    else:
        B, T = r.choice([1, 2, 5]), r.choice([1, 31, 32, 33, 64, 200, 517, 1100])
        n = B
    run_recurrence(*recurrence_inputs(B, T, C, n, dtype, seed, state), on_gpu, offsets, scale=r.choice([1.0, 8.0]))
    K = r.randint(1, 8)
    run_conv(*conv_inputs(B, T, C, K, n, dtype, seed, state, r.random() < 0.5), r.choice(["silu", None]), on_gpu, offsets)
    g = torch.Generator().manual_seed(seed)
    w, b = randn(g, C, dtype=dtype), randn(g, C, dtype=dtype)
    run_norm(randn(g, B, T, C, dtype=dtype), w, b, randn(g, B, T, C, dtype=dtype, grad=False))


def test_rows_that_the_copy_engine_cannot_address():
    """Odd strides in one operand, an expanded batch in another, an expanded gradient: the same values as
    for contiguous tensors, forward and backward."""
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(51)
    B, T, C = 2, 150, 72
    u, v = randn(g, B, T, C, grad=False), randn(g, B, T, C, grad=False)
    odd = randn(g, B, T, C + 1, grad=False)[..., :C]
    one = randn(g, 1, T, C, grad=False).expand(B, T, C)
    decay = (torch.rand(C, generator=g) * 6 - 8).cuda()
    w = randn(g, C, 1, 4, grad=False)
    dys = [randn(g, B, T, C, grad=False), torch.ones((), device="cuda").expand(B, T, C), odd]
    for x in (odd, one):
        for dy in dys:
            for f in (lambda t: d.gated_linear_recurrence(t, u, v, decay), lambda t: d.depthwise_conv1d_causal(t, w),
                      lambda t: d.gated_linear_recurrence(u, t, v, decay)):
                a, b = x.detach().requires_grad_(), x.contiguous().requires_grad_()
                ya, yb = f(a), f(b)
                assert torch.equal(ya, yb)
                ga, = torch.autograd.grad(ya, a, dy)
                gb, = torch.autograd.grad(yb, b, dy.contiguous())
                assert torch.equal(ga, gb)


def test_interpreted_nodes_give_the_same_gradients():
    """The autograd functions that run without the compiled module."""
    import dwconv_b200 as d
    from dwconv_b200 import sequence as S
    x, u, v, decay, w = three_inputs(52, T=70)
    b, c0 = torch.randn(66, device="cuda", requires_grad=True), torch.randn(2, 3, 66, device="cuda", requires_grad=True)
    h0 = torch.randn(2, 66, device="cuda", requires_grad=True)
    pairs = [
        (d.depthwise_conv1d_causal(x, w, b, "silu", c0, return_state=True),
         S.CausalConv1dFunction.apply(x, w, b, c0, None, 3, True), [x, w, b, c0]),
        (d.gated_linear_recurrence(x, u, v, decay, h0, return_state=True),
         S.GatedLinearRecurrenceFunction.apply(x, u, v, decay, h0, None, 8.0, True), [x, u, v, decay, h0]),
        ((d.layer_norm(x, b, b),), (S.LayerNormFunction.apply(x, b, b, 1e-5),), [x, b]),
    ]
    for native, plain, leaves in pairs:
        given = [torch.randn_like(t) for t in native]
        for p, q in zip(native, plain):
            assert torch.equal(p, q)
        for p, q in zip(torch.autograd.grad(native, leaves, given, retain_graph=True),
                        torch.autograd.grad(plain, leaves, given)):
            assert torch.equal(p, q)
        # a graph is released behind its first use; asking for the input alone is enough
        torch.autograd.grad(native, leaves[:1], given)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(native, leaves[:1], given)


def test_no_wait_ran_out():
    """After all of the above: no kernel gave up waiting for its copies or its cluster."""
    from dwconv_b200 import _lib
    assert _lib.device_status() == 0


# ---- refusals on the device --------------------------------------------------------------------

def test_refusals():
    import dwconv_b200 as d
    from dwconv_b200 import sequence as S
    dev = dict(device="cuda")
    x, w = torch.randn(2, 5, 6, **dev), torch.randn(6, 1, 4, **dev)
    decay = torch.zeros(6, **dev)
    o = torch.tensor([0, 5], dtype=torch.int32, **dev)
    conv, rec = "conv1d_causal", "recurrence"
    cases = [
        (conv, (x.double(), w, None, 0, None, None, False), "unsupported dtype"),
        (conv, (x[0], w, None, 0, None, None, False), r"expected input \[B, T, C\]"),
        (conv, (x, w[:5], None, 0, None, None, False), r"weight must be \[C, 1, taps\] with C = 6"),
        (conv, (x, torch.randn(6, 1, 9, **dev), None, 0, None, None, False), "1 to 8 taps"),
        (conv, (x, w.half(), None, 0, None, None, False), "weight must be float on"),
        (conv, (x, w.cpu(), None, 0, None, None, False), "weight must be float on"),
        (conv, (x, w, decay[:5], 0, None, None, False), r"bias must be \(6,\), got \(5,\)"),
        (conv, (x, w, None, 0, torch.zeros(2, 4, 6, **dev), None, False), r"initial_state must be \(2, 3, 6\)"),
        (conv, (x, w, None, 0, None, o, False), "need a batch of 1"),
        (conv, (x[:1], w, None, 0, None, o.long(), False), "offsets must be a contiguous 1-d int32"),
        (conv, (x[:1], w, None, 0, None, o.cpu(), False), "offsets must be a contiguous 1-d int32"),
        (conv, (x[:1], w, None, 0, None, o[:1], False), "at least 2 row numbers"),
        (conv, (x, w, None, 9, None, None, False), "depthwise_conv1d_causal: bad argument"),
        (rec, (x, x[:1], x, decay, None, None, 8.0, False, False), "recurrence_gate must be"),
        (rec, (x, x, x.half(), decay, None, None, 8.0, False, False), "input_gate must be float on"),
        (rec, (x, x, x, decay.half(), None, None, 8.0, False, False), "decay must be float on"),
        (rec, (x, x, x, decay, torch.zeros(3, 6, **dev), None, 8.0, False, False), "initial_state must be"),
        (rec, (x, x, x, decay, None, None, 0.0, False, False), "scale must be positive"),
        (rec, (x, x, x, decay, None, None, float("nan"), False, False), "scale must be positive"),
        ("recurrence_step", (x[0], x[0], x[0], decay, torch.zeros(5, 12, **dev)[:, ::2], 8.0), "must be contiguous"),
        ("recurrence_step", (x[0], x[0], x[0], decay, torch.zeros(5, 6, **dev).half(), 8.0), "state must be float on"),
        ("conv1d_causal_step", (x[0], w, torch.zeros(5, 4, 6, **dev), None, 0), r"state must be \(5, 3, 6\)"),
        ("conv1d_causal_step", (x, w, torch.zeros(5, 3, 6, **dev), None, 0), r"expected input \[B, C\]"),
        ("layer_norm", (x, decay[:5], None, 1e-5, False), r"weight must be \(6,\), got \(5,\)"),
        ("layer_norm", (x, None, decay.half(), 1e-5, False), "bias must be float on"),
        ("layer_norm", (x, None, None, -1.0, False), "eps must not be negative"),
        ("layer_norm", (x.double(), None, None, 1e-5, False), "unsupported dtype"),
    ]
    for name, args, text in cases:
        said = []
        for fn in (getattr(S._forms, name), S.CTYPES_FORMS[name]):
            with pytest.raises(RuntimeError, match=text) as e:
                fn(*args)
            said.append(str(e.value).splitlines()[0])
        assert said[0] == said[1]
    leaf = x[0].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="updated in place"):
        d.gated_linear_recurrence_step(leaf, leaf, leaf, decay, torch.zeros(5, 6, **dev))
    with pytest.raises(RuntimeError, match="updated in place"):
        d.depthwise_conv1d_causal_step(leaf, w, torch.zeros(5, 3, 6, **dev))
    y = d.layer_norm(leaf)
    g, = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_ctypes_forms_give_the_same_bits():
    from dwconv_b200 import sequence as S
    x, u, v, decay, w = (t.detach() for t in three_inputs(50, T=40))
    offsets = torch.tensor([0, 30, 40], dtype=torch.int32, device="cuda")
    x1, u1, v1 = x[:1], u[:1], v[:1]
    h0, c0, b = torch.randn(2, 66, device="cuda"), torch.randn(2, 3, 66, device="cuda"), torch.randn(66, device="cuda")
    ck = S.CTYPES_FORMS["recurrence"](x1, u1, v1, decay, h0, offsets, 8.0, True, True)[2]
    stats = S.CTYPES_FORMS["layer_norm"](x, b, b, 1e-5, True)[1]
    calls = {
        "conv1d_causal": (x1, w, b, 3, c0, offsets, True),
        "conv1d_causal_backward": (x1, w, b, 3, c0, offsets, u1, c0, True),
        "conv1d_causal_step": lambda: (x[:, 0], w, c0.clone(), b, 3),
        "recurrence": (x1, u1, v1, decay, h0, offsets, 8.0, True, False),
        "recurrence_backward": (x1, u1, v1, decay, h0, offsets, 8.0, ck, u1, h0, True),
        "recurrence_step": lambda: (x[:, 0], u[:, 0], v[:, 0], decay, h0.clone(), 8.0),
        "layer_norm": (x, b, b, 1e-5, True),
        "layer_norm_backward": (x, b, stats, u, True, True),
    }
    for name, args in calls.items():
        got = []
        for fn in (getattr(S._forms, name), S.CTYPES_FORMS[name]):
            out = fn(*(args() if callable(args) else args))
            got.append(out if isinstance(out, tuple) else (out,))
        for a, c in zip(*got):
            assert (a is None and c is None) or torch.equal(a, c), name
