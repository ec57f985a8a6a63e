"""The sequence operators on the GPU where something goes wrong or is out of the ordinary: waits that run out,
non-finite parameters, gradients of gradients, saved tensors, mixed precision, long runs and many rows."""
import pytest
import torch

import sequence_util as ref
from test_sequence_gpu import DTYPES, by_dtype, conv_inputs, packed, randn, recurrence_inputs

pytestmark = pytest.mark.gpu


# ---- waits that run out ------------------------------------------------------------------------

@pytest.fixture
def expire():
    """Makes waits run out, or (0) leaves them as they are."""
    from dwconv_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    yield _lib.lib.dwconv_b200_debug_expire
    _lib.lib.dwconv_b200_debug_expire(0)
    _lib.device_status()


@by_dtype
@pytest.mark.parametrize("lengths", [None, [700, 0, 1, 1299]], ids=["dense", "packed"])
@pytest.mark.parametrize("size", [(1, 2000, 64), (1, 2000, 63), (2, 1000, 200), (1, 8, 64), (1, 40, 63), (1, 8, 63)],
                         ids=lambda s: "x".join(map(str, s)))
def test_a_wait_that_runs_out_is_reported_and_ends(size, lengths, dtype, expire):
    """Rows copied ahead (even widths) and read in place (odd ones), alone and in clusters of CTAs, some of which
    leave early while their peers wait in vain: the kernels end, say so, and leave the device as they found it."""
    import dwconv_b200 as d
    from dwconv_b200 import _lib
    B, T, C = size
    offsets = on_gpu = None
    n = B
    if lengths is not None:
        if (B, T) != (1, 2000):
            pytest.skip("the list has 2000 rows")
        offsets, _, on_gpu = packed(lengths)
        n = len(lengths)
    x, u, v, dy, decay, init, dstate = recurrence_inputs(B, T, C, n, dtype, 60, True)
    leaves = [x, u, v, decay, init]

    def both():
        out = d.gated_linear_recurrence(x, u, v, decay, init, on_gpu, return_state=True)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, [dy, dstate]))

    want = both()
    assert _lib.device_status() == 0
    for how in (1, 2, 2, 1):
        expire(how)
        both()
        status = _lib.device_status()
        if T >= 1000:       # clusters, and more tiles than a cluster has CTAs
            assert status == 8
        elif C % 2:         # no copies; no peers, or none that leave before the walk's end
            assert status == (8 if how == 1 and T > 32 else 0)
        else:               # the copies of the only tile, which may have landed before the first look at them
            assert status == 0 or (status == 8 and how == 1)
        expire(0)
        for a, b in zip(both(), want):
            assert torch.equal(a, b)
        assert _lib.device_status() == 0


def test_checked_calls_report_a_wait_that_ran_out(expire, monkeypatch):
    """With the status checks on, every call says so itself: with a graph, without one, and backward."""
    import dwconv_b200 as d
    from dwconv_b200 import sequence as S
    monkeypatch.setattr(S._lib, "CHECK_STATUS", True)
    monkeypatch.setattr(S, "_nodes", None)
    x, u, v, dy, decay, _, _ = recurrence_inputs(1, 2000, 64, 1, torch.float32, 65, False)
    y = d.gated_linear_recurrence(x, u, v, decay)
    gone = pytest.raises(RuntimeError, match="a kernel's bounded wait expired .*sequence operators")
    expire(1)
    with gone:
        d.gated_linear_recurrence(x, u, v, decay)
    with gone, torch.no_grad():
        d.gated_linear_recurrence(x, u, v, decay)
    with gone:
        torch.autograd.grad(y, x, dy)
    expire(0)
    for name, call, leaves in calls():
        torch.autograd.grad(call().sum(), leaves)
    gr = torch.cuda.CUDAGraph()     # a captured call cannot be checked, and is not
    with torch.no_grad(), torch.cuda.graph(gr):
        z = d.gated_linear_recurrence(x, u, v, decay)
    gr.replay()
    assert torch.equal(z, y)


# ---- autograd ----------------------------------------------------------------------------------

def calls(dtype=torch.float32, B=2, T=20, C=10):
    """Every operator over the compiled nodes and over the interpreted ones: (name, call, leaves)."""
    import dwconv_b200 as d
    from dwconv_b200 import sequence as S
    g = torch.Generator().manual_seed(61)
    x, u, v = (randn(g, B, T, C, dtype=dtype) for _ in range(3))
    w, b = randn(g, C, 1, 4, dtype=dtype), randn(g, C, dtype=dtype)
    decay = (torch.rand(C, generator=g) * 6 - 8).cuda().requires_grad_()
    return [
        ("conv", lambda: d.depthwise_conv1d_causal(x, w, b, "silu"), [x, w, b]),
        ("conv interpreted", lambda: S.CausalConv1dFunction.apply(x, w, b, None, None, 3, False), [x, w, b]),
        ("recurrence", lambda: d.gated_linear_recurrence(x, u, v, decay), [x, u, v, decay]),
        ("recurrence interpreted",
         lambda: S.GatedLinearRecurrenceFunction.apply(x, u, v, decay, None, None, 8.0, False), [x, u, v, decay]),
        ("norm", lambda: d.layer_norm(x, b, b), [x, b]),
        ("norm interpreted", lambda: S.LayerNormFunction.apply(x, b, b, 1e-5), [x, b]),
    ]


def test_a_penalty_on_gradients_is_refused_whatever_came_in():
    """The gradients depend on the inputs; taken for constants, a penalty on them would lose its part without a word.
    What does not differentiate them goes on."""
    for name, call, leaves in calls():
        first = torch.autograd.grad(call().sum(), leaves)
        grads = torch.autograd.grad(call().sum(), leaves, create_graph=True)
        for a, b in zip(first, grads):
            assert torch.equal(a, b), name
            with pytest.raises(RuntimeError, match="once_differentiable"):
                ((b * b).sum() + (leaves[0] ** 2).sum()).backward()
        for t in leaves:
            t.grad = None
        y = call()
        y.sum().backward(create_graph=True)
        for t, a in zip(leaves, first):
            assert torch.equal(t.grad, a), name
            t.grad = None


def test_saved_tensor_hooks_see_all_that_is_kept():
    """Offloading moves all that a graph keeps to the host, what the kernels leave for their backward passes
    included, and brings the same gradients back."""
    kept = {}
    for name, call, leaves in calls():
        want = torch.autograd.grad(call().sum(), leaves)
        sizes = []

        def pack(t):
            sizes.append((tuple(t.shape), t.dtype))
            return t.cpu()

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
            y = call()
        for a, b in zip(torch.autograd.grad(y.sum(), leaves), want):
            assert torch.equal(a, b), name
        kept[name] = sorted(map(str, sizes))
    for name in ("conv", "recurrence", "norm"):
        assert kept[name] == kept[name + " interpreted"], name
    assert len(kept["recurrence"]) == 5 and len(kept["norm"]) == 3


def test_checkpointed_operators_give_the_same_gradients():
    from torch.utils.checkpoint import checkpoint
    for name, call, leaves in calls():
        want = torch.autograd.grad(call().sum(), leaves)
        got = torch.autograd.grad(checkpoint(call, use_reentrant=False).sum(), leaves)
        for a, b in zip(got, want):
            assert torch.equal(a, b), name


def test_what_a_hook_hands_back_is_checked():
    for name, call, leaves in calls():
        if name.startswith("conv"):
            continue
        # the last of the saved tensors is the kernel's own
        for spoil, text in ((lambda t: t.cpu(), "must be float on"), (lambda t: t.half(), "must be float on"),
                            (lambda t: t[:-1], r"must be \(.*got"),
                            (lambda t: t.repeat_interleave(2, -1)[..., ::2], "must be contiguous")):
            own = {"recurrence": 1, "norm": 2}[name.split()[0]]   # its rank, which no other fp32 one of its size has

            def unpack(t):
                mine = t.dtype == torch.float32 and t.dim() == own and t.shape != leaves[-1].shape
                return spoil(t) if mine else t

            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = call()
            with pytest.raises(RuntimeError, match=text):
                torch.autograd.grad(y.sum(), leaves)


# ---- non-finite parameters ----------------------------------------------------------------------

@by_dtype
@pytest.mark.parametrize("value", [float("inf"), float("nan")], ids=str)
@pytest.mark.parametrize("C", [12, 7])
@pytest.mark.parametrize("K", [1, 2, 4, 7])
def test_conv_taps_reach_only_rows_of_the_sequence(K, C, value, dtype):
    """A tap that is not finite shows in the gradients of the rows that it multiplies and in no other: not behind the
    last sequence, nor where the sequence ends before its product, nor in initial rows it does not reach."""
    import dwconv_b200 as d
    offsets, T, on_gpu = packed([40, 3, 0, 1, 70], 6)
    n = 5
    for tap in range(K):
        x, dy, w, b, init, dstate = conv_inputs(1, T, C, K, n, dtype, 62, True, True)
        with torch.no_grad():
            w[::2, 0, tap] = value
        y, state = d.depthwise_conv1d_causal(x, w, b, None, init, on_gpu, return_state=True)
        leaves = [x, b] + ([init] if K > 1 else [])
        got = torch.autograd.grad([y, state], leaves, [dy, dstate])
        want, _ = ref.conv(x, w, b, None, init, offsets, dy, dstate)
        assert not y[:, offsets[-1]:].any() and not got[0][:, offsets[-1]:].any()
        for a, c in zip(got, (want["dx"], want["dbias"], want["dinitial"])):
            a, c = ref.wide(a), c
            assert torch.equal(a.isnan(), c.isnan()) and torch.equal(a == float("inf"), c == float("inf"))
            assert torch.equal(a == float("-inf"), c == float("-inf"))


@by_dtype
@pytest.mark.parametrize("value", [float("inf"), float("nan")], ids=str)
@pytest.mark.parametrize("C", [10, 7])
def test_recurrence_rows_of_no_sequence_are_zero_whatever_the_decay(C, value, dtype):
    import dwconv_b200 as d
    offsets, T, on_gpu = packed([40, 3, 0, 30], 70)
    x, u, v, dy, decay, init, dstate = recurrence_inputs(1, T, C, 4, dtype, 63, True)
    with torch.no_grad():
        decay[::2] = value
    y, state = d.gated_linear_recurrence(x, u, v, decay, init, on_gpu, return_state=True)
    for t in (y, *torch.autograd.grad([y, state], [x, u, v], [dy, dstate])):
        assert not t[:, offsets[-1]:].any()


@by_dtype
@pytest.mark.parametrize("C", [8, 5])
@pytest.mark.parametrize("act", ["relu", "relu6", "silu", "hardswish"])
def test_a_nan_passes_every_activation(act, C, dtype):
    """Row 3 of one channel is NaN: so are the outputs of the taps that reach it and no others, forward and in the
    one-row step, and the gradients of the filter; dx gets the slope that torch gives a NaN, or a NaN."""
    import dwconv_b200 as d
    x, dy, w, b, _, _ = conv_inputs(2, 20, C, 4, 2, dtype, 64, False, True)
    with torch.no_grad():
        x[0, 3, 1] = float("nan")
    y = d.depthwise_conv1d_causal(x, w, b, act)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 3:7, 1] = True
    assert torch.equal(y.isnan(), bad)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    keep = [c for c in range(C) if c != 1]
    assert dw[1].isnan().all() and not dw[keep].isnan().any() and not dx[..., keep].isnan().any()
    assert not dx[0, 7:].isnan().any() and not dx[1].isnan().any()
    if act in ("relu", "relu6"):
        # rows 3 to 6 pass dy on: dx[3] takes all of them and is finite, and not zero
        want = (w[1, 0].float().flip(0) * dy[0, 3:7, 1].float()).sum()
        assert abs(dx[0, 3, 1].float() - want) <= 4 * 2 ** -8 * (w[1, 0].float().flip(0) * dy[0, 3:7, 1].float()).abs().sum()
    with torch.no_grad():
        step = d.depthwise_conv1d_causal_step(x[:, 3], w, torch.zeros(2, 3, C, device="cuda", dtype=dtype), b, act)
    only = torch.zeros_like(step, dtype=torch.bool)
    only[0, 1] = True
    assert torch.equal(step.isnan(), only)


# ---- mixed precision ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows", ["fp32", "16 bits"])
def test_the_mixer_trains_and_serves_under_autocast(rows, dtype):
    """fp32 parameters, 16-bit activations: the same bits as the functions on parameters converted by hand."""
    import dwconv_b200 as d
    F = torch.nn.functional
    torch.manual_seed(66)
    m = d.RecurrentMixer(48, width=64).cuda()
    x = torch.randn(2, 40, 48, device="cuda", dtype=torch.float32 if rows == "fp32" else dtype, requires_grad=True)
    dy = torch.randn(2, 40, 48, device="cuda")
    leaves = [x, *m.parameters()]

    def by_hand():
        def linear(t, layer):
            return F.linear(t.to(dtype), layer.weight.to(dtype), layer.bias.to(dtype))
        gate, z = linear(d.layer_norm(x.float(), m.norm.weight, m.norm.bias, m.norm.eps), m.project_in).chunk(2, -1)
        z = d.depthwise_conv1d_causal(z, m.conv.weight.to(dtype), m.conv.bias.to(dtype))
        u, v = linear(z, m.project_gates).chunk(2, -1)
        h = d.gated_linear_recurrence(z, u, v, m.recurrence.decay, scale=m.recurrence.scale)
        return x + linear(h * F.gelu(gate), m.project_out)

    want = by_hand()
    want_grads = torch.autograd.grad(want, leaves, dy.to(want.dtype))
    with torch.autocast("cuda", dtype=dtype):
        got, state = m(x)
        assert torch.equal(got, want) and state[0].dtype == dtype and state[1].dtype == torch.float32
        for (name, p), a, b in zip([("x", x), *m.named_parameters()],
                                   torch.autograd.grad(got, leaves, dy.to(got.dtype)), want_grads):
            assert a.dtype == p.dtype and torch.equal(a, b), name
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        step_state = m.initial_state(2)
        assert step_state[0].dtype == dtype
        for t in range(40):
            m.step(x[:, t], step_state)
        # the last rows that the convolution keeps: sums of 48 products in another order, each rounded once to 16
        # bits, at most a step apart (2^-7 in bf16); twice that
        assert torch.allclose(step_state[0].float(), state[0].float(), rtol=2 ** -6, atol=2 ** -6)
    # without autocast the types have to agree, as they have to in torch's own layers
    with pytest.raises(RuntimeError, match="weight must be float|weight must be c10::"):
        m.conv(torch.zeros(1, 4, 64, device="cuda", dtype=dtype))
    with pytest.raises(RuntimeError, match="weight must be c10::"):
        m.norm(torch.zeros(1, 4, 48, device="cuda", dtype=dtype))


# ---- layer norm: every way a row is held -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "unaligned"])
def test_norm_of_every_width(aligned, dtype):
    """All widths up to 700 and some of each kind above, three rows each: whatever vectors, threads and warps hold
    a row, forward and backward."""
    import dwconv_b200 as d
    g = torch.Generator().manual_seed(67)
    widths = list(range(1, 701)) + list(range(704, 1600, 8)) + list(range(1600, 8193, 412)) + [4095, 4097, 8191, 8193]
    full = torch.randn(3, 8200, generator=g) * 2 + 0.5
    x, dy = full.to(dtype).cuda(), torch.randn(3, 8200, generator=g).to(dtype).cuda()
    w, b = (1 + 0.3 * torch.randn(8200, generator=g)).to(dtype).cuda(), torch.randn(8200, generator=g).to(dtype).cuda()
    for C in widths:
        leaf = (x[:, :C].contiguous() if aligned else x[:, 1:1 + C]).detach().requires_grad_()
        wt, bt = w[:C].contiguous(), b[:C].contiguous()
        y = d.layer_norm(leaf, wt, bt)
        dx, = torch.autograd.grad(y, leaf, dy[:, :C])
        want, tol = ref.norm(leaf, wt, bt, 1e-5, dy[:, :C])
        ref.check(y, want["y"], tol["y"], dtype, f"y of {C}")
        ref.check(dx, want["dx"], tol["dx"], dtype, f"dx of {C}")


# ---- long runs and many rows ---------------------------------------------------------------------

LONG = {
    # batch and rows that warps walk in runs of 32 to 128, several times what is copied ahead
    "dense": ((4, 4096, 1024), None),
    "odd width": ((2, 4096, 1281), None),
    # borders inside the runs, at their ends, next to one another, and rows behind the last sequence
    "packed": ((1, 16387, 1024), [5000, 1, 0, 43, 2, 3, 1000, 4096, 47, 48, 6140]),
    "packed, odd width": ((1, 8191, 1281), [2000, 3, 0, 4500, 1, 1680]),
}


@by_dtype
@pytest.mark.parametrize("K, act", [(1, "silu"), (2, "silu"), (3, None), (4, "silu"), (4, "hardswish"), (5, None),
                                    (7, "silu"), (8, "silu")], ids=str)
@pytest.mark.parametrize("problem", list(LONG))
def test_conv_in_long_runs(problem, K, act, dtype):
    """Problems large enough that a warp's run fills its copies ahead many times over; channels at the borders of
    lanes, warps and the tensor against the definition."""
    import dwconv_b200 as d
    (B, T, C), lengths = LONG[problem]
    offsets = on_gpu = None
    n = B
    if lengths is not None:
        offsets, _, on_gpu = packed(lengths)
        n = len(lengths)
        assert offsets[-1] <= T
    x, dy, w, b, init, dstate = conv_inputs(B, T, C, K, n, dtype, 70 + K, True, True)
    y, state = d.depthwise_conv1d_causal(x, w, b, act, init, on_gpu, return_state=True)
    leaves = {"dx": x, "dweight": w, "dbias": b, "dinitial": init}
    grads = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, dstate])))
    at = [0, 1, 2, 3, 63, 64, 66, 127, 128, C // 2 + 1, C - 5, C - 2, C - 1]
    if act == "hardswish":
        # away from its kinks, where fp32 and 64 bits may take different sides
        p = ref.conv(x[..., at], w[at], b[at], None, init[..., at], offsets)[0]["y"]
        dy = dy.clone()
        dy[..., at] = torch.where(((p.abs() - 3).abs() < 1e-3).cuda(), torch.zeros_like(dy[..., at]), dy[..., at])
        y, state = d.depthwise_conv1d_causal(x, w, b, act, init, on_gpu, return_state=True)
        grads = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, dstate])))
    want, tol = ref.conv(x[..., at], w[at], b[at], act, init[..., at], offsets, dy[..., at], dstate[..., at])
    # a run of 128 rows, 8 warps and 16 parts: 152 sums, of which the tolerance counts 144; times 1.25
    for name in ("dweight", "dbias"):
        tol[name] = 1.25 * tol[name]
    ref.check(y[..., at], want["y"], tol["y"], dtype, "y")
    ref.check(state[..., at], want["state"], tol["state"], dtype, "state")
    for name, got in grads.items():
        got = got[at] if name in ("dweight", "dbias") else got[..., at]
        ref.check(got, want[name], tol[name], dtype, name)


@by_dtype
@pytest.mark.parametrize("size", [(4800, 4096), (4800, 2048), (4801, 1032), (200000, 96), (40001, 40), (4000, 1001),
                                  (100003, 7), (700, 8200), (700, 5001), (299, 12288)], ids=lambda s: "x".join(map(str, s)))
def test_norm_weight_gradients_over_many_rows(size, dtype, monkeypatch):
    """Threads, warps and CTAs that take row after row, in every way that a row is held: what they add up over the
    rows.  The definition on the device."""
    import dwconv_b200 as d
    monkeypatch.setattr(ref, "wide", lambda t: None if t is None else t.detach().double())
    rows, C = size
    g = torch.Generator().manual_seed(71)
    x = (torch.randn(rows, C, generator=g) * 2 + 0.5).to(dtype).cuda().requires_grad_()
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dtype).cuda().requires_grad_()
    b = randn(g, C, dtype=dtype)
    dy = randn(g, rows, C, dtype=dtype, grad=False)
    got = torch.autograd.grad(d.layer_norm(x, w, b), [x, w, b], dy)
    # the definition makes the bias zeros on the host where there is none; here it is there
    want, tol = ref.norm(x, w, b, 1e-5, dy)
    for name, a in zip(("dx", "dweight", "dbias"), got):
        ref.check(a, want[name], tol[name], dtype, name)
    for a, c in zip(torch.autograd.grad(d.layer_norm(x, w, b), [w, b], dy), got[1:]):
        assert torch.equal(a, c)


@pytest.mark.parametrize("op", ["conv", "recurrence", "norm"])
def test_capture_beside_a_live_eager_graph_of_leaves_further_down(op):
    """The leaf is behind a view and a conversion: a captured backward is refused there too, and runs once the eager
    graph is gone.  A leaf that the backward is not asked for is no reason."""
    import gc
    import dwconv_b200 as d
    if not d.sequence._nodes:
        pytest.skip("the compiled nodes are not in use")
    g = torch.Generator().manual_seed(72)
    x, other = randn(g, 2, 20, 8), randn(g, 2, 20, 8)
    w, decay = randn(g, 8, 1, 4, grad=False, dtype=torch.float16), torch.zeros(8, device="cuda")

    def work():
        a = (x.half() + other.half())[:, 1:]
        if op == "conv":
            return d.depthwise_conv1d_causal(a, w)
        return d.gated_linear_recurrence(a, a, a, decay) if op == "recurrence" else d.layer_norm(a)

    seeds = torch.ones(2, 19, 8, device="cuda", dtype=torch.float16)

    def captured():
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got, = torch.autograd.grad(work(), x, seeds)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)

    want, = torch.autograd.grad(work(), x, seeds)
    alive = x * 2
    with pytest.raises(RuntimeError, match="still alive on the default stream"):
        captured()
    del alive
    gc.collect()
    captured()
    alive = other * 2
    captured()
    assert alive.requires_grad
