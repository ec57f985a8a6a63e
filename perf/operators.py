"""Cases of the sequence operators: the causal depthwise convolution, the gated linear recurrence
and the layer norm, each in its plain form (elementary torch operations) and as a user calls it.

``own`` false: the plain form; true: the calls of ``dwconv_b200``.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SCALE = 8.0   # exponent scale of the recurrence's decay
_EPS = 1e-5


def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "depthwise-conv-pytorch_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dwconv_b200
    return dwconv_b200


# ---- cases -----------------------------------------------------------------------------------

def _seq(name, op, mode, dtype, batch, length, channels, packed=0, state=False, taps=0,
         activation="", bias=False):
    c = {"op": op, "mode": mode, "dtype": dtype, "batch": batch, "length": length,
         "channels": channels, "packed": packed, "state": state}
    if op == "conv":
        c.update(taps=taps, activation=activation, bias=bias)
    if name:
        c["name"] = name
    return c


def _norm(name, mode, dtype, rows, channels):
    c = {"op": "norm", "mode": mode, "dtype": dtype, "rows": rows, "channels": channels}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token for each of eight conversations: the smallest call a decoder makes
        _seq("recurrence step 8x2048 bf16", "recurrence", "step", "bfloat16", 8, 1, 2048, state=True),
        # prompts of a serving batch, packed end to end, each carried on from a state
        _seq("recurrence packed prefill bf16", "recurrence", "forward", "bfloat16", 1, 8191, 2560, packed=17, state=True),
        # an ordinary training step
        _seq("recurrence train 4x2048x2048 bf16", "recurrence", "train", "bfloat16", 4, 2048, 2048),
        # one long document, trained in full precision, piece after piece (state in and out)
        _seq("recurrence train 32771x1152 fp32", "recurrence", "train", "float32", 1, 32771, 1152, state=True),
        # the largest training step
        _seq("recurrence train 8x8192x4096 bf16", "recurrence", "train", "bfloat16", 8, 8192, 4096),
        # one token for each of 128 conversations
        _seq("conv step 128x2048 k4 bf16", "conv", "step", "bfloat16", 128, 1, 2048, state=True, taps=4, activation="silu", bias=True),
        # packed prompts with an odd number of channels
        _seq("conv packed prefill 4099x1001 fp16", "conv", "forward", "float16", 1, 4099, 1001, packed=9, state=True, taps=4, activation="silu", bias=True),
        # an ordinary training step
        _seq("conv train 4x4096x2560 k4 bf16", "conv", "train", "bfloat16", 4, 4096, 2560, taps=4, activation="silu", bias=True),
        # a longer filter in full precision, no bias and no activation
        _seq("conv train 2x8192x576 k7 fp32", "conv", "train", "float32", 2, 8192, 576, taps=7),
        # the norm of a decoder's step: few rows, an odd width
        _norm("norm 64x1001 fp32", "forward", "float32", 64, 1001),
        # an ordinary training step
        _norm("norm train 16384x4096 bf16", "train", "bfloat16", 16384, 4096),
        # the norm behind a 7x7 depthwise convolution: 64 channels-last maps of 56x56 pixels
        _norm("norm train 200704x96 fp16", "train", "float16", 64 * 56 * 56, 96),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "conv", "norm"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    most = 1 << 26  # values of one tensor
    channels = _spread(rng, 24, 8192)
    if rng.random() < 0.7:
        channels = -(-channels // 8) * 8
    if op == "norm":
        rows = min(_spread(rng, 1, 262144), most // channels)
        return _norm("", rng.choice(["forward", "train", "train"]), dtype, rows, channels)
    mode = rng.choice(["step", "forward", "forward", "train", "train", "train"])
    extra = {}
    if op == "conv":
        extra = {"taps": rng.choice([2, 3, 4, 4, 4, 5, 7]), "activation": rng.choice(["", "silu", "silu"]),
                 "bias": rng.random() < 0.6}
    if mode == "step":
        return _seq("", op, mode, dtype, _spread(rng, 1, 512), 1, channels, state=True, **extra)
    packed = rng.choice([0, 0, _spread(rng, 1, 64)])
    batch = 1 if packed else _spread(rng, 1, 16)
    length = max(1, min(_spread(rng, 1, 65536), most // (batch * channels)))
    return _seq("", op, mode, dtype, batch, length, channels, packed=packed,
                state=rng.random() < 0.5, **extra)


def _offsets(total, count, gen):
    """Starts of ``count`` packed sequences and the end of the last: lengths of zero and one among
    them, and a few rows of padding behind the last where there is room."""
    used = total - min(5, total // 8)
    cuts = torch.randint(0, used + 1, (max(count - 1, 0),), generator=gen)
    if count >= 6 and used >= 2:
        cuts[0] = cuts[1]                                  # an empty sequence
        cuts[2] = min(int(cuts[3]) + 1, used)              # one of a single row, or another empty one
    cuts = torch.sort(cuts).values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([used])]).to(torch.int32)


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    train = case["mode"] == "train"

    def normal(*shape, dtype=dtype, leaf=True):
        t = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
        return t.requires_grad_(train and leaf)

    C = case["channels"]
    s = {"case": case, "dtype": dtype}
    if case["op"] == "norm":
        s["x"] = normal(case["rows"], C)
        with torch.no_grad():
            s["weight"] = (1 + 0.1 * normal(C, leaf=False).float()).to(dtype)
            s["bias"] = (0.1 * normal(C, leaf=False).float()).to(dtype)
        s["weight"].requires_grad_(train)
        s["bias"].requires_grad_(train)
        if train:
            s["dy"] = normal(case["rows"], C, leaf=False)
        return s
    B, T = case["batch"], case["length"]
    step = case["mode"] == "step"
    shape = (B, C) if step else (B, T, C)
    s["x"] = normal(*shape)
    if train:
        s["dy"] = normal(*shape, leaf=False)
    s["offsets"] = None
    rows = B
    if case["packed"]:
        s["offsets"] = _offsets(T, case["packed"], torch.Generator().manual_seed(seed)).cuda()
        rows = case["packed"]
    if case["op"] == "conv":
        K = case["taps"]
        with torch.no_grad():
            s["weight"] = (normal(C, 1, K, leaf=False).float() / math.sqrt(K)).to(dtype)
        s["weight"].requires_grad_(train)
        s["bias"] = normal(C) if case["bias"] else None
        state_shape, state_dtype = (rows, K - 1, C), dtype
    else:
        s["u"], s["v"] = normal(*shape), normal(*shape)
        # decays between 0.9 and 0.999 for a fully open gate
        a = 0.9 + 0.099 * torch.rand(C, generator=gen, device="cuda", dtype=torch.float64)
        s["decay"] = torch.log(torch.expm1(-torch.log(a) / _SCALE)).float().requires_grad_(train)
        state_shape, state_dtype = (rows, C), torch.float32
    s["state"] = normal(*state_shape, dtype=state_dtype) if case["state"] else None
    if train and case["state"]:
        s["dstate"] = normal(*state_shape, dtype=state_dtype, leaf=False)
    return s


# ---- the framework's calls ---------------------------------------------------------------------

def _own(s):
    api = _package()
    case = s["case"]
    op, mode = case["op"], case["mode"]
    if op == "norm":
        y = api.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
        if mode == "forward":
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "conv":
        activation = case["activation"] or None
        if mode == "step":
            y = api.depthwise_conv1d_causal_step(s["x"], s["weight"], s["state"], s["bias"], activation)
            return {"y": y, "state": s["state"]}
        out = api.depthwise_conv1d_causal(s["x"], s["weight"], s["bias"], activation, s["state"],
                                          s["offsets"], return_state=case["state"])
        leaves = {"dx": s["x"], "dweight": s["weight"]}
        if s["bias"] is not None:
            leaves["dbias"] = s["bias"]
    else:
        if mode == "step":
            y = api.gated_linear_recurrence_step(s["x"], s["u"], s["v"], s["decay"], s["state"], _SCALE)
            return {"y": y, "state": s["state"]}
        out = api.gated_linear_recurrence(s["x"], s["u"], s["v"], s["decay"], s["state"], s["offsets"],
                                          return_state=case["state"], scale=_SCALE)
        leaves = {"dx": s["x"], "du": s["u"], "dv": s["v"], "ddecay": s["decay"]}
    outs = {"y": out[0], "state": out[1]} if case["state"] else {"y": out}
    if mode == "forward":
        return outs
    given = [s["dy"]]
    if case["state"]:
        leaves["dinitial"] = s["state"]
        given.append(s["dstate"])
    grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), given)
    return {**{k: v.detach() for k, v in outs.items()}, **dict(zip(leaves, grads))}


# ---- plain forms -------------------------------------------------------------------------------

def _rows_of(offsets, T):
    """For packed rows: the sequence of each row (clamped), whether it belongs to one, whether it
    is a sequence's first row."""
    t = torch.arange(T, device=offsets.device)
    seq = torch.searchsorted(offsets.long(), t, right=True) - 1
    inside = seq < offsets.numel() - 1
    seq = seq.clamp(max=offsets.numel() - 2)
    return t, seq, inside, inside & (offsets.long()[seq] == t)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h = 0: the associative scan over pairs
    (a, b), spans doubled in each of the log2(T) rounds (a linear recurrence has no closed
    elementary form that does not overflow)."""
    n = 1
    while n < b.shape[1]:
        b = torch.cat([b[:, :n], torch.addcmul(b[:, n:], a[:, n:], b[:, :-n])], 1)
        if 2 * n < b.shape[1]:
            a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _plain_recurrence(s):
    case, dtype = s["case"], s["dtype"]
    x, u, v = (s[k].float() for k in ("x", "u", "v"))
    step = case["mode"] == "step"
    if step:
        x, u, v = x[:, None], u[:, None], v[:, None]
    softplus = torch.log1p(torch.exp(s["decay"]))
    r, i = 1 / (1 + torch.exp(-u)), 1 / (1 + torch.exp(-v))
    z = _SCALE * softplus * r
    a = 1 + torch.expm1(-z)     # near 1 a long memory multiplies the error of exp itself
    beta = torch.sqrt(-torch.expm1(-2 * z))
    b = beta * i * x
    T = x.shape[1]
    carry = a.clone()                     # a, and 0 where a sequence starts
    first = torch.zeros_like(b)           # the state each row starts from, at the first rows
    offsets = s["offsets"]
    if offsets is not None:
        t, seq, inside, start = _rows_of(offsets, T)
        keep = inside[None, :, None]
        b = torch.where(keep, b, 0)
        carry = torch.where((inside & ~start)[None, :, None], a, 0)
        if s["state"] is not None:
            first = torch.where(start[None, :, None], s["state"][seq][None], 0)
    else:
        carry[:, 0] = 0
        if s["state"] is not None:
            first[:, 0] = s["state"]
    h = _scan(carry, b + a * first)
    y = h.to(dtype)
    if step:
        s["state"].copy_(h[:, 0])
        return {"y": y[:, 0], "state": s["state"]}
    out = {"y": y}
    if s["state"] is not None:
        if offsets is None:
            out["state"] = h[:, -1]
        else:
            o = offsets.long()
            filled = (o[1:] > o[:-1])[:, None]
            out["state"] = torch.where(filled, h[0, (o[1:] - 1).clamp(min=0)], s["state"])
    if case["mode"] == "forward":
        return out
    dy = s["dy"].float()
    if offsets is not None:
        dy = torch.where(keep, dy, 0)
    if s["state"] is not None:
        if offsets is None:
            dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dstate"][:, None]], 1)
        else:
            last = inside & (o[seq + 1] - 1 == t)
            dy = dy + torch.where(last[None, :, None], s["dstate"][seq][None], 0)
    later = torch.cat([carry[:, 1:], torch.zeros_like(carry[:, :1])], 1)
    g = _scan(later.flip(1), dy.flip(1)).flip(1)
    before = first + torch.where(carry != 0, torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1), 0)
    dz = g * (-a * before + a * a / beta * i * x)
    out["dx"] = (g * beta * i).to(dtype)
    out["du"] = (dz * z * (1 - r)).to(dtype)
    out["dv"] = (g * beta * x * i * (1 - i)).to(dtype)
    out["ddecay"] = _SCALE * (dz * r).sum((0, 1)) / (1 + torch.exp(-s["decay"]))
    if s["state"] is not None:
        if offsets is None:
            out["dinitial"] = (a * g)[:, 0]
        else:
            out["dinitial"] = torch.where(filled, (a * g)[0, o[:-1].clamp(max=T - 1)], s["dstate"])
    return out


def _plain_conv(s):
    case, dtype = s["case"], s["dtype"]
    K, C = case["taps"], case["channels"]
    w = s["weight"].float()[:, 0]
    bias = s["bias"].float() if s["bias"] is not None else torch.zeros(C, device=w.device)
    x = s["x"].float()
    step = case["mode"] == "step"
    if step:
        x = x[:, None]
    B, T = x.shape[:2]
    offsets = s["offsets"]
    packed = case["packed"]
    state = s["state"].float() if s["state"] is not None else torch.zeros(packed or B, K - 1, C, device=w.device)
    inside = None
    if offsets is None:
        source = torch.cat([state, x], 1)
        tail = source[:, T:]

        def read(k):                    # the rows that tap k multiplies
            return source[:, k:k + T]

        def add(total, k, rows):
            total[:, k:k + T] += rows
    else:
        # one list of rows: the sequences' initial rows, then the packed ones
        source = torch.cat([state.reshape(-1, C), x[0]])
        base, o = packed * (K - 1), offsets.long()
        t, seq, inside, _ = _rows_of(offsets, T)
        back = t[:, None] - (K - 1) + torch.arange(K, device=w.device)      # row read by each tap
        old = back - o[seq][:, None]                                        # negative: an initial row
        at = torch.where(old >= 0, base + back, (seq * (K - 1))[:, None] + old + K - 1)
        at = torch.where(inside[:, None], at, base + T - 1)                 # those are not used
        back = o[1:, None] - (K - 1) + torch.arange(K - 1, device=w.device)
        old = back - o[:-1, None]
        end = torch.where(old >= 0, base + back,
                          torch.arange(packed, device=w.device)[:, None] * (K - 1) + old + K - 1)
        tail = source[end]

        def read(k):
            return source[at[:, k]][None]

        def add(total, k, rows):        # a tap's rows are all different, but for unused zeros
            total.index_add_(0, at[:, k], rows[0])
    taps = w.t()                                                            # [K, C]
    p = bias + sum(taps[k] * read(k) for k in range(K))
    sig = 1 / (1 + torch.exp(-p)) if case["activation"] else None
    y = p * sig if case["activation"] else p
    keep = inside[None, :, None] if inside is not None else None
    if keep is not None:
        y = torch.where(keep, y, 0)
    if step:
        s["state"].copy_(tail)
        return {"y": y[:, 0].to(dtype), "state": s["state"]}
    out = {"y": y.to(dtype)}
    if case["state"]:
        out["state"] = tail.to(dtype)
    if case["mode"] == "forward":
        return out
    dp = s["dy"].float()
    if case["activation"]:
        dp = dp * sig * (1 + p * (1 - sig))
    if keep is not None:
        dp = torch.where(keep, dp, 0)
    dsource = torch.zeros_like(source)
    for k in range(K):
        add(dsource, k, dp * taps[k])
    if offsets is None:
        if case["state"]:
            dsource[:, T:] += s["dstate"]
        dinitial, dx = dsource[:, :K - 1], dsource[:, K - 1:]
    else:
        if case["state"]:
            dsource.index_add_(0, end.reshape(-1), s["dstate"].float().reshape(-1, C))
        dinitial, dx = dsource[:base].view(packed, K - 1, C), dsource[None, base:]
    out["dx"] = dx.to(dtype)
    out["dweight"] = torch.stack([(dp * read(k)).sum((0, 1)) for k in range(K)], 1)[:, None].to(dtype)
    if s["bias"] is not None:
        out["dbias"] = dp.sum((0, 1)).to(dtype)
    if case["state"]:
        out["dinitial"] = dinitial.to(dtype)
    return out


def _plain_norm(s):
    dtype = s["dtype"]
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    scale = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    normal = centred * scale
    out = {"y": (normal * w + b).to(dtype)}
    if s["case"]["mode"] == "forward":
        return out
    dy = s["dy"].float()
    q = dy * w
    dx = scale * (q - q.mean(1, keepdim=True) - normal * (q * normal).mean(1, keepdim=True))
    out.update(dx=dx.to(dtype), dweight=(dy * normal).sum(0).to(dtype), dbias=dy.sum(0).to(dtype))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        plain = {"recurrence": _plain_recurrence, "conv": _plain_conv, "norm": _plain_norm}
        return plain[state["case"]["op"]](state)


# ---- the definition in 64 bits -----------------------------------------------------------------

def _spans(s, T):
    """(batch index, row slice, state index) of every sequence."""
    if s["offsets"] is None:
        return [(b, slice(0, T), b) for b in range(s["case"]["batch"])]
    o = s["offsets"].tolist()
    return [(0, slice(o[j], o[j + 1]), j) for j in range(len(o) - 1)]


def _wide(t):
    return None if t is None else t.detach().double()


def _exact_recurrence(s):
    case = s["case"]
    train, step = case["mode"] == "train", case["mode"] == "step"
    x, u, v = (_wide(s[k]) for k in ("x", "u", "v"))
    if step:
        x, u, v = x.unsqueeze(1), u.unsqueeze(1), v.unsqueeze(1)
    leaves = [t.requires_grad_(train) for t in (x, u, v, _wide(s["decay"]))]
    z = _SCALE * torch.nn.functional.softplus(leaves[3], threshold=50) * torch.sigmoid(u)
    a = torch.exp(-z)
    b = (-torch.expm1(-2 * z)).sqrt() * torch.sigmoid(v) * x
    T = x.shape[1]
    spans = _spans(s, T)
    # the definition, row by row; sequences that share no rows advance together
    A, Bv = a.detach(), b.detach()
    H = torch.zeros_like(A)
    before = torch.zeros_like(A)
    initial = _wide(s["state"])
    final = initial.clone() if initial is not None else None
    if s["offsets"] is None:
        h = initial if initial is not None else torch.zeros_like(A[:, 0])
        for t in range(T):
            before[:, t] = h
            h = torch.addcmul(Bv[:, t], A[:, t], h)
            H[:, t] = h
        if final is not None:
            final = h
    else:
        for bi, rows, j in spans:
            h = initial[j] if initial is not None else torch.zeros_like(A[0, 0])
            for t in range(rows.start, rows.stop):
                before[bi, t] = h
                h = torch.addcmul(Bv[bi, t], A[bi, t], h)
                H[bi, t] = h
            if final is not None:
                final[j] = h
    if step:
        return {"y": H[:, 0], "state": final}
    out = {"y": H}
    if final is not None:
        out["state"] = final
    if not train:
        return out
    dy = _wide(s["dy"])
    G = torch.zeros_like(A)
    dfinal = _wide(s.get("dstate"))
    dinitial = torch.zeros_like(initial) if initial is not None else None
    if s["offsets"] is None:
        q = dfinal if dfinal is not None else torch.zeros_like(A[:, 0])
        for t in reversed(range(T)):
            g = dy[:, t] + q
            G[:, t] = g
            q = A[:, t] * g
        if dinitial is not None:
            dinitial = q
    else:
        for bi, rows, j in spans:
            q = dfinal[j] if dfinal is not None else torch.zeros_like(A[0, 0])
            for t in reversed(range(rows.start, rows.stop)):
                g = dy[bi, t] + q
                G[bi, t] = g
                q = A[bi, t] * g
            if dinitial is not None:
                dinitial[j] = q
    dx, du, dv, dd = torch.autograd.grad((a, b), leaves, (G * before, G))
    out.update(dx=dx, du=du, dv=dv, ddecay=dd)
    if dinitial is not None:
        out["dinitial"] = dinitial
    return out


def _exact_conv(s):
    case = s["case"]
    K, train, step = case["taps"], case["mode"] == "train", case["mode"] == "step"
    x = _wide(s["x"])
    x = (x.unsqueeze(1) if step else x).requires_grad_(train)
    w, bias, initial = _wide(s["weight"]).requires_grad_(train), _wide(s["bias"]), _wide(s["state"])
    for t in (bias, initial):
        if t is not None:
            t.requires_grad_(train)

    def one(rows, head, spot):
        """[n, T, C] rows behind [n, K-1, C] earlier ones; the windows' products, tap by tap."""
        if head is None:
            head = torch.zeros(rows.shape[0], K - 1, rows.shape[2], dtype=rows.dtype, device=rows.device)
        full = torch.cat([head, rows], 1)
        n = rows.shape[1]
        p = torch.zeros_like(rows) if bias is None else bias.expand_as(rows)
        for k in range(K):
            p = p + full.narrow(1, k, n) * w[:, 0, k]
        return (torch.nn.functional.silu(p) if case["activation"] else p), full[:, n:]

    T = x.shape[1]
    if s["offsets"] is None:
        y, final = one(x, initial, None)
    else:
        parts, finals, end = [], [], 0
        for bi, rows, j in _spans(s, T):
            yy, ff = one(x[:, rows], None if initial is None else initial[j:j + 1], j)
            parts.append(yy)
            finals.append(ff)
            end = rows.stop
        parts.append(torch.zeros_like(x[:, end:]))
        y, final = torch.cat(parts, 1), torch.cat(finals)
    if step:
        return {"y": y[:, 0], "state": final}
    out = {"y": y.detach()}
    if case["state"]:
        out["state"] = final.detach()
    if not train:
        return out
    leaves = {"dx": x, "dweight": w}
    if bias is not None:
        leaves["dbias"] = bias
    outs, given = [y], [_wide(s["dy"])]
    if case["state"]:
        leaves["dinitial"] = initial
        outs.append(final)
        given.append(_wide(s["dstate"]))
    out.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), given)))
    return out


def _exact_norm(s):
    train = s["case"]["mode"] == "train"
    x, w, b = (_wide(s[k]).requires_grad_(train) for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + _EPS) * w + b
    if not train:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), _wide(s["dy"]))
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "conv": _exact_conv, "norm": _exact_norm}[case["op"]](s)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; floating-point operations of the formulas
    (a transcendental counted as one)."""
    e = 4 if case["dtype"] == "float32" else 2
    C, mode = case["channels"], case["mode"]
    if case["op"] == "norm":
        n = case["rows"] * C
        if mode == "forward":
            return {"bytes": 2 * n * e + 2 * C * e, "flops": 7 * n}
        return {"bytes": 4 * n * e + 4 * C * e, "flops": 21 * n}
    n = case["batch"] * case["length"] * C
    rows = case["packed"] or case["batch"]
    if case["op"] == "conv":
        K = case["taps"]
        state = rows * (K - 1) * C * e if case["state"] else 0
        par = (K + (1 if case["bias"] else 0)) * C * e
        act = 4 if case["activation"] else 0
        if mode == "train":
            return {"bytes": 4 * n * e + 2 * par + 4 * state, "flops": n * (6 * K + 2 * act + 2)}
        return {"bytes": 2 * n * e + par + 2 * state, "flops": n * (2 * K + act)}
    state = rows * C * 4 if case["state"] else 0
    if mode == "train":
        return {"bytes": 8 * n * e + 8 * C + 4 * state, "flops": 40 * n}
    return {"bytes": 4 * n * e + 4 * C + 2 * state, "flops": 15 * n}
