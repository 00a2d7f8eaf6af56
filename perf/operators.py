"""Cases for timing the recurrent mixers' operators through their public entry points: the
short causal convolution, the selective state space scan and the group norm around them.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call
from a seed, on the GPU; ``run`` makes one pass, in the operators' plain form (elementary
torch operations in 32 bits) or, where ``own`` is true, through ``kernels``; ``exact``
computes the same outputs in float64 token by token, its gradients by autograd; ``work``
counts the bytes and operations a pass cannot do without; ``draw`` makes further cases of
the same ranges.

Paths:

* ``conv_step``, ``conv_prefill``, ``conv_train``: ``short_conv`` for one token per
  sequence, for prompts with their state, and with its gradients;
* ``ssm_step``, ``ssm_prefill``, ``ssm_train``: ``ssm`` likewise;
* ``norm_forward``, ``norm_train``: ``group_norm`` without and with gradients.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
DT_RANK = 128     # columns before B and C in the projection that holds them


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _conv(path, batch, length, channels, taps=4, bias=True, activation=True, ragged=False,
          dtype="bf16"):
    return dict(path=path, batch=batch, length=length, channels=channels, taps=taps, bias=bias,
                activation=activation, ragged=ragged, dtype=dtype)


def _ssm(path, batch, length, channels, state=16, groups=1, gate=True, ragged=False,
         dtype="bf16"):
    return dict(path=path, batch=batch, length=length, channels=channels, state=state,
                groups=groups, gate=gate, ragged=ragged, dtype=dtype)


def _norm(path, batch, length, groups, width, form="gate", affine=True, heads=False,
          dtype="bf16"):
    return dict(path=path, batch=batch, length=length, groups=groups, width=width, form=form,
                affine=affine, heads=heads, dtype=dtype)


def listed():
    return [
        # one token of one sequence at the model's hidden size: the smallest call
        dict(_conv("conv_step", 1, 1, 2048), name="conv_step"),
        # a batch of prompts of unequal length, an odd number of channels, half a
        # projection's columns, after a kept state
        dict(_conv("conv_prefill", 5, 1021, 2050, ragged=True), name="conv_prompts_odd"),
        # training at twice the hidden size
        dict(_conv("conv_train", 4, 2048, 4096), name="conv_train"),
        # one token of one sequence, and of a batch of sequences being served
        dict(_ssm("ssm_step", 1, 1, 4096), name="ssm_step"),
        dict(_ssm("ssm_step", 64, 1, 4096), name="ssm_step_batch"),
        # one prompt
        dict(_ssm("ssm_prefill", 1, 2048, 4096), name="ssm_prompt"),
        # a batch of prompts of unequal length, after a kept state
        dict(_ssm("ssm_prefill", 5, 1531, 2048, ragged=True), name="ssm_prompts_ragged"),
        # one long prompt at the hidden size: little to run side by side
        dict(_ssm("ssm_prefill", 1, 16384, 2048), name="ssm_prompt_long"),
        # training, and training in fp32 at sizes no tile divides, two groups
        dict(_ssm("ssm_train", 4, 2048, 4096), name="ssm_train"),
        dict(_ssm("ssm_train", 2, 777, 1040, state=24, groups=2, dtype="fp32"),
             name="ssm_train_odd_fp32"),
        # the heads of a linear attention output, [B, H, L, D] in memory, normalised into
        # the rows that the output projection reads
        dict(_norm("norm_forward", 3, 1021, 32, 64, heads=True), name="norm_heads"),
        # training at twice the hidden size, 32 heads
        dict(_norm("norm_train", 4, 2048, 32, 128), name="norm_train"),
    ]


def _span(rng, lo, hi):
    """A whole number, spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows(rng, elements, most_length):
    """(batch, length) of up to 8 sequences within a number of elements."""
    length = _span(rng, 1, most_length)
    return _span(rng, 1, max(1, min(8, int(elements // length)))), length


def draw(rng):
    path = rng.choice(["conv_step", "conv_prefill", "conv_train", "ssm_step", "ssm_prefill",
                       "ssm_prefill", "ssm_train", "ssm_train", "norm_forward", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    kind, form = path.split("_")
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if kind == "norm":
        groups = _span(rng, 1, 64)
        width = _span(rng, 8, max(8, 4096 // groups))
        batch, length = _rows(rng, 2 ** 24 // (groups * width), 4096)
        return _norm(path, batch, length, groups, width, rng.choice(["gate", "silu", "none"]),
                     yes(), yes(), dtype)
    channels = _span(rng, 32, 4096)
    if yes():
        channels = max(8, channels // 8 * 8)
    if kind == "conv":
        batch, length = _rows(rng, 2 ** 24 // channels, 8192)
        if form == "step":
            batch, length = _span(rng, 1, 128), 1
        return _conv(path, batch, length, channels, rng.choice([2, 3, 4, 4, 4]), yes(), yes(),
                     form == "prefill" and yes(), dtype)
    state = rng.choice([4, 8, 16, 16, 16, 16, 24, 32, 64, _span(rng, 1, 64)])
    groups = rng.choice([1, 1, 1, 2])
    channels += channels % groups
    # at most the elements of the largest listed case, whatever the state's size
    most = 2 ** (28 if form == "train" else 27) // (channels * max(16, state))
    batch, length = _rows(rng, max(1, most), min(8192, max(1, most)))
    if form == "step":
        batch, length = _span(rng, 1, 128), 1
    return _ssm(path, batch, length, channels, state, groups, yes(), form == "prefill" and yes(),
                dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case, g):
    """Lengths of the padded batch's sequences, the longest filling it."""
    if not case["ragged"]:
        return None
    n = case["length"]
    lengths = torch.randint(1, n + 1, (case["batch"],), device="cuda", generator=g,
                            dtype=torch.int32)
    lengths[0] = n
    return lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    kind, form = case["path"].split("_")

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)
    b, n = case["batch"], case["length"]
    s = dict(case)
    if kind == "conv":
        c, k = case["channels"], case["taps"]
        # the mixer's half of a projection that holds its gate beside it
        x = randn(b, n, 2 * c).to(dtype)[..., :c]
        s["weight"] = randn(c, k) * k ** -0.5
        s["bias"] = 0.1 * randn(c) if case["bias"] else None
        shape, leaves = (b, n, c), ["x", "weight", "bias"]
        if form != "train":
            s["state"] = randn(b, k - 1, c).to(dtype)
    elif kind == "ssm":
        e, m, groups = case["channels"], case["state"], case["groups"]
        # x comes from the convolution, the gate is half of a projection, B and C are the
        # last columns of another
        x = torch.nn.functional.silu(randn(b, n, e)).to(dtype)
        s["z"] = randn(b, n, 2 * e).to(dtype)[..., e:] if case["gate"] else None
        s["dt"] = (0.5 * randn(b, n, e)).to(dtype)
        columns = randn(b, n, DT_RANK + 2 * groups * m).to(dtype)
        s["B"], s["C"] = (columns[..., DT_RANK + i * groups * m:DT_RANK + (i + 1) * groups * m]
                          .unflatten(-1, (groups, m)) for i in (0, 1))
        # decays of 1 .. N, steps of 1e-3 .. 1e-1 spread over their logarithm
        step = torch.exp(torch.rand(e, device="cuda", generator=g) * math.log(100.0)
                         + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -(torch.arange(1, m + 1, device="cuda") * (1 + 0.05 * randn(e, m)))
        s["D"] = 1 + 0.1 * randn(e)
        shape, leaves = (b, n, e), ["x", "dt", "A", "B", "C", "D", "z", "dt_bias"]
        if form != "train":
            s["state"] = randn(b, e, m)
    else:
        groups, width = case["groups"], case["width"]
        shape, leaves = (b, n, groups, width), ["x", "weight", "bias", "gate"]
        if case["heads"]:   # heads before tokens, as the attention operators write them
            x = (1.5 * randn(b, groups, n, width) + 0.5).to(dtype).transpose(1, 2)
        else:
            shape = (b, n, groups * width)
            x = (1.5 * randn(*shape) + 0.5).to(dtype)
        s["gate"] = randn(*shape).to(dtype) if case["form"] == "gate" else None
        s["weight"] = 1 + 0.1 * randn(groups * width) if case["affine"] else None
        s["bias"] = 0.1 * randn(groups * width) if case["affine"] else None
    s["x"] = x
    s["lengths"] = _lengths(case, g) if form == "prefill" else None
    if form == "step":
        for name in ("x", "dt", "B", "C", "z"):
            if s.get(name) is not None:
                s[name] = s[name][:, 0]
    if form == "train":
        s["dy"] = randn(*shape).to(dtype)
        s["leaves"] = [name for name in leaves if s[name] is not None]
        for name in s["leaves"]:
            s[name] = s[name].detach().requires_grad_()
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _silu(x):
    return x * _sigmoid(x)


def _silu_slope(x):
    s = _sigmoid(x)
    return s * (1 + x * (1 - s))


def _wide(s, name):
    return None if s[name] is None else s[name].detach().float()


def _before(lengths, n):
    """[B, L, 1]: the positions that a sequence of the padded batch has."""
    return (torch.arange(n, device="cuda") < lengths[:, None])[..., None]


def _plain_conv(s):
    form = s["path"].split("_")[1]
    x, w, bias = _wide(s, "x"), _wide(s, "weight"), _wide(s, "bias")
    k, act = s["taps"], s["activation"]
    if form == "step":
        x = x[:, None]
    b, n, c = x.shape
    before = s["state"].float() if form != "train" else x.new_zeros(b, k - 1, c)
    rows = torch.cat([before, x], 1)
    windows = rows.unfold(1, k, 1)                       # [B, L, C, K]
    pre = (windows * w).sum(-1)
    if bias is not None:
        pre = pre + bias
    y = _silu(pre) if act else pre
    if form == "step":
        s["state"].copy_(rows[:, 1:])
        return y[:, 0].to(s["x"].dtype), s["state"]
    if form == "prefill":
        last = rows[:, n:]
        if s["lengths"] is not None:
            y = torch.where(_before(s["lengths"], n), y, 0.0)
            at = s["lengths"].long()[:, None] + torch.arange(k - 1, device="cuda")
            last = rows.gather(1, at[..., None].expand(-1, -1, c))
        return y.to(s["x"].dtype), last.to(s["x"].dtype)
    g = _wide(s, "dy")
    if act:
        g = g * _silu_slope(pre)
    ahead = torch.cat([g, g.new_zeros(b, k - 1, c)], 1).unfold(1, k, 1)
    dx = (ahead * w.flip(-1)).sum(-1)
    dw = (windows * g[..., None]).sum((0, 1))
    out = [y.to(s["x"].dtype), dx.to(s["x"].dtype), dw]
    return out + [g.sum((0, 1))] if bias is not None else out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, from zero: each round joins runs of twice the
    length."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_ssm(s):
    form = s["path"].split("_")[1]
    names = ("x", "dt", "z", "B", "C")
    x, dt, z, B, C = (t if t is None or form != "step" else t[:, None]
                      for t in (_wide(s, name) for name in names))
    A, D, dt_bias = (_wide(s, name) for name in ("A", "D", "dt_bias"))
    b, n, e = x.shape
    groups, m = s["groups"], s["state"].shape[-1] if form != "train" else A.shape[-1]
    pre = dt + dt_bias
    delta = pre.clamp_min(0) + torch.log1p(torch.exp(-pre.abs()))
    u = delta * x
    if s["lengths"] is not None:
        inside = _before(s["lengths"], n)
        delta, u = torch.where(inside, delta, 0.0), torch.where(inside, u, 0.0)

    def channels(t):   # [B, L, E] -> [B, L, G, E / G, 1]
        return t.unflatten(2, (groups, e // groups))[..., None]
    A = A.view(groups, e // groups, m)
    B, C = B[:, :, :, None], C[:, :, :, None]            # [B, L, G, 1, N]
    a = torch.exp(channels(delta) * A)
    into = channels(u) * B
    if form != "train":
        into[:, 0] += a[:, 0] * s["state"].view(b, groups, e // groups, m)
    h = _scan(a, into)
    mixed = (h * C).sum(-1).flatten(2) + D * x
    y = mixed * _silu(z) if z is not None else mixed
    if form != "train":
        last = h[:, -1].reshape(b, e, m)
        if form == "step":
            s["state"].copy_(last)
            return y[:, 0].to(s["x"].dtype), s["state"]
        if s["lengths"] is not None:
            y = torch.where(inside, y, 0.0)
        return y.to(s["x"].dtype), last
    dy = _wide(s, "dy")
    dmixed = dy * _silu(z) if z is not None else dy
    ahead = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(ahead.flip(1), (channels(dmixed) * C).flip(1)).flip(1)
    back = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * a * g
    du = (g * B).sum(-1).flatten(2)
    ddt = ((back * A).sum(-1).flatten(2) + du * x) * _sigmoid(pre)
    grads = dict(x=du * delta + D * dmixed, dt=ddt,
                 A=(back * channels(delta)).sum((0, 1)).view(e, m),
                 B=(g * channels(u)).sum(3), C=(h * channels(dmixed)).sum(3),
                 D=(dmixed * x).sum((0, 1)), dt_bias=ddt.sum((0, 1)))
    if z is not None:
        grads["z"] = dy * mixed * _silu_slope(z)
    return [y.to(s["x"].dtype)] + [grads[name].to(s[name].dtype) for name in s["leaves"]]


def _plain_norm(s):
    x = _wide(s, "x")
    groups, width = s["groups"], s["width"]
    shape = x.shape
    rows = x.reshape(-1, groups, width)
    w, bias, gate = _wide(s, "weight"), _wide(s, "bias"), _wide(s, "gate")
    mean = rows.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((rows - mean).square().mean(-1, keepdim=True) + EPS)
    unit = (rows - mean) * rstd
    out = unit
    if w is not None:
        out = unit * w.view(groups, width) + bias.view(groups, width)
    if gate is not None:
        gate = gate.reshape(-1, groups, width)
        y = out * _silu(gate)
    else:
        y = _silu(out) if s["form"] == "silu" else out
    y = y.reshape(shape).to(s["x"].dtype)
    if "dy" not in s:
        return y
    dy = _wide(s, "dy").reshape(-1, groups, width)
    dout = dy
    if gate is not None:
        dout = dy * _silu(gate)
    elif s["form"] == "silu":
        dout = dy * _silu_slope(out)
    dunit = dout * w.view(groups, width) if w is not None else dout
    dx = rstd * (dunit - dunit.mean(-1, keepdim=True)
                 - unit * (dunit * unit).mean(-1, keepdim=True))
    grads = dict(x=dx.reshape(shape), weight=(dout * unit).sum(0).flatten(),
                 bias=dout.sum(0).flatten())
    if gate is not None:
        grads["gate"] = (dy * out * _silu_slope(gate)).reshape(shape)
    return [y] + [grads[name].to(s[name].dtype) for name in s["leaves"]]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own(s):
    from lizard_reproduction_amd import kernels
    kind, form = s["path"].split("_")
    if kind == "conv":
        act = "silu" if s["activation"] else None
        if form == "step":
            y = kernels.short_conv_decode_step(s["x"], s["weight"], s["state"], s["bias"], act)
            return y, s["state"]
        if form == "prefill":
            return kernels.short_conv_prefill(s["x"], s["weight"], s["bias"], act,
                                              state=s["state"], lengths=s["lengths"])
        y = kernels.short_conv(s["x"], s["weight"], s["bias"], act)
    elif kind == "ssm":
        more = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
        operands = [s[name] for name in ("x", "dt", "A", "B", "C")]
        if form == "step":
            return kernels.ssm_decode_step(*operands, s["state"], **more), s["state"]
        if form == "prefill":
            return kernels.ssm_prefill(*operands, **more, state=s["state"], lengths=s["lengths"])
        y = kernels.ssm(*operands, **more)
    else:
        act = None if s["form"] == "none" else "silu"
        # heads apart: the last two dimensions are the groups
        y = kernels.group_norm(s["x"], None if s["heads"] else s["groups"], s["weight"],
                               s["bias"], gate=s["gate"], activation=act, eps=EPS)
    if form != "train":
        return y
    return [y, *torch.autograd.grad(y, [s[name] for name in s["leaves"]], s["dy"])]


def run(state):
    if own:
        return _own(state)
    kind = state["path"].split("_")[0]
    with torch.no_grad():
        return {"conv": _plain_conv, "ssm": _plain_ssm, "norm": _plain_norm}[kind](state)


# ---------------------------------------------------------------------------
# the same in float64, from the definitions
# ---------------------------------------------------------------------------

def _exact_conv(s, t):
    """Tap by tap."""
    form = s["path"].split("_")[1]
    x = t["x"][:, None] if form == "step" else t["x"]
    n, k = x.shape[1], s["taps"]
    before = t["state"] if form != "train" else x.new_zeros(x.shape[0], k - 1, x.shape[2])
    rows = torch.cat([before, x], 1)
    y = sum(t["weight"][:, j] * rows[:, j:j + n] for j in range(k))
    if t["bias"] is not None:
        y = y + t["bias"]
    if s["activation"]:
        y = torch.nn.functional.silu(y)
    if form == "train":
        return y
    if form == "step":
        return y[:, 0], rows[:, 1:]
    ends = [n] * len(x) if s["lengths"] is None else s["lengths"].tolist()
    for i, end in enumerate(ends):
        y[i, end:] = 0
    return y, torch.stack([rows[i, end:end + k - 1] for i, end in enumerate(ends)])


def _exact_ssm(s, t):
    """Token by token."""
    form = s["path"].split("_")[1]
    if form == "step":
        t = dict(t, **{name: t[name][:, None] for name in ("x", "dt", "B", "C", "z")
                       if t[name] is not None})
    x, B, C = t["x"], t["B"], t["C"]
    b, n, e = x.shape
    each = e // s["groups"]
    delta = torch.nn.functional.softplus(t["dt"] + t["dt_bias"], threshold=60)
    h = t["state"] if form != "train" else x.new_zeros(b, e, t["A"].shape[1])
    ends = torch.full((b,), n, device=x.device) if s["lengths"] is None else s["lengths"]
    rows = []
    for i in range(n):
        grown = (torch.exp(delta[:, i, :, None] * t["A"]) * h
                 + (delta[:, i] * x[:, i])[..., None] * B[:, i].repeat_interleave(each, 1))
        h = grown if s["lengths"] is None else torch.where((i < ends)[:, None, None], grown, h)
        rows.append((h * C[:, i].repeat_interleave(each, 1)).sum(-1))
    y = torch.stack(rows, 1) + t["D"] * x
    if t["z"] is not None:
        y = y * torch.nn.functional.silu(t["z"])
    if form == "train":
        return y
    if form == "step":
        return y[:, 0], h
    return torch.where((torch.arange(n, device=x.device) < ends[:, None])[..., None], y, 0.0), h


def _exact_norm(s, t):
    rows = t["x"].unflatten(-1, (s["groups"], s["width"])) if t["x"].dim() == 3 else t["x"]
    var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
    y = (rows - mean) / (var + EPS).sqrt()
    if t["weight"] is not None:
        y = y * t["weight"].view(y.shape[-2:]) + t["bias"].view(y.shape[-2:])
    y = y.reshape(t["x"].shape)
    silu = torch.nn.functional.silu
    return y * silu(t["gate"]) if t["gate"] is not None else silu(y) if s["form"] == "silu" else y


def exact(case, seed):
    if case["path"] == "ssm_train" and case["length"] * case["channels"] * case["batch"] * \
            max(16, case["state"]) > 2 ** 30:
        return None       # the graph of the tokens would not fit
    s = prepare(case, seed)
    train = "leaves" in s
    wide = {name: v.detach().double().requires_grad_(train and name in s["leaves"])
            if isinstance(v, torch.Tensor) and v.is_floating_point() else v
            for name, v in s.items()}
    kind = case["path"].split("_")[0]
    with torch.set_grad_enabled(train):
        y = {"conv": _exact_conv, "ssm": _exact_ssm, "norm": _exact_norm}[kind](s, wide)
    if not train:
        return y
    return [y, *torch.autograd.grad(y, [wide[name] for name in s["leaves"]], wide["dy"])]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once; flops: a multiply-add 2, an
    exponential, a division or a square root 1."""
    size = 4 if case["dtype"] == "fp32" else 2
    kind, form = case["path"].split("_")
    tokens = case["batch"] * case["length"]
    if kind == "conv":
        c, k = case["channels"], case["taps"]
        params = c * (k + case["bias"]) * 4
        if form == "train":       # x, dy -> y, dx and the parameters' gradients
            return dict(bytes=4 * tokens * c * size + 2 * params,
                        flops=tokens * c * (6 * k + 8))
        kept = case["batch"] * (k - 1) * c * size
        return dict(bytes=2 * tokens * c * size + 2 * kept + params,
                    flops=tokens * c * (2 * k + 4))
    if kind == "ssm":
        e, m = case["channels"], case["state"]
        rows = 3 + case["gate"]                             # x, dt, (z), y
        shared = 2 * case["groups"] * m * tokens * size
        params = (e * m + 2 * e) * 4
        # per token, channel and n: the decay, the state's step and its product with C
        flops = tokens * e * (7 * m + 12)
        if form == "train":   # x, dt, z, dy, B, C -> y, dx, ddt, dz, dB, dC
            return dict(bytes=tokens * e * size * (2 * rows) + 2 * shared + 2 * params,
                        flops=tokens * e * (24 * m + 30))
        kept = case["batch"] * e * m * 4
        return dict(bytes=tokens * e * size * rows + shared + params + 2 * kept, flops=flops)
    c = case["groups"] * case["width"]
    rows = 2 + (case["form"] == "gate")
    params = 2 * c * 4 if case["affine"] else 0
    if form == "train":           # x, gate, dy -> y, dx, dgate
        return dict(bytes=tokens * c * size * 2 * rows + 2 * params, flops=tokens * c * 30)
    return dict(bytes=tokens * c * size * rows + params, flops=tokens * c * 10)
