"""CPU tests of the recurrent mixers' operators: the plain float64 forms against autograd and
differences, the operators' refusals, and the C ABI's (which run where no GPU is visible)."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from lizard_reproduction_amd import _lib, kernels
from tests import mixers_reference as ref
from tests.test_capi import lib, no_gpu, refused  # noqa: F401  (lib: a fixture)


@pytest.fixture(autouse=True)
def gpu_as_it_is(monkeypatch):
    """The presence of a GPU asked anew (kernels.py remembers one, and other tests say so)."""
    monkeypatch.setattr(kernels, "_GPU_SEEN", False)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def _agree(got, want):
    assert set(got) == set(want)
    for name in got:
        torch.testing.assert_close(got[name], want[name], rtol=1e-10, atol=1e-10, msg=name)


def _grads(outputs, names):
    return {n: outputs["d" + n][0] for n in names}


# --- the plain forms: their gradients are autograd's of the same definitions ----------

@pytest.mark.parametrize("taps, act, length", [(4, True, 9), (3, False, 2), (1, True, 5), (2, True, 1)])
def test_plain_conv_gradients(taps, act, length):
    g = torch.Generator().manual_seed(0)
    x, w, b = _randn(g, 2, length, 5), _randn(g, 5, taps), _randn(g, 5)
    dy = _randn(g, 2, length, 5)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = F.conv1d(F.pad(x.transpose(1, 2), (taps - 1, 0)), w[:, None], b, groups=5).transpose(1, 2)
    y = F.silu(y) if act else y
    got = ref.conv(x, w, b, act, dy)
    torch.testing.assert_close(got["y"][0], y.detach(), rtol=1e-10, atol=1e-10)
    want = dict(zip(("x", "weight", "bias"), torch.autograd.grad(y, leaves, dy)))
    _agree(_grads(got, want), want)


def _ssm_case(length=7, e=6, n=3, groups=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=_randn(g, 2, length, e), dt=_randn(g, 2, length, e),
             A=-torch.rand(e, n, generator=g, dtype=torch.float64),
             B=_randn(g, 2, length, groups, n), C=_randn(g, 2, length, groups, n), D=_randn(g, e),
             z=_randn(g, 2, length, e), dt_bias=_randn(g, e))
    return c, _randn(g, 2, length, e)


def _ssm_autograd(c, softplus=True):
    e, groups = c["x"].shape[2], c["B"].shape[2]
    delta = c["dt"] + c["dt_bias"]
    delta = F.softplus(delta, threshold=60) if softplus else delta
    h, rows = 0, []
    for t in range(c["x"].shape[1]):
        B, C = (c[k][:, t].repeat_interleave(e // groups, 1) for k in ("B", "C"))
        h = torch.exp(delta[:, t, :, None] * c["A"]) * h + (delta * c["x"])[:, t, :, None] * B
        rows.append((h * C).sum(-1))
    return (torch.stack(rows, 1) + c["D"] * c["x"]) * F.silu(c["z"])


@pytest.mark.parametrize("softplus", [True, False])
def test_plain_ssm_gradients(softplus):
    c, dy = _ssm_case()
    for t in c.values():
        t.requires_grad_()
    y = _ssm_autograd(c, softplus)
    got = ref.ssm(**c, softplus=softplus, dy=dy)
    torch.testing.assert_close(got["y"][0], y.detach(), rtol=1e-10, atol=1e-10)
    want = dict(zip(c, torch.autograd.grad(y, list(c.values()), dy)))
    _agree(_grads(got, want), want)


def test_plain_ssm_gradients_are_differences():
    """Central differences along a random direction of every operand: the third
    derivative's share is h^2 = 1e-10 of order one."""
    c, dy = _ssm_case(seed=3)
    grads = ref.ssm(**c, dy=dy)
    g = torch.Generator().manual_seed(4)
    for name in c:
        v = _randn(g, *c[name].shape)
        ends = [(ref.ssm(**dict(c, **{name: c[name] + s * 1e-5 * v}))["y"][0] * dy).sum()
                for s in (1, -1)]
        want = (ends[0] - ends[1]) / 2e-5
        got = (grads["d" + name][0] * v).sum()
        assert abs(got - want) <= 1e-6 * max(1.0, abs(want)), name


@pytest.mark.parametrize("gate, act", [(True, True), (True, False), (False, True), (False, False)])
def test_plain_norm_gradients(gate, act):
    g = torch.Generator().manual_seed(0)
    x, w, b, z, dy = (_randn(g, *s) for s in ((3, 4, 12), (12,), (12,), (3, 4, 12), (3, 4, 12)))
    leaves = dict(x=x, weight=w, bias=b, gate=z) if gate else dict(x=x, weight=w, bias=b)
    for t in leaves.values():
        t.requires_grad_()
    o = F.group_norm(x.reshape(12, 12), 3, w, b, 1e-5).view(3, 4, 12)
    f = F.silu if act else (lambda t: t)
    y = o * f(z) if gate else f(o)
    got = ref.norm(x, 3, w, b, z if gate else None, act, dy=dy)
    torch.testing.assert_close(got["y"][0], y.detach(), rtol=1e-10, atol=1e-10)
    want = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    _agree(_grads(got, want), want)


# --- refusals of the operators: made before anything is launched ------------------------

def _f(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_ssm_refusals():
    good = dict(x=_f(2, 5, 8), dt=_f(2, 5, 8), A=_f(8, 4), B=_f(2, 5, 4), C=_f(2, 5, 4))

    def bad(match, **over):
        with pytest.raises(ValueError, match=match):
            kernels.ssm(**dict(good, **over))
    bad("ROCm GPU")
    bad("x must be", x=_f(5, 8))
    bad("dt must be", dt=_f(2, 5, 7))
    bad("z must be", z=_f(2, 4, 8))
    bad("A must be", A=_f(7, 4))
    bad("A must be", A=_f(8, 65))
    bad("A must be", A=_f(8, 0))
    bad("A must be", A=None)
    bad("D must be", D=_f(7))
    bad("dt_bias must be", dt_bias=_f(8, 1))
    bad("D must be a floating", D=torch.zeros(8, dtype=torch.int32))
    bad("B and C must be", B=_f(2, 5, 3), C=_f(2, 5, 3))
    bad("B and C must be", B=_f(2, 5, 3, 4), C=_f(2, 5, 3, 4))
    bad("B and C must be", B=_f(2, 5, 2, 4), C=_f(2, 5, 1, 4))
    bad("bf16 or fp32", x=_f(2, 5, 8, dtype=torch.float16))
    bad("bf16 or fp32", B=_f(2, 5, 4, dtype=torch.float64))
    bad("must be a tensor", B=None)


def test_ssm_prefill_and_step_refusals():
    good = dict(x=_f(2, 5, 8), dt=_f(2, 5, 8), A=_f(8, 4), B=_f(2, 5, 4), C=_f(2, 5, 4))
    with pytest.raises(ValueError, match="ROCm GPU"):
        kernels.ssm_prefill(**good, state=_f(2, 8, 4))
    step = dict(x=_f(2, 8), dt=_f(2, 8), A=_f(8, 4), B=_f(2, 4), C=_f(2, 4), state=_f(2, 8, 4))
    with pytest.raises(ValueError, match="ROCm GPU"):
        kernels.ssm_decode_step(**step)
    with pytest.raises(ValueError, match="x must be"):
        kernels.ssm_decode_step(**dict(step, x=_f(2, 1, 8)))
    with pytest.raises(ValueError, match="B and C must be"):
        kernels.ssm_decode_step(**dict(step, B=_f(3, 4), C=_f(3, 4)))


@pytest.fixture
def as_gpu(monkeypatch):
    """The checks behind the device's, on CPU tensors; a launch would fail."""
    monkeypatch.setattr(kernels, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(kernels._ops, "load", lambda: pytest.fail("a bad call reached the library"))


def test_states_and_lengths_are_checked(as_gpu):
    seq = dict(x=_f(2, 5, 8), dt=_f(2, 5, 8), A=_f(8, 4), B=_f(2, 5, 4), C=_f(2, 5, 4))
    for state in (_f(2, 8, 3), _f(2, 8, 4, dtype=torch.bfloat16), "state"):
        with pytest.raises(ValueError, match="state must be"):
            kernels.ssm_prefill(**seq, state=state)
    for lengths in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), [5, 5]):
        with pytest.raises(ValueError, match="lengths must be"):
            kernels.ssm_prefill(**seq, lengths=lengths)
        with pytest.raises(ValueError, match="lengths must be"):
            kernels.short_conv_prefill(seq["x"], _f(8, 4), lengths=lengths)
    step = dict(x=_f(2, 8), dt=_f(2, 8), A=_f(8, 4), B=_f(2, 4), C=_f(2, 4))
    for state in (_f(2, 4, 8).transpose(1, 2), _f(2, 8, 4, dtype=torch.float64), None):
        with pytest.raises(ValueError, match="state must be"):
            kernels.ssm_decode_step(**step, state=state)
    with pytest.raises(ValueError, match="require gradients"):
        kernels.ssm_decode_step(**step, state=_f(2, 8, 4).requires_grad_())
    for state in (_f(2, 2, 8), _f(2, 3, 8, dtype=torch.bfloat16), _f(2, 8, 3).transpose(1, 2)):
        with pytest.raises(ValueError, match="state must be"):
            kernels.short_conv_decode_step(_f(2, 8), _f(8, 4), state)
    with pytest.raises(ValueError, match="state must be"):
        kernels.short_conv_prefill(seq["x"], _f(8, 4), state=_f(2, 4, 8))


def test_conv_refusals(as_gpu):
    def bad(match, x=_f(2, 5, 8), w=_f(8, 4), *more):
        with pytest.raises(ValueError, match=match):
            kernels.short_conv(x, w, *more)
    bad("x must be", _f(2, 8))
    bad("weight must be", w=_f(8, 5))
    bad("weight must be", w=_f(8, 0))
    bad("weight must be", w=_f(7, 4))
    bad("weight must be", w=_f(8, 1, 4))
    bad("bias must be", _f(2, 5, 8), _f(8, 4), _f(4))
    bad("activation", _f(2, 5, 8), _f(8, 4), None, "gelu")
    bad("bf16 or fp32", _f(2, 5, 8, dtype=torch.float64))


def test_norm_refusals(as_gpu):
    def bad(match, x=_f(2, 5, 8), groups=2, **more):
        with pytest.raises(ValueError, match=match):
            kernels.group_norm(x, groups, **more)
    bad("groups must be", groups=3)
    bad("groups must be", groups=0)
    bad("groups must be", groups=2.0)
    bad("x must be", _f(8), None)
    bad("channels expected", _f(2, 8193), 1)
    bad("gate must be", gate=_f(2, 5, 4))
    bad("weight must be", weight=_f(4))
    bad("bias must be", bias=_f(2, 4))
    bad("activation", activation="relu")
    bad("eps", eps=-1.0)
    bad("eps", eps=float("nan"))
    bad("bf16 or fp32", _f(2, 8, dtype=torch.float16))


def test_transforms_are_refused(monkeypatch):
    monkeypatch.setattr(kernels, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(kernels._ops, "plain", lambda: False)
    with pytest.raises(RuntimeError, match="transforms"):
        kernels.short_conv(_f(2, 5, 8), _f(8, 4))
    with pytest.raises(RuntimeError, match="transforms"):
        kernels.group_norm(_f(2, 5, 8), 2)
    with pytest.raises(RuntimeError, match="transforms"):
        kernels.ssm(_f(2, 5, 8), _f(2, 5, 8), _f(8, 4), _f(2, 5, 4), _f(2, 5, 4))


def test_limits_are_the_modules():
    from lizard_reproduction_amd import _ops
    m = _ops.load()
    assert (m.CONV_MAX_TAPS, m.SSM_MAX_STATE, m.NORM_MAX_WIDTH) == (
        kernels.CONV_MAX_TAPS, kernels.SSM_MAX_STATE, kernels.NORM_MAX_WIDTH)


# --- refusals of the C entry points ---------------------------------------------------------

P = ctypes.c_void_p(16)


def _ssm_args(**over):
    a = _lib.SsmArgs(x=16, dt=16, B=16, C=16, A=16, batch=2, length=40, channels=8, state=4, groups=1,
                     x_token=8, dt_token=8, z_token=8, B_token=4, C_token=4)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@no_gpu
def test_ssm_entry_points_refuse(lib):  # noqa: F811
    def fwd(needle, **over):
        refused(lib, lib.lz_ssm_fwd(_ssm_args(**over), None, None, None, P, None, P, 1 << 30, None),
                needle)
        refused(lib, lib.lz_ssm_bwd(_ssm_args(**over), P, P, P, P, P, P, P, P, P, P, P, 1 << 30, None),
                needle)
    refused(lib, lib.lz_ssm_fwd(None, None, None, None, P, None, P, 0, None), b"null")
    fwd(b"null", x=None)
    fwd(b"null", A=None)
    fwd(b"positive", batch=0)
    fwd(b"positive", length=0)
    fwd(b"positive", state=-1)
    fwd(b"beyond 64", state=65)
    fwd(b"divide", groups=3)
    fwd(b"strides", x_token=-1)
    fwd(b"strides", B_token=(1 << 24) + 1)
    fwd(b"strides", C_group=-4)
    fwd(b"strides", x_batch=-8)
    fwd(b"tokens", batch=2048, length=1 << 20)
    fwd(b"beyond", channels=(1 << 24) + 1)
    refused(lib, lib.lz_ssm_fwd(_ssm_args(), None, None, None, None, None, P, 1 << 30, None), b"null")
    refused(lib, lib.lz_ssm_bwd(_ssm_args(z=16), P, P, P, P, None, P, P, P, P, P, P, 1 << 30, None),
            b"null")
    long = dict(batch=1, length=4096, channels=64)
    need = lib.lz_ssm_fwd_workspace_bytes(1, 4096, 64, 4, 1)
    assert need > 0     # one workgroup's channels: the sequence is split
    refused(lib, lib.lz_ssm_fwd(_ssm_args(**long), None, None, None, P, None, P, need - 1, None),
            b"workspace")
    refused(lib, lib.lz_ssm_fwd(_ssm_args(**long), None, None, None, P, None, None, need, None),
            b"workspace")
    need = lib.lz_ssm_bwd_workspace_bytes(1, 4096, 64, 4, 1)
    refused(lib, lib.lz_ssm_bwd(_ssm_args(**long), P, P, P, P, P, P, P, P, P, P, P, need - 1, None),
            b"workspace")
    refused(lib, lib.lz_ssm_decode_step(_ssm_args(), None, P, None), b"null")
    refused(lib, lib.lz_ssm_decode_step(_ssm_args(batch=70000), P, P, None), b"grid")


@no_gpu
def test_conv_entry_points_refuse(lib):  # noqa: F811
    def fwd(needle, x=P, w=P, y=P, b=2, n=5, c=8, k=4, xb=40, xt=8):
        refused(lib, lib.lz_short_conv_fwd(x, xb, xt, w, None, None, None, None, y, b, n, c, k, 1, 1,
                                           None), needle)
    fwd(b"null", x=None)
    fwd(b"null", w=None)
    fwd(b"null", y=None)
    fwd(b"positive", c=0)
    fwd(b"taps", k=5)
    fwd(b"strides", xt=-1)
    fwd(b"strides", xb=-1)
    fwd(b"tokens", b=2048, n=1 << 20)
    refused(lib, lib.lz_short_conv_decode_step(P, 8, P, None, None, P, 2, 8, 4, 1, 1, None), b"null")
    need = lib.lz_short_conv_bwd_workspace_bytes(2, 5, 8, 4)
    assert need > 0
    refused(lib, lib.lz_short_conv_bwd(P, 40, 8, P, None, P, P, P, None, 2, 5, 8, 4, 1, 1, P, need - 1,
                                       None), b"workspace")


@no_gpu
def test_norm_entry_points_refuse(lib):  # noqa: F811
    def args(**over):
        a = _lib.GroupNormArgs(x=16, batch=2, length=5, groups=2, width=8, eps=1e-5)
        for k, v in over.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    def fwd(needle, **over):
        refused(lib, lib.lz_group_norm_fwd(args(**over), P, None), needle)
    refused(lib, lib.lz_group_norm_fwd(None, P, None), b"null")
    refused(lib, lib.lz_group_norm_fwd(args(), None, None), b"null")
    fwd(b"null", x=None)
    fwd(b"positive", width=0)
    fwd(b"beyond 8192", width=8193)
    fwd(b"strides", x_token=-1)
    fwd(b"eps", eps=-1.0)
    need = lib.lz_group_norm_bwd_workspace_bytes(2, 5, 2, 8)
    assert need > 0
    refused(lib, lib.lz_group_norm_bwd(args(), P, P, None, P, P, P, need - 1, None), b"workspace")
    refused(lib, lib.lz_group_norm_bwd(args(gate=16), P, P, None, P, P, P, need, None), b"null")


def test_workspaces_of_refused_sizes_are_empty(lib):  # noqa: F811
    assert lib.lz_ssm_bwd_workspace_bytes(1, 16, 8, 65, 1) == 0
    assert lib.lz_ssm_states_bytes(0, 16, 8, 4, 1) == 0
    assert lib.lz_ssm_states_bytes(2, 17, 8, 4, 0) == 2 * 2 * 8 * 4 * 4
    assert lib.lz_ssm_states_bytes(2, 17, 8, 4, 1) == 2 * (2 * 4 + 17) * 8 * 4
    assert lib.lz_group_norm_bwd_workspace_bytes(1, 1, 1, 8193) == 0
    # sequences and channels that fill the GPU by themselves are not split
    assert lib.lz_ssm_fwd_workspace_bytes(64, 2048, 4096, 16, 1) == 0
