"""Host side of ops/layer_norm.py and ops/adamw.py: what is refused before a kernel is launched, and the arithmetic of
moments in 8 bits, in its plain form."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from _train_reference import decode, encode, random_bits
from switchml_b200._native import library_path
from switchml_b200.ops.adamw import FusedAdamW, dequantized, grad_norm
from switchml_b200.ops.layer_norm import FusedLayerNorm, layer_norm


def test_layer_norm_refuses():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        layer_norm(x.half())
    with pytest.raises(ValueError):
        FusedLayerNorm((2, 8))


@pytest.mark.parametrize("where", ["x", "residual", "weight", "bias"])
@pytest.mark.parametrize("grad", [False, True])
def test_layer_norm_refuses_forward_mode(where, grad):
    """Whether anything requires a gradient or not: the result would have no tangent."""
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        args = {"x": torch.ones(2, 8), "residual": torch.ones(2, 8), "weight": torch.ones(8), "bias": torch.ones(8)}
        args[where] = torch.autograd.forward_ad.make_dual(args[where], torch.ones_like(args[where]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(**args)


@pytest.mark.parametrize("call", [lambda x: layer_norm(x), lambda x: grad_norm([x])], ids=["layer_norm", "grad_norm"])
def test_tracers_are_refused(call):
    """They would record the allocation of the result without the kernel that writes it."""
    x = torch.ones(2, 8)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    for options in ({}, {"pre_dispatch": True}, {"tracing_mode": "fake"}):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call, **options)(x)
    with FakeTensorMode(), pytest.raises(RuntimeError, match="cannot be traced"):
        call(torch.ones(2, 8))
    with pytest.raises(ValueError, match="CUDA"):  # (and not for good)
        call(x)


def test_layer_norm_in_c_refuses():
    """Before a pointer is followed."""
    lib = ctypes.CDLL(library_path("libswitchml_train.so"))
    lib.switchml_layer_norm_workspace.restype = ctypes.c_longlong
    p, rows, eps = ctypes.c_void_p(64), ctypes.c_longlong(1), ctypes.c_float(1e-5)

    def forward(features, x=p, y=p, type=0):
        return lib.switchml_layer_norm_forward(x, None, None, None, y, None, None, None, rows, features, eps, type, 0, None)

    def backward(features, dweight=None):
        return lib.switchml_layer_norm_backward(p, None, p, None, p, p, p, dweight, None, None, rows, features, 0, 0, None)

    for features in (-1, 0, 2 ** 30 + 1, 2 ** 31 - 1):
        assert forward(features) == -1 and backward(features) == -1
        assert lib.switchml_layer_norm_workspace(rows, features, 0) == 0
    assert forward(8, x=None) == -1 and forward(8, y=None) == -1 and forward(8, type=2) == -1
    assert backward(8, dweight=p) == -1  # (no workspace)


def test_layer_norm_in_c_refuses_addresses_between_elements():
    lib = ctypes.CDLL(library_path("libswitchml_train.so"))
    rows, eps = ctypes.c_longlong(1), ctypes.c_float(1e-5)
    for type, wtype in ((0, 0), (1, 0), (1, 1)):
        sizes = {"x": type, "residual": type, "weight": wtype, "bias": wtype, "y": type, "sum": type, "mean": 0, "rstd": 0}
        for bad, kind in sizes.items():
            at = {name: ctypes.c_void_p(64 + (name == bad) * (1 if kind else 2)) for name in sizes}
            assert lib.switchml_layer_norm_forward(*at.values(), rows, 8, eps, type, wtype, None) == -1, bad
        sizes = {"dy": type, "dsum": type, "s": type, "weight": wtype, "mean": 0, "rstd": 0, "dx": type, "dweight": wtype, "dbias": wtype,
                 "workspace": 0}
        for bad, kind in sizes.items():
            at = {name: ctypes.c_void_p(64 + (name == bad) * (1 if kind else 2)) for name in sizes}
            assert lib.switchml_layer_norm_backward(*at.values(), rows, 8, type, wtype, None) == -1, bad


class _Tensor(ctypes.Structure):
    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("numel", ctypes.c_longlong), ("place", ctypes.c_uint),
                ("step", ctypes.c_int)]


class _State(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "remainder", "steps", "ticket")] + \
               [("bits", ctypes.c_int), ("seed", ctypes.c_uint), ("first", ctypes.c_ulonglong)]


class _Step(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "decay")] + \
               [("lr_tensor", ctypes.c_void_p), ("norm", ctypes.c_void_p), ("max_norm", ctypes.c_float)]


class _NormTensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("numel", ctypes.c_longlong), ("type", ctypes.c_int)]


def test_adamw_in_c_refuses_addresses():
    """Flat buffers that whole vectors cannot be read from. (Calls that are in order have no tensors: they launch nothing.)"""
    lib = ctypes.CDLL(library_path("libswitchml_train.so"))
    good = {"exp_avg": 4096, "exp_avg_sq": 8192, "exp_avg_scale": 1, "exp_avg_sq_scale": 3, "remainder": 16, "steps": 4, "ticket": 8}

    def step(bits, type, tensors=(), lr_tensor=None, norm=None, **state):
        array = (_Tensor * 2)(*tensors)
        return lib.switchml_adamw_step(array, len(tensors), ctypes.byref(_State(**{**good, **state}, bits=bits)),
                                       ctypes.byref(_Step(lr_tensor=lr_tensor, norm=norm)), type, None)

    for bits, multiple in ((32, 32), (8, 8)):
        for type, size in ((0, 4), (1, 2)):
            assert step(bits, type) == 0 and step(bits, type, exp_avg=64 + multiple, lr_tensor=4, norm=8) == 0
            for name in ("exp_avg", "exp_avg_sq"):
                for off in {1, 4, multiple // 2}:
                    assert step(bits, type, **{name: 4096 + off}) == -1
            assert step(bits, type, remainder=24) == -1
            for name in ("steps", "ticket", "lr_tensor", "norm"):
                assert step(bits, type, **{name: 6}) == -1
            for param, grad in ((64 + size // 2, 64), (64, 64 + size // 2)):
                assert step(bits, type, [(param, grad, 8, 0, 0)]) == -1

    def masters(out, remainder, type, tensors=()):
        return lib.switchml_adamw_masters((_Tensor * 2)(*tensors), len(tensors), ctypes.c_void_p(remainder), ctypes.c_void_p(out), type, None)

    assert masters(32, 16, 1) == 0 and masters(32, None, 0) == 0
    assert masters(16, 16, 1) == -1 and masters(16, None, 0) == -1 and masters(32, 8, 1) == -1
    assert masters(32, 16, 1, [(65, None, 8, 0, 0)]) == -1 and masters(32, 16, 0, [(66, None, 8, 0, 0)]) == -1

    def norm(data, type, workspace=8, ticket=None, out=4):
        return lib.switchml_grad_norm((_NormTensor * 1)((data, 8, type)), 1, ctypes.c_void_p(workspace), ctypes.c_void_p(ticket), ctypes.c_void_p(out), None)

    assert norm(65, 1) == -1 and norm(66, 0) == -1 and norm(64, 0, workspace=4) == -1 and norm(64, 0, ticket=2) == -1 and norm(64, 0, out=2) == -1


def test_grad_norm_in_c_refuses_what_its_workspace_is_not_for():
    """More tiles of 8192 values than one launch counts: tensors that share memory, which no GPU could hold side by side."""
    lib = ctypes.CDLL(library_path("libswitchml_train.so"))
    tensors = (_NormTensor * 384)(*[(64, 1 << 38, 1)] * 384)
    for count in (64, 65, 384):
        assert lib.switchml_grad_norm(tensors, count, ctypes.c_void_p(64), None, ctypes.c_void_p(64), None) == -1


def test_grad_norm_refuses():
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(ValueError, match="CUDA"):
        grad_norm([torch.zeros(3)])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, dtype=torch.int32)])
    with pytest.raises(TypeError):
        grad_norm([torch.eye(3).to_sparse()])


def test_grad_norm_refuses_what_would_want_a_gradient():
    w = torch.ones(3, requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    for bad in (w, g):
        with pytest.raises(RuntimeError, match="has no gradient"):
            grad_norm([bad])
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            grad_norm([bad])
        with pytest.raises(ValueError, match="CUDA"):
            grad_norm([bad.detach()])
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        grad_norm([torch.autograd.forward_ad.make_dual(w.detach(), torch.ones(3))])


@pytest.mark.parametrize("options", [{"state_bits": 16}, {"max_norm": 0.0}, {"max_norm": float("nan")}, {"seed": -1}, {"seed": 1 << 32},
                                     {}, {"lr": -1.0}])
def test_adamw_refuses(options):
    with pytest.raises(ValueError):
        FusedAdamW([torch.nn.Parameter(torch.zeros(4))], **options)


@pytest.mark.parametrize("option", ["amsgrad", "maximize", "differentiable"])
def test_adamw_refuses_options_of_torch_s(option):
    with pytest.raises(ValueError, match=option):
        FusedAdamW([{"params": [torch.nn.Parameter(torch.zeros(4))], option: True}])
    with pytest.raises(ValueError, match="CUDA"):
        FusedAdamW([{"params": [torch.nn.Parameter(torch.zeros(4))], option: False}])


def test_adamw_refuses_types():
    with pytest.raises(TypeError):
        FusedAdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))])


def test_random_bits_are_uniform_and_independent():
    """Means and correlations of 2^18 values lie within 5 standard deviations."""
    n = 1 << 18
    halves = []
    for step in (1, 2, 1000):
        h = random_bits(0, n, 7, step)
        for half in (h & 0xFFFF, h >> 16):
            u = (half.double() + 0.5) / 65536 - 0.5
            assert abs(u.mean()) < 5 / math.sqrt(12 * n)
            for lag in (1, 2, 32, 256):
                assert abs((u[lag:] * u[:-lag]).mean()) < 5 / 12 / math.sqrt(n)
            halves.append(u)
    for i in range(len(halves)):
        for j in range(i):
            assert abs((halves[i] * halves[j]).mean()) < 5 / 12 / math.sqrt(n)


def test_rounding_to_8_bits():
    """Every value becomes one of its two neighbours among the codes, and their mean is the value."""
    torch.manual_seed(0)
    x = torch.randn(64, 32).abs() * torch.exp(3 * torch.randn(64, 1))
    x[0, 0], x[1] = 0.0, 0.0
    flat = x.reshape(-1)
    total, n = torch.zeros(flat.numel(), dtype=torch.float64), 2000
    for step in range(n):
        codes, scales = encode(flat, random_bits(0, flat.numel(), 3, step) & 0xFFFF, False)
        got = decode(codes, scales)
        total += got.double()
        biggest = torch.exp2(torch.floor(torch.log2(x.amax(1, keepdim=True).clamp(min=2.0 ** -100)))) / 128
        step_size = torch.maximum(torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -120))) - 3), biggest * 2.0 ** -9).reshape(-1)
        assert ((got - flat).abs() <= step_size).all()
    assert (got[flat == 0] == 0).all()
    # The mean of n values that are at most a step apart: 6 standard deviations of at most half a step each.
    assert ((total / n - flat).abs() <= 6 * 0.5 / math.sqrt(n) * step_size + 1e-30).all()
    # A block that is on codes already comes back unchanged, whatever the random bits.
    again, scales2 = encode(got, random_bits(5, flat.numel(), 9, 1) & 0xFFFF, False)
    assert torch.equal(decode(again, scales2), got)


def test_second_moments_stay_above_zero():
    v = torch.full((32,), 1e-30)
    v[0] = 1.0
    v[5] = 0.0
    codes, scales = encode(v, torch.zeros(32, dtype=torch.int64), True)
    got = decode(codes, scales)
    assert got[5] == 0 and (got[torch.arange(32) != 5] > 0).all()


def test_dequantized_on_the_cpu():
    codes = torch.arange(0, 120, dtype=torch.uint8).view(4, 30)
    scales = torch.tensor([127, 128, 126, 127], dtype=torch.uint8)
    got = dequantized(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))
    assert torch.equal(got.reshape(-1), decode(codes.view(-1), scales))
