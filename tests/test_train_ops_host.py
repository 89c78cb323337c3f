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


def test_grad_norm_refuses():
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(ValueError, match="CUDA"):
        grad_norm([torch.zeros(3)])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, dtype=torch.int32)])
    with pytest.raises(TypeError):
        grad_norm([torch.eye(3).to_sparse()])


@pytest.mark.parametrize("options", [{"state_bits": 16}, {"max_norm": 0.0}, {"max_norm": float("nan")}, {"seed": -1}, {"seed": 1 << 32},
                                     {}, {"lr": -1.0}])
def test_adamw_refuses(options):
    with pytest.raises(ValueError):
        FusedAdamW([torch.nn.Parameter(torch.zeros(4))], **options)


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
