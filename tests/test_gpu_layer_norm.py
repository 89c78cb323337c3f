"""ops/layer_norm.py against its formulas in 64 bits."""
import ctypes

import pytest
import torch
import torch.utils.checkpoint
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from _train_reference import check, layer_norm64
from switchml_b200._native import library_path
from switchml_b200.ops.layer_norm import FusedLayerNorm, layer_norm

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(shape, dtype, wtype, residual, affine, seed=0, mean=0.5, offset=0):
    gen = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=gen)

    def place(t):  # on the GPU, `offset` elements behind an aligned address
        flat = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        return flat[offset:].view(t.shape).copy_(t)

    n = shape[-1]
    data = {"x": (rand(*shape) * 2 + mean).to(dtype), "residual": rand(*shape).to(dtype) if residual else None,
            "weight": (1 + 0.3 * rand(n)).to(wtype) if affine else None, "bias": (0.3 * rand(n)).to(wtype) if affine else None,
            "dy": rand(*shape).to(dtype), "ds": rand(*shape).to(dtype) if residual else None}
    return data, {k: None if v is None else place(v) for k, v in data.items()}


def run_and_check(data, dev, eps, use_ds):
    leaves = [dev[k].requires_grad_() for k in ("x", "residual", "weight", "bias") if dev[k] is not None]
    out = layer_norm(dev["x"], dev["weight"], dev["bias"], eps, residual=dev["residual"])
    outs = (out,) if dev["residual"] is None else out
    grads = (dev["dy"],) if dev["residual"] is None or not use_ds else (dev["dy"], dev["ds"])
    got = dict(zip([k for k in ("x", "residual", "weight", "bias") if dev[k] is not None],
                   torch.autograd.grad(outs[:len(grads)], leaves, grads)))
    values, bounds = layer_norm64(data["x"], data["residual"], data["weight"], data["bias"], eps, data["dy"],
                                  data["ds"] if len(grads) > 1 else None)
    check("y", outs[0], values["y"].reshape(outs[0].shape), bounds["y"].reshape(outs[0].shape))
    if dev["residual"] is not None:
        assert torch.equal(outs[1].cpu(), values["s"])
        assert torch.equal(got["x"], got["residual"])
    check("dx", got["x"], values["dx"].reshape(got["x"].shape), bounds["dx"].reshape(got["x"].shape))
    if dev["weight"] is not None:
        check("dweight", got["weight"], values["dweight"], bounds["dweight"])
        check("dbias", got["bias"], values["dbias"], bounds["dbias"])
        assert got["weight"].dtype == dev["weight"].dtype
    return outs, got


FEATURES = [1, 2, 7, 8, 31, 33, 64, 127, 256, 257, 511, 512, 768, 1000, 1021, 1024, 1025, 2048, 4096, 4100, 5000, 8192, 8200, 16384,
            20000, 33000, 70001]


@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("features", FEATURES)
def test_features(features, dtype, wtype):
    rows = 5 if features > 4096 else 37
    run_and_check(*make((rows, features), dtype, wtype, features % 2 == 0, True, seed=features), 1e-12 if features > 1 else 1e-5, features % 4 == 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 8, 147, 149, 593, 4099])
def test_rows(rows, residual, dtype):
    run_and_check(*make((rows, 264), dtype, F32, residual, True, seed=rows), 1e-5, True)


@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,features", [(300, 12000), (301, 12002), (299, 8193), (150, 16385), (160, 20001), (80, 33000), (75, 65535)])
def test_many_rows_that_several_blocks_share(rows, features, dtype, wtype):
    run_and_check(*make((rows, features), dtype, wtype, rows % 2 == 0, True, seed=rows), 1e-5, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 36, 37, 38, 73, 75])
def test_rows_around_the_number_of_clusters(rows, dtype):
    run_and_check(*make((rows, 20002), dtype, F32, True, rows % 2 == 0, seed=rows), 1e-5, False)


@pytest.mark.parametrize("features", [8200, 12000, 20001, 40001])
def test_long_rows_on_two_streams_and_replayed(features):
    """Every run adds in the same order."""
    _, dev = make((301, features), BF16, F32, True, True)
    leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias")]

    def once():
        y, s = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
        return (y, s) + torch.autograd.grad((y, s), leaves, (dev["dy"], dev["ds"]))

    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for stream in streams:
        with torch.cuda.stream(stream):
            results.append(once())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for _ in range(2):
        for o in out:
            o.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(out, *results))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("features", [512, 4096, 12000])
def test_in_c_with_a_workspace_at_an_odd_address(features, dtype):
    lib = ctypes.CDLL(library_path("libswitchml_train.so"))
    lib.switchml_layer_norm_workspace.restype = ctypes.c_longlong
    data, dev = make((50, features), dtype, F32, False, True)
    x, dy, w, size = dev["x"], dev["dy"], dev["weight"], ctypes.c_longlong(50)
    kind = 0 if dtype == F32 else 1
    space = torch.empty(lib.switchml_layer_norm_workspace(size, features, kind) + 1, device="cuda")
    mean, rstd, dx, dw, db = (torch.empty_like(t) for t in (x[:, 0].float(), x[:, 0].float(), x, w, w))
    y = torch.empty_like(x)

    def at(t):
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.switchml_layer_norm_forward(at(x), None, at(w), at(dev["bias"]), at(y), None, at(mean), at(rstd), size, features,
                                           ctypes.c_float(1e-5), kind, 0, stream) == 0
    assert lib.switchml_layer_norm_backward(at(dy), None, at(x), at(w), at(mean), at(rstd), at(dx), at(dw), at(db), at(space[1:]), size,
                                            features, kind, 0, stream) == 0
    values, bounds = layer_norm64(data["x"], None, data["weight"], data["bias"], 1e-5, data["dy"])
    for name, got in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
        check(name, got, values[name], bounds[name])


@pytest.mark.parametrize("features", [12000, 20001])
def test_values_that_are_not_finite_in_a_long_row(features):
    data, dev = make((40, features), BF16, F32, False, True)
    dev["x"][2, 5], dev["x"][4, features - 1] = float("nan"), float("inf")
    y = layer_norm(dev["x"], dev["weight"], dev["bias"])
    assert y[2].isnan().all() and y[4].isnan().all()
    values, bounds = layer_norm64(data["x"], None, data["weight"], data["bias"], 1e-5)
    keep = [r for r in range(40) if r not in (2, 4)]
    check("y", y[keep], values["y"][keep], bounds["y"][keep])


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("features", [96, 1000, 1024, 4096, 6000])
def test_addresses_behind_an_aligned_one(features, offset):
    for dtype, wtype in ((F32, F32), (BF16, BF16), (BF16, F32)):
        run_and_check(*make((19, features), dtype, wtype, True, True, seed=offset, offset=offset), 1e-6, True)


def test_only_some_tensors_behind_an_aligned_address():
    for name in ("x", "residual", "weight", "bias", "dy", "ds"):
        data, dev = make((9, 1024), BF16, F32, True, True)
        flat = torch.empty(dev[name].numel() + 1, dtype=dev[name].dtype, device="cuda")
        dev[name] = flat[1:].view(dev[name].shape).copy_(dev[name])
        run_and_check(data, dev, 1e-6, True)


@pytest.mark.parametrize("shape", [(1024,), (2, 3, 5, 320), (4, 0, 64), (0, 64)])
@pytest.mark.parametrize("affine", [False, True])
def test_shapes(shape, affine):
    run_and_check(*make(shape, F32, F32, True, affine), 1e-5, True)


def test_weight_or_bias_alone():
    for missing in ("weight", "bias"):
        data, dev = make((11, 320), BF16, BF16, False, True)
        data[missing] = dev[missing] = None
        leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias") if dev[k] is not None]
        y = layer_norm(dev["x"], dev["weight"], dev["bias"])
        got = torch.autograd.grad(y, leaves, dev["dy"])
        values, bounds = layer_norm64(data["x"], None, data["weight"], data["bias"], 1e-5, data["dy"])
        check("y", y, values["y"], bounds["y"])
        other = "dweight" if missing == "bias" else "dbias"
        check("dx", got[0], values["dx"], bounds["dx"])
        check(other, got[1], values[other], bounds[other] * (1 if missing == "bias" else 1) + 2.0 ** -8 * values[other].abs())


def test_mean_far_larger_than_the_spread():
    """A variance from squares would have nothing left."""
    run_and_check(*make((16, 1024), F32, F32, False, True, mean=3e3), 1e-12, False)


def test_rows_without_spread():
    """All values the same: the variance is 0, y the bias and the gradient bounded by eps."""
    x = torch.full((3, 640), 1.75, device="cuda", requires_grad=True)
    w, b = torch.randn(640, device="cuda"), torch.randn(640, device="cuda")
    y = layer_norm(x, w, b, 1e-5)
    assert torch.equal(y, b.expand(3, 640))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("n", [96, 100, 101, 1000, 1001, 6600])
def test_large_rows_without_spread(n):
    """2^112 everywhere: centred values are 0, but what lies behind a row's end, taken as 0, would be infinitely far from the mean."""
    x = torch.full((5, n), 2.0 ** 112, device="cuda", requires_grad=True)
    w, dy = (1 + torch.rand(n)).requires_grad_(), torch.randn(5, n)
    y = layer_norm(x, w.cuda(), None, 1e-12)
    dx, = torch.autograd.grad(y, x, dy.cuda())
    assert not y.any()
    g = dy.double() * w.detach().double()
    want = 1e6 * (g - g.mean(1, keepdim=True))
    bound = 1e6 * 2.0 ** -24 * (n / 32 + 24) * (g.abs() + g.abs().mean(1, keepdim=True))
    check("dx", dx, want, bound)


def test_values_that_are_not_finite_stay_in_their_row():
    data, dev = make((6, 1024), BF16, F32, False, True)
    dev["x"][2, 5], dev["x"][4, 1000] = float("nan"), float("inf")
    y = layer_norm(dev["x"], dev["weight"], dev["bias"])
    assert y[2].isnan().all() and y[4].isnan().all()
    values, bounds = layer_norm64(data["x"], None, data["weight"], data["bias"], 1e-5)
    keep = [0, 1, 3, 5]
    check("y", y[keep], values["y"][keep], bounds["y"][keep])


def test_gradients_against_differences():
    """d(sum y dy) along a direction is the gradient along it: central differences of the 64-bit formula."""
    data, dev = make((4, 96), F32, F32, True, True)
    run_and_check(data, dev, 1e-5, True)
    leaves = [dev[k] for k in ("x", "weight", "bias")]
    y, s = layer_norm(dev["x"], dev["weight"], dev["bias"], 1e-5, residual=dev["residual"])
    got = torch.autograd.grad((y, s), leaves, (dev["dy"], dev["ds"]))

    def loss(x, w, b):
        v = x + data["residual"].double()
        mean = v.mean(1, keepdim=True)
        out = (v - mean) / ((v - mean).square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b
        return (out * data["dy"].double()).sum() + (v * data["ds"].double()).sum()

    gen = torch.Generator().manual_seed(3)
    at = [data[k].double() for k in ("x", "weight", "bias")]
    for i in range(3):
        u = torch.randn(at[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        plus, minus = [a.clone() for a in at], [a.clone() for a in at]
        plus[i] += h * u
        minus[i] -= h * u
        slope = (loss(*plus) - loss(*minus)) / (2 * h)
        along = (got[i].double().cpu() * u).sum()
        # s is rounded to float32 in the kernel, and the differences leave h^2 of the third derivative.
        scale = (got[i].double().cpu() * u).abs().sum()
        assert abs(slope - along) <= 1e-5 * scale


def test_gradients_that_are_not_contiguous_or_not_there():
    data, dev = make((8, 256), F32, F32, True, True)
    x = dev["x"].requires_grad_()
    y, s = layer_norm(x, dev["weight"], dev["bias"], residual=dev["residual"])
    assert torch.equal(torch.autograd.grad(s.sum(), x, retain_graph=True)[0], torch.ones_like(x))
    values, bounds = layer_norm64(data["x"], data["residual"], data["weight"], data["bias"], 1e-5, torch.ones(8, 256))
    check("dx", torch.autograd.grad(y.sum(), x, retain_graph=True)[0], values["dx"], bounds["dx"])  # an expanded gradient
    dy = torch.randn(256, 8, device="cuda").t()
    values, bounds = layer_norm64(data["x"], data["residual"], data["weight"], data["bias"], 1e-5, dy.cpu())
    check("dx", torch.autograd.grad(y, x, dy)[0], values["dx"], bounds["dx"])


def test_inputs_that_are_not_contiguous():
    data, dev = make((2, 6, 128), F32, F32, True, True)
    x = dev["x"].transpose(0, 1).contiguous().transpose(0, 1)
    x = x.detach().requires_grad_()
    assert not x.is_contiguous()
    w = torch.stack([dev["weight"], dev["bias"]], 1)
    y, s = layer_norm(x, w[:, 0], w[:, 1], residual=dev["residual"])
    values, bounds = layer_norm64(data["x"], data["residual"], data["weight"], data["bias"], 1e-5, data["dy"])
    check("y", y, values["y"].reshape(y.shape), bounds["y"].reshape(y.shape))
    check("dx", torch.autograd.grad(y, x, dev["dy"])[0], values["dx"].reshape(x.shape), bounds["dx"].reshape(x.shape))


def test_residual_that_is_the_input_itself():
    x = torch.randn(6, 320, device="cuda", requires_grad=True)
    dy = torch.randn(6, 320, device="cuda")
    y, s = layer_norm(x, residual=x)
    got, = torch.autograd.grad(y, x, dy)
    values, bounds = layer_norm64(x.detach().cpu(), x.detach().cpu(), None, None, 1e-5, dy.cpu())
    check("y", y, values["y"], bounds["y"])
    check("dx", got, 2 * values["dx"], 2 * bounds["dx"])


def test_gradients_of_input_and_residual_are_two_tensors():
    data, dev = make((6, 320), F32, F32, True, True)
    x, r = dev["x"].requires_grad_(), dev["residual"].requires_grad_()
    layer_norm(x, dev["weight"], dev["bias"], residual=r)[0].backward(dev["dy"])
    kept = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, kept)


@pytest.mark.parametrize("n", [8192, 8200])
def test_more_values_than_31_bits_count(n):
    """The last rows of 2^31 and some values, forward and backward, against the formula."""
    rows = 262150
    x = torch.empty(rows, n, device="cuda", dtype=BF16).normal_().requires_grad_()
    w = (1 + 0.1 * torch.randn(n, device="cuda")).requires_grad_()
    y = layer_norm(x, w)
    dy = torch.zeros_like(y)
    dy[-3:] = torch.randn(3, n, device="cuda")
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    values, bounds = layer_norm64(x[-3:].detach().cpu(), None, w.detach().cpu(), None, 1e-5, dy[-3:].cpu())
    check("y", y[-3:], values["y"], bounds["y"])
    check("dx", dx[-3:], values["dx"], bounds["dx"])
    check("dweight", dw, values["dweight"], bounds["dweight"])
    assert not dx[:-3].any()


def test_the_same_bits_in_every_run():
    _, dev = make((4099, 1024), BF16, F32, True, True)
    leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias")]

    def once():
        y, s = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
        return (y, s) + torch.autograd.grad((y, s), leaves, (dev["dy"], dev["ds"]))

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_another_stream_and_two_at_once():
    data, dev = make((2000, 1024), BF16, F32, True, True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias")]
            y, s = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
            results.append((y, s) + torch.autograd.grad((y, s), leaves, (dev["dy"], dev["ds"])))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_captured_and_replayed():
    data, dev = make((64, 1024), BF16, F32, True, True)
    leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias")]

    def once():
        y, s = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
        return (y,) + torch.autograd.grad((y, s), leaves, (dev["dy"], dev["ds"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = once()
        graphs.append((graph, out))
    with torch.no_grad():
        dev["x"].copy_(torch.randn_like(dev["x"]))
    want = once()
    for graph, out in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for graph, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_under_autocast():
    """Inputs are cast to the type of autocast, weights stay float32."""
    x = torch.randn(5, 256, device="cuda", requires_grad=True)
    r = torch.randn(5, 256, device="cuda").bfloat16()
    layer = FusedLayerNorm(256, eps=1e-12).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x, r)
    assert y.dtype == BF16
    values, bounds = layer_norm64(x.detach().bfloat16().cpu(), r.cpu(), layer.weight.detach().cpu(), layer.bias.detach().cpu(), 1e-12)
    check("y", y, values["y"], bounds["y"])
    y.sum().backward()
    assert x.grad.dtype == F32 and layer.weight.grad.dtype == F32


def test_refusals_on_the_gpu():
    x = torch.randn(4, 64, device="cuda")
    for error, args, kw in ((TypeError, (x.half(),), {}), (TypeError, (x.double(),), {}),
                            (TypeError, (x, torch.ones(64, device="cuda").bfloat16()), {}),
                            (ValueError, (x, torch.ones(32, device="cuda")), {}), (ValueError, (x, torch.ones(64)), {}),
                            (TypeError, (x.bfloat16(), torch.ones(64, device="cuda"), torch.ones(64, device="cuda").bfloat16()), {}),
                            (ValueError, (x,), {"residual": x[:3]}), (ValueError, (x,), {"residual": x.bfloat16()}),
                            (ValueError, (x,), {"eps": -1.0}), (ValueError, (x[:, :0],), {}), (ValueError, (x.cpu(),), {})):
        with pytest.raises(error):
            layer_norm(*args, **kw)
    x.requires_grad_()
    y = layer_norm(x)
    with pytest.raises(RuntimeError, match="gradient of its gradient"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)


def test_module_in_the_place_of_torch_s():
    torch.manual_seed(0)
    plain, fused = torch.nn.LayerNorm(320).cuda(), FusedLayerNorm(320).cuda()
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(7, 320, device="cuda")
    torch.testing.assert_close(fused(x), plain(x))
    with pytest.raises(ValueError):
        FusedLayerNorm((4, 320))
    with pytest.raises(ValueError):
        fused(x[:, :319])


def test_tracers_of_a_backward_pass_are_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    dy = torch.randn(4, 64, device="cuda")
    y = layer_norm(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(dy)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(FusedLayerNorm(64).cuda(), (x,))
    assert torch.autograd.grad(y, x, dy)[0].isfinite().all()


def test_gradients_with_a_tangent_are_refused():
    """Forward mode over reverse mode: the gradient would come without its tangent."""
    x, r = (torch.randn(4, 64, device="cuda", requires_grad=True) for _ in range(2))
    dy = torch.randn(4, 64, device="cuda")
    y, s = layer_norm(x, residual=r)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(dy, dy.clone())
        for out in (y, s):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, dual, retain_graph=True)
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(torch.autograd.forward_ad.make_dual(x.detach(), dy))
        torch.autograd.grad(y, x, dy)


def backward_through_hooks(change, residual=False):
    """Gradients of x, weight and bias where hooks give back `change` of every saved tensor."""
    _, dev = make((6, 64), BF16, F32, residual, True)
    leaves = [dev[k].requires_grad_() for k in ("x", "weight", "bias")]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        out = layer_norm(dev["x"], dev["weight"], dev["bias"], residual=dev["residual"])
    return torch.autograd.grad(out[0] if residual else out, leaves, dev["dy"])


@pytest.mark.parametrize("residual", [False, True])
def test_saved_tensors_that_come_back_in_another_layout(residual):
    def apart(t):
        return torch.stack([t, t + 1], -1)[..., 0]

    assert all(torch.equal(a, b) for a, b in zip(backward_through_hooks(apart, residual), backward_through_hooks(lambda t: t, residual)))


# (Only what is as large as the saved tensor or larger, and of no narrower type than it says: the refusal is what is tested.)
@pytest.mark.parametrize("change", [lambda t: t.double(), lambda t: t.cpu(), lambda t: torch.cat([t, t]), lambda t: t.unsqueeze(0), lambda t: t.int()])
def test_saved_tensors_that_come_back_as_others_are_refused(change):
    for dims, dtype in ((1, F32), (2, F32), (2, BF16)):  # weight, statistics, x
        # (Whole numbers in the place of what requires a gradient are refused by autograd before the node sees them.)
        with pytest.raises(RuntimeError, match="not what the forward pass saved|can require gradients"):
            backward_through_hooks(lambda t: change(t) if (t.dim(), t.dtype) == (dims, dtype) else t)


def test_data_exchanged_between_the_passes_is_refused():
    x, w = torch.randn(4, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    for leaf, other_leaf in ((x, w), (w, x)):  # (another type takes the exchanged one itself out of the graph)
        y, keep = layer_norm(x, w), leaf.data
        for other in (keep.bfloat16(), torch.cat([keep, keep])):
            leaf.data = other
            with pytest.raises(RuntimeError, match="not what the forward pass saved"):
                torch.autograd.grad(y, other_leaf, torch.ones_like(y), retain_graph=True)
        leaf.data = keep
        torch.autograd.grad(y, other_leaf, torch.ones_like(y))


def test_saved_tensors_on_the_cpu_and_recomputed():
    _, dev = make((6, 64), BF16, F32, True, True)
    leaves = [dev[k].requires_grad_() for k in ("x", "residual", "weight", "bias")]

    def grads(f=lambda f, *a: f(*a)):
        def norm(x, r, w, b):
            return layer_norm(x, w, b, residual=r)
        return torch.autograd.grad(f(norm, *leaves), leaves, (dev["dy"], dev["ds"]))

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    again = grads(lambda f, *a: torch.utils.checkpoint.checkpoint(f, *a, use_reentrant=False))
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


def test_autocast_leaves_float64_alone():
    """As for a linear layer; the type is refused then, as without autocast."""
    x = torch.randn(4, 64, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        assert torch.nn.functional.linear(x.double(), x.double()).dtype == torch.float64
        for args, kw in (((x.double(),), {}), ((x,), {"residual": x.double()}), ((x.double(),), {"residual": x})):
            with pytest.raises((TypeError, ValueError)):
                layer_norm(*args, **kw)
        assert layer_norm(x.half(), residual=x)[1].dtype == BF16


def test_views_that_are_to_be_negated():
    """Tensors whose memory holds the opposite of their values (as imag() of a conjugate gives them)."""
    _, dev = make((6, 64), BF16, F32, True, True)

    def grads(change):
        data = {k: change(v) for k, v in dev.items()}
        leaves = [data[k].requires_grad_() for k in ("x", "residual", "weight", "bias")]
        out = layer_norm(data["x"], data["weight"], data["bias"], residual=data["residual"])
        return out + torch.autograd.grad(out, leaves, (data["dy"], data["ds"]))

    want = grads(lambda t: t.detach().clone())
    got = grads(lambda t: torch._neg_view(-t.detach()))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_gradients_of_zeros_that_are_not_written_out():
    x, r = (torch.randn(4, 64, device="cuda", requires_grad=True) for _ in range(2))
    out = layer_norm(x, residual=r)
    for zeros in (torch._efficientzerotensor((4, 64), device="cuda"), torch.zeros(4, 64, device="cuda")):
        for grads in ((zeros, None), (None, zeros), (zeros, zeros)):
            got = torch.autograd.grad([o for o, g in zip(out, grads) if g is not None], (x, r), [g for g in grads if g is not None], retain_graph=True)
            assert all(g.shape == x.shape and not g.any() for g in got)


def test_weight_without_memory_is_refused():
    """It must not count as one that is not there: storage given up, a fake tensor outside of its mode, a functionalised one."""
    x, weight = torch.randn(4, 64, device="cuda"), torch.randn(64, device="cuda")
    fake = FakeTensorMode().from_tensor(weight)
    with pytest.raises(RuntimeError, match="no memory"):
        layer_norm(x, fake)
    with pytest.raises(RuntimeError, match="no memory"):
        torch.func.functionalize(lambda w: layer_norm(x, w))(weight)
    weight.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="no memory"):
        layer_norm(x, weight)


@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,features", [(75, 65537), (300, 70001), (9, 65568), (8, 131072)])
def test_many_rows_that_no_cluster_holds(rows, features, dtype, wtype):
    """Warps that add several rows of a column, and a last block of columns that is not full."""
    run_and_check(*make((rows, features), dtype, wtype, rows % 2 == 0, True, seed=rows), 1e-5, True)
