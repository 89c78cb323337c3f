"""ops/adamw.py against its formulas: moments to the bit, parameters in 64 bits."""
import copy

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import _train_reference as ref
from switchml_b200.ops.adamw import FusedAdamW, dequantized, grad_norm

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
SIZES = [1, 7, 31, 32, 33, 64, 255, 256, 257, 1000, 1023, 1024, 1025, 2048, 5000, 70001]


def make(sizes, dtype, seed=0, offset=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    params = []
    for i, n in enumerate(sizes):
        def place(t):
            flat = torch.empty(n + offset, dtype=dtype, device="cuda")
            return flat[offset:].copy_(t)
        p = place(torch.randn(n, generator=gen) * 0.05).requires_grad_()
        p.grad = place(torch.randn(n, generator=gen) * scale * 10.0 ** -(i % 4) * torch.exp(torch.randn(n, generator=gen)))
        params.append(p)
    return params


def in_memory(t):
    return t.detach().as_strided((t.numel(),), (1,)).cpu()


def value(opt, p):
    """The parameter with its remainder, in the order of memory."""
    flat = in_memory(p)
    if p.dtype == F32:
        return flat
    return ((flat.view(torch.int16).int() << 16) + in_memory(opt.state[p]["remainder"]).int()).view(F32)


class Checker:
    """A plain optimizer of every parameter beside `opt`."""

    def __init__(self, opt, bits, seed=0, first=0, groups=None):
        self.opt, self.plain = opt, []
        for group in groups or opt.param_groups:
            for p in group["params"]:
                plain = ref.Adamw(p, bits, seed, first)
                plain.p = value(opt, p).clone()
                self.plain.append((p, group, plain))
                first += -(-p.numel() // 256) * 256

    def step(self, clip=1.0, lr=None):
        grads = [None if p.grad is None else in_memory(p.grad.as_strided(p.shape, p.stride()) if p.grad.stride() == p.stride() else
                                                       torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(p.grad))
                 for p, _, _ in self.plain]
        self.opt.step()
        self.check(grads, clip, lr)

    def check(self, grads, clip=1.0, lr=None):
        for (p, group, plain), grad in zip(self.plain, grads):
            state = self.opt.state[p]
            if grad is not None:
                want, bound = plain.step(grad, group["lr"] if lr is None else lr, group["betas"], group["eps"], group["weight_decay"], clip)
                full = value(self.opt, p)
                ref.check("value", full, want, bound if p.dtype == F32 else bound - 2.0 ** -8 * want.abs())
                ref.check("param", in_memory(p), want, bound)
                plain.p = full.clone()
            assert int(state["step"]) == plain.step_count
            if plain.bits == 32:
                assert torch.equal(in_memory(state["exp_avg"]), plain.m) and torch.equal(in_memory(state["exp_avg_sq"]), plain.v)
            else:
                for name, codes, scales in (("exp_avg", plain.m, plain.em), ("exp_avg_sq", plain.v, plain.ev)):
                    assert torch.equal(state[name + "_scale"].view(torch.uint8).cpu(), scales), name
                    assert torch.equal(in_memory(state[name].view(torch.uint8)), codes), name


@pytest.mark.parametrize("offset", [0, 1, 4, 8, 16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(bits, dtype, offset):
    params = make(SIZES, dtype, offset=offset)
    opt = FusedAdamW(params, lr=1e-3, weight_decay=0.1, state_bits=bits, seed=11)
    checker = Checker(opt, bits, 11)
    for i in range(4):
        checker.step()
        for p in params:
            p.grad.mul_(-0.7 if i % 2 else 1.6)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_only_some_tensors_behind_an_aligned_address(bits, dtype):
    for move_grad in (False, True):
        params = make([3000, 4096], dtype)
        for p in params:
            moved = torch.empty(p.numel() + 1, dtype=dtype, device="cuda")[1:]
            if move_grad:
                p.grad = moved.copy_(p.grad)
            else:
                p.data = moved.copy_(p.data)
        checker = Checker(FusedAdamW(params, state_bits=bits), bits)
        checker.step()
        checker.step()


def test_places_beyond_32_bits():
    """The random bits of values around number 2^32."""
    opt = FusedAdamW(make([10], F32), state_bits=8, seed=3)
    opt._values = first = (1 << 32) - 1024
    params = make([700, 5000, 300], F32, 2)
    opt.add_param_group({"params": params})
    checker = Checker(opt, 8, 3, first, opt.param_groups[1:])
    checker.step()
    checker.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_betas_of_zero(bits):
    checker = Checker(FusedAdamW(make([100, 3000], F32), betas=(0.0, 0.0), state_bits=bits), bits)
    checker.step()
    checker.step()


def test_a_second_moment_that_overflows_takes_its_parameter_along():
    """v = inf while m is finite: in 8 bits the block of v is NaN from then on, and so are the parameters' values."""
    for dtype in (F32, BF16):
        p = torch.zeros(64, device="cuda", dtype=dtype, requires_grad=True)
        p.grad = torch.full_like(p, 1e-3)
        p.grad[3] = 1e25
        opt = FusedAdamW([p], state_bits=8, weight_decay=0.0)
        opt.step()
        p.grad[3] = 1e-3
        opt.step()
        assert p[:32].isnan().all() and not p[32:].isnan().any()


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_changed_from_outside(bits):
    """What loads a checkpoint, or broadcasts parameters through ``.data``, counts; the state does not bring back old values."""
    params = make([1000, 300], BF16)
    opt = FusedAdamW(params, state_bits=bits)
    opt.step()
    for p in params:
        p.data.copy_(torch.full_like(p, 3.0))
    opt.step()
    for p in params:  # half a bf16 step of remainder, and an update of at most about lr
        assert ((p.float() - 3.0).abs() <= 3 * 2.0 ** -7 + 5e-3).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_zero_blocks(bits):
    params = make([512, 64], F32)
    params[0].grad[64:256] = 0
    params[1].grad.zero_()
    checker = Checker(FusedAdamW(params, state_bits=bits), bits)
    for _ in range(3):
        checker.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_extreme_sizes(bits):
    """From 1e-30 to 1e18 (whose square still is a float32), in one block too."""
    params = make([320, 320], F32)
    params[0].grad.copy_(torch.logspace(-30, 18, 320))
    params[1].grad.copy_(torch.logspace(-45, -20, 320))
    checker = Checker(FusedAdamW(params, state_bits=bits), bits)
    for _ in range(3):
        checker.step()


def test_values_that_are_not_finite_stay_in_their_block():
    params = make([256], F32)
    params[0].grad[40], params[0].grad[200] = float("nan"), float("inf")
    opt = FusedAdamW(params, state_bits=8)
    plain = ref.Adamw(params[0], 8)
    opt.step()
    plain.step(params[0].grad, 1e-3)
    state = opt.state[params[0]]
    for name, codes, scales in (("exp_avg", plain.m, plain.em), ("exp_avg_sq", plain.v, plain.ev)):
        assert torch.equal(state[name + "_scale"].view(torch.uint8).cpu(), scales)
        assert torch.equal(state[name].view(torch.uint8).cpu(), codes)
    finite = torch.isfinite(params[0])
    assert finite.sum() >= 254 and not finite[40]  # the values themselves are lost one by one
    opt.step()
    finite = torch.isfinite(params[0]).cpu()
    assert finite[:32].all() and finite[64:192].all() and finite[224:].all()
    assert not finite[32:64].any() and not finite[192:224].any()


def test_layouts_of_parameters_and_gradients():
    for bits in (32, 8):
        a = torch.randn(6, 5, 3, 3, device="cuda").to(memory_format=torch.channels_last).requires_grad_()
        b = torch.randn(40, 30, device="cuda").t().requires_grad_()
        c = torch.randn(7, 11, device="cuda").requires_grad_()
        d = torch.tensor(0.5, device="cuda").requires_grad_()
        a.grad = torch.randn(6, 5, 3, 3, device="cuda")
        b.grad = torch.randn(40, 30, device="cuda").t()
        c.grad = torch.randn(11, 7, device="cuda").t()
        d.grad = torch.tensor(2.0, device="cuda")
        opt = FusedAdamW([a, b, c, d], state_bits=bits)
        checker = Checker(opt, bits)
        checker.step()
        checker.step()
        assert opt.state[a]["exp_avg"].stride() == a.stride()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_two_types_and_groups(bits):
    """More tensors than a launch takes, in two groups of mixed types; some without a gradient, some without values."""
    a = make([(i * 37) % 700 for i in range(1, 500)], F32, 1) + [torch.zeros(0, device="cuda", requires_grad=True)]
    a[-1].grad = torch.zeros(0, device="cuda")
    b = make([100 + i for i in range(20)], BF16, 2) + make([333], F32, 3)
    a[5].grad = b[3].grad = None
    opt = FusedAdamW([{"params": a, "weight_decay": 0.0}, {"params": b, "lr": 1e-2, "betas": (0.8, 0.95), "eps": 1e-6}], lr=1e-3, state_bits=bits,
                     seed=5)
    checker = Checker(opt, bits, 5)
    checker.step()
    a[5].grad = torch.randn_like(a[5])
    a[9].grad = None
    checker.step()


def test_parameters_without_gradients_do_nothing():
    p = torch.ones(5, device="cuda", requires_grad=True)
    opt = FusedAdamW([p], max_norm=1.0)
    opt.step()
    assert int(opt.state[p]["step"]) == 0 and torch.equal(p.detach().cpu(), torch.ones(5)) and float(opt.grad_norm) == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_clipping(dtype, bits):
    for max_norm in (0.01, 1e6):
        params = make(SIZES + [100] * 400, dtype)
        opt = FusedAdamW(params, max_norm=max_norm, state_bits=bits)
        checker = Checker(opt, bits)
        norm = torch.cat([p.grad.double() for p in params]).square().sum().sqrt().float().cpu()
        clip = torch.clamp(torch.tensor(max_norm) / (norm + 1e-6), max=1.0)
        checker.step(clip=float(clip))
        assert torch.equal(opt.grad_norm.cpu(), norm)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
def test_a_norm_that_is_not_finite_leaves_everything(bad):
    params = make([100, 3000], F32)
    opt = FusedAdamW(params, max_norm=1.0, state_bits=8)
    opt.step()
    kept = copy.deepcopy([{k: v.clone() for k, v in opt.state[p].items()} for p in params])
    values = [p.detach().clone() for p in params]
    good = params[1].grad.clone()
    params[1].grad.fill_(bad)
    opt.step()
    assert not torch.isfinite(opt.grad_norm)
    for p, state, v in zip(params, kept, values):
        assert torch.equal(p, v)
        for k, t in state.items():
            assert torch.equal(opt.state[p][k].view(torch.uint8) if t.element_size() == 1 else opt.state[p][k],
                               t.view(torch.uint8) if t.element_size() == 1 else t)
    params[1].grad.copy_(good)
    opt.step()
    assert all(int(opt.state[p]["step"]) == 2 for p in params)


def test_many_steps_on_average_go_where_the_moments_should():
    """A constant gradient g: v tends to g^2 (1 - beta2^t). Rounding to the nearest would stop far below it. 65536
    values of one size: the mean of their v is off by less than its own spread (at most half) over sqrt(65536) times 6."""
    n, g = 1 << 16, 0.01
    p = torch.zeros(n, device="cuda", requires_grad=True)
    p.grad = torch.full((n,), g, device="cuda")
    p.grad[::32] = 4 * g  # the largest of every block, which the others have to follow under one scale
    opt = FusedAdamW([p], state_bits=8, betas=(0.9, 0.99), lr=0.0, weight_decay=0.0)
    for _ in range(300):
        opt.step()
    others = torch.arange(n, device="cuda") % 32 != 0
    v = dequantized(opt.state[p]["exp_avg_sq"], opt.state[p]["exp_avg_sq_scale"])[others].double().mean()
    m = dequantized(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_scale"])[others].double().mean()
    want = g * g * (1 - 0.99 ** 300)
    assert abs(v - want) <= 6 * 0.5 * want / 256 and abs(m - g) <= 6 * 0.5 * g / 256


def test_learning_rate_as_a_tensor():
    for bits in (32, 8):
        params = make([1000], F32)
        lr = torch.tensor(2e-3, device="cuda")
        opt = FusedAdamW(params, lr=lr, state_bits=bits)
        checker = Checker(opt, bits)
        checker.step(lr=float(lr))
        lr.fill_(5e-4)
        checker.step(lr=float(lr))
    with pytest.raises(ValueError):
        FusedAdamW(params, lr=torch.tensor(1e-3))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    params = make(SIZES, F32) + make([777], BF16, 4)
    lr = torch.tensor(1e-3, device="cuda")
    opt = FusedAdamW(params, lr=lr, state_bits=bits, max_norm=1e9)
    checker = Checker(opt, bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        checker.step(lr=float(lr))
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            opt.step()
    for i, graph in enumerate(graphs + graphs):
        lr.fill_(1e-3 * (i + 1))
        for p in params:
            p.grad.mul_(1.3)
        graph.replay()
        torch.cuda.synchronize()
        checker.check([in_memory(p.grad) for p in params], lr=float(lr))


def test_same_run_same_bits_and_another_seed_other_bits():
    def run(seed):
        params = make([5000, 40], F32)
        opt = FusedAdamW(params, state_bits=8, seed=seed)
        for _ in range(3):
            opt.step()
        return [p.detach() for p in params] + [opt.state_buffers()[0][k].view(torch.uint8) for k in ("exp_avg", "exp_avg_sq")]

    a, b, c = run(1), run(1), run(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[2], c[2]) and not torch.equal(a[3], c[3])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict(bits, dtype):
    def once(opt):
        opt.step()
        return [in_memory(p) for g in opt.param_groups for p in g["params"]]

    params = make(SIZES, dtype)
    opt = FusedAdamW(params, state_bits=bits, lr=1e-2)
    once(opt)
    saved = copy.deepcopy(opt.state_dict())
    others = make(SIZES, dtype)
    for p, q in zip(params, others):
        q.data.copy_(p.data)
    other = FusedAdamW(others, state_bits=bits)
    addresses = {k: t.data_ptr() for k, t in other.state_buffers()[0].items()}
    other.load_state_dict(saved)
    assert {k: t.data_ptr() for k, t in other.state_buffers()[0].items()} == addresses
    assert other.param_groups[0]["lr"] == 1e-2
    assert all(torch.equal(a, b) for a, b in zip(once(opt), once(other)))
    # into the other form, and from torch's own optimizer
    converted = FusedAdamW(others, state_bits=40 - bits)
    converted.load_state_dict(saved)
    for i, q in enumerate(others):
        for name in ("exp_avg", "exp_avg_sq"):
            def wide(entry):
                return dequantized(entry[name], entry[name + "_scale"]) if entry[name].dtype == torch.float8_e4m3fn else entry[name]
            a, b = wide(saved["state"][i]), wide(converted.state[q])
            if bits == 8:
                assert torch.equal(a, b)
            else:  # half a step of e4m3, or half of the equal steps next to zero: 2^-10 of a scale that is at most 2^-7 of the largest
                assert ((a - b).abs() <= a.abs() / 16 + a.abs().max() * 2.0 ** -16).all()
                assert name == "exp_avg" or ((a > 0) == (b > 0)).all()
    torch_s = torch.optim.AdamW(make(SIZES, F32))
    torch_s.step()
    mine = FusedAdamW(make(SIZES, F32))
    mine.load_state_dict(torch_s.state_dict())
    for p, q in zip(torch_s.param_groups[0]["params"], mine.param_groups[0]["params"]):
        assert int(mine.state[q]["step"]) == 1
        assert torch.equal(mine.state[q]["exp_avg"], torch_s.state[p]["exp_avg"])
    with pytest.raises(ValueError):
        mine.load_state_dict(FusedAdamW(make([4], F32)).state_dict())
    for p, q in zip(params, others):
        q.data.copy_(p.data)
    other.load_state_dict({"state": {k: {n: t.cpu() for n, t in v.items()} for k, v in opt.state_dict()["state"].items()},
                           "param_groups": opt.state_dict()["param_groups"]})
    assert all(torch.equal(a, b) for a, b in zip(once(opt), once(other)))


def test_state_of_another_layout_is_put_in_order():
    """Scales belong to values that are neighbours in memory: codes of another layout are converted, not copied."""
    a = torch.randn(8, 16, 3, 3, device="cuda", requires_grad=True)
    a.grad = torch.randn_like(a) * torch.logspace(-4, 0, 8, device="cuda").view(8, 1, 1, 1)
    opt = FusedAdamW([a], state_bits=8)
    opt.step()
    b = a.detach().to(memory_format=torch.channels_last).requires_grad_()
    other = FusedAdamW([b], state_bits=8)
    other.load_state_dict(opt.state_dict())
    want = dequantized(opt.state[a]["exp_avg"], opt.state[a]["exp_avg_scale"])
    got = dequantized(other.state[b]["exp_avg"], other.state[b]["exp_avg_scale"])
    assert ((got - want).abs() <= want.abs() / 16 + want.abs().max() * 2.0 ** -16).all()


def test_master_buffers():
    params = make([1000, 31], BF16) + make([500], F32)
    opt = FusedAdamW(params)
    opt.step()
    flat = opt.master_buffers()[0].cpu()
    at = 0
    for p in params:
        assert torch.equal(flat[at:at + p.numel()], value(opt, p))
        at += -(-p.numel() // 256) * 256


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16]])
def test_grad_norm(dtypes):
    tensors = [t for i, d in enumerate(dtypes) for off in (0, 1, 3) for t in (p.grad for p in make(SIZES + [0, 300000], d, i, off))]
    tensors.append(torch.randn(64, 33, device="cuda")[:, :32])  # with gaps
    tensors.append(torch.randn(40, 30, device="cuda").t())
    got = grad_norm(tensors)
    want = torch.cat([t.double().reshape(-1) for t in tensors]).square().sum().sqrt()
    assert got.dtype == F32 and got.dim() == 0
    assert abs(got.double() - want) <= want * 2.0 ** -24 * (1 + 1e-6)
    assert torch.equal(got, grad_norm(tensors))


def test_grad_norm_of_much_and_of_extremes():
    big = torch.randn(3 * (1 << 24) + 5, device="cuda")
    want = big.double().square().sum().sqrt()
    assert abs(grad_norm([big]).double() - want) <= want * 2.0 ** -24 * (1 + 1e-6)
    assert float(grad_norm([torch.full((5,), 1e30, device="cuda")])) == pytest.approx(5 ** 0.5 * 1e30, rel=1e-6)
    assert float(grad_norm([torch.full((4,), 1e-30, device="cuda")])) == pytest.approx(2e-30, rel=1e-6)
    assert float(grad_norm([torch.zeros(0, device="cuda")])) == 0
    assert grad_norm([torch.tensor([1.0, float("nan")], device="cuda")]).isnan()
    assert float(grad_norm([torch.tensor([1.0, float("inf")], device="cuda")])) == float("inf")
    assert float(grad_norm(torch.full((1,), 2.0, device="cuda") for _ in range(900))) == 60


def test_grad_norms_captured_side_by_side():
    xs = [torch.randn(100000, device="cuda") for _ in range(2)]
    grad_norm(xs)
    graphs = []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = grad_norm([x])
        graphs.append((graph, out))
    for x in xs:
        x.mul_(3)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for x, (_, out) in zip(xs, graphs):
        assert torch.equal(out, grad_norm([x]))


def test_autograd_notices_the_step():
    p = torch.randn(10, device="cuda", requires_grad=True)
    opt = FusedAdamW([p])
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_closures_and_schedulers():
    p = torch.ones(4, device="cuda", requires_grad=True)
    opt = FusedAdamW([p], lr=0.1, weight_decay=0.0)
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)

    def closure():
        opt.zero_grad()
        loss = p.sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 4
    schedule.step()
    assert opt.param_groups[0]["lr"] == 0.05
    assert ((p - 0.9).abs() < 1e-6).all()


def test_refusals_on_the_gpu():
    p = torch.zeros(8, device="cuda", requires_grad=True)
    for error, params in ((TypeError, [p.detach().half().requires_grad_()]), (ValueError, [p, torch.zeros(3, requires_grad=True)]),
                          (ValueError, [torch.zeros(8, 8, device="cuda")[:, :4].requires_grad_()]),
                          (ValueError, [torch.zeros(1, device="cuda").expand(4).requires_grad_()])):
        with pytest.raises(error):
            FusedAdamW(params)
    for options in ({"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8}, {"weight_decay": -1.0}, {"lr": float("nan")}):
        with pytest.raises(ValueError):
            FusedAdamW([p], **options)
    opt = FusedAdamW([p])
    before = opt.state[p]["exp_avg"].clone()
    p.grad = torch.ones(8, device="cuda")
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    p.grad = torch.eye(8, device="cuda")[0].to_sparse()
    with pytest.raises(RuntimeError, match="strided"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(9, device="cuda")
    p.grad = torch.zeros(9, device="cuda")
    with pytest.raises(RuntimeError, match="another size"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(8)
    p.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match="another size, type or device"):
        opt.step()
    with pytest.raises(RuntimeError, match="another size, type or device"):
        opt.master_buffers()
    p.grad = None
    p.data = torch.zeros(8, device="cuda", dtype=torch.float16)
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="another size, type or device"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(8, device="cuda")
    assert torch.equal(opt.state[p]["exp_avg"], before)
    flat = torch.zeros(20, device="cuda")
    for bad in ([torch.zeros(3)], [], [flat[:10].requires_grad_(), flat[9:].requires_grad_()], [p.detach().requires_grad_()]):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": bad})
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="share memory"):
        FusedAdamW([flat.requires_grad_(), flat])
    assert len(opt.param_groups) == 1
    with pytest.raises(TypeError):
        copy.deepcopy(opt)
    p.data, p.grad = torch.zeros(8, device="cuda"), torch.ones(8, device="cuda")
    opt.step()
    assert int(opt.state[p]["step"]) == 1


def test_a_training_step_with_aggregated_gradients():
    """Buckets, layer norm, norm and step as ddp_train.py uses them together: the same step as torch's, up to rounding."""
    import switchml_b200 as sml
    from switchml_b200.models import BertForMaskedLM, BertConfig
    from switchml_b200.parallel.ddp import DistributedDataParallel
    ctx = sml.Context.get_instance()
    assert ctx.start(sml.make_config("cuda", packet_numel=256, mode="float_sum", launch="inline", average=True, symm_heap_mb=64))
    try:
        options = {"vocab_size": 96, "hidden": 64, "layers": 2, "heads": 4, "ffn": 128, "max_pos": 32, "dropout": 0.0}
        torch.manual_seed(0)
        plain = BertForMaskedLM(BertConfig(**options)).cuda()
        fused = BertForMaskedLM(BertConfig(fused_norm=True, **options)).cuda()
        fused.load_state_dict(plain.state_dict())
        net = DistributedDataParallel(fused, ctx, bucket_mb=1)
        ids, labels = torch.randint(0, 96, (4, 32), device="cuda"), torch.randint(0, 96, (4, 32), device="cuda")
        a = torch.optim.AdamW(plain.parameters(), lr=1e-3)
        b = FusedAdamW(fused.parameters(), lr=1e-3, max_norm=1e9)
        for _ in range(3):
            a.zero_grad()
            net.zero_grad()
            plain(ids, labels).backward()
            net(ids, labels).backward()
            norm = torch.stack([p.grad.norm() for p in plain.parameters()]).norm()
            for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
                torch.testing.assert_close(q.grad, p.grad, rtol=2e-3, atol=2e-5 * float(p.grad.abs().max() + 1e-3), msg=name)
            for p, q in zip(plain.parameters(), fused.parameters()):
                p.grad.copy_(q.grad)  # signs of gradients next to zero would decide whole steps
            a.step()
            b.step()
            assert abs(float(b.grad_norm) - float(norm)) <= 1e-4 * float(norm)
            for (name, p), q in zip(plain.named_parameters(), fused.named_parameters()):
                torch.testing.assert_close(q[1], p, rtol=1e-5, atol=1e-6, msg=name)
    finally:
        ctx.stop()


def test_training_command():
    """ddp_train.py with everything fused: runs, and says what it ran."""
    import json
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cmd = [sys.executable, os.path.join(root, "p4app-switchML_b200", "benchmarks", "ddp_train.py"), "--model", "bert", "--batch", "2",
           "--steps", "2", "--warmup", "1", "--fused-norm", "1", "--fused-wgrad", "1", "--optimizer", "fused8", "--max-norm", "1"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    out = json.loads([line for line in r.stdout.splitlines() if line.startswith("{")][-1])
    assert out["config"]["optimizer"] == "AdamW fused, 8-bit moments" and out["config"]["fused_norm"]
    assert 0 < out["final_loss"] < 100


def test_tracers_are_refused():
    p = torch.zeros(8, device="cuda", requires_grad=True)
    p.grad = torch.ones(8, device="cuda")
    opt = FusedAdamW([p], lr=0.1, weight_decay=0.0)
    for call in (lambda g: opt.step(), lambda g: opt.master_buffers()[0], lambda g: grad_norm([g])):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call)(p.grad)
    assert int(opt.state[p]["step"]) == 0 and not p.any()


@pytest.mark.parametrize("bits", [32, 8])
def test_another_memory_format_than_the_state_has(bits):
    """Refused: moments would meet other values' gradients. A format chosen before goes on as it is."""
    torch.manual_seed(0)
    for before, after in ((torch.contiguous_format, torch.channels_last), (torch.channels_last, torch.contiguous_format)):
        layer = torch.nn.Conv2d(4, 5, 3).cuda().to(memory_format=before)
        opt = FusedAdamW(layer.parameters(), state_bits=bits)
        checker = Checker(opt, bits)
        for p in layer.parameters():
            p.grad = torch.randn_like(p)
        checker.step()
        layer.to(memory_format=after)
        for call in (opt.step, opt.master_buffers):
            with pytest.raises(RuntimeError, match="another order"):
                call()
        assert all(int(opt.state[p]["step"]) == 1 for p in layer.parameters())
        layer.to(memory_format=before)
        checker.step()
    # Formats that are the same order of values, and contiguous tensors of other sizes, are no change.
    p = torch.randn(6, 4, 1, 1, device="cuda", requires_grad=True)
    opt = FusedAdamW([p], state_bits=bits)
    for data in (p.data.to(memory_format=torch.channels_last), p.data.as_strided(p.shape, (4, 1, 7, 9)), p.data.view(4, 6)):
        p.grad = None
        p.data = data
        p.grad = torch.randn_like(p)
        opt.step()
        opt.master_buffers()
    p.grad = None
    p.data = p.data.t()
    p.grad = torch.randn_like(p)
    with pytest.raises(RuntimeError, match="another order"):
        opt.step()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("path", ["as it is", "from 32 bits", "anew"])
def test_a_good_state_loaded_behind_values_that_were_not_finite(path, dtype):
    """Sizes that leave a block of moments with a few of the tensor's values: nothing of the bad ones is left in the others."""
    sizes = [7, 33, 1000, 256, 1]
    start = make(sizes, dtype)
    source = FusedAdamW(start, lr=1e-2, state_bits=32 if path == "from 32 bits" else 8, seed=5)
    source.step()
    good = copy.deepcopy(source.state_dict())
    if path == "anew":
        good["state"] = {}
    results = []
    for bad in (False, True):
        params = [p.detach().clone().requires_grad_() for p in start]
        opt = FusedAdamW(params, lr=1e-2, state_bits=8, seed=5)
        if bad:
            for p in params:
                p.grad = torch.full_like(p, float("nan"))
            opt.step()
            opt.step()
            assert all(p.isnan().all() for p in params)
            for p, q in zip(params, start):
                p.data.copy_(q)
        opt.load_state_dict(good)
        for i in range(3):
            for p, q in zip(params, start):
                p.grad = q.grad * (1 - 0.4 * i)
            opt.step()
        assert all(p.isfinite().all() for p in params)
        (masters,), (state,) = opt.master_buffers(), opt.state_buffers()
        at = 0
        for n in sizes:
            end = at + -(-n // 256) * 256
            for flat in [masters, state["exp_avg"].view(torch.uint8), state["exp_avg_sq"].view(torch.uint8)] + \
                    ([state["remainder"]] if dtype == BF16 else []):
                assert not flat[at + n:end].any()
            at = end
        results.append(params + [masters] + [state[k].view(torch.uint8) for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_remainders_behind_the_end_where_the_learning_rate_is_not_finite():
    params = make([5, 300], BF16)
    opt = FusedAdamW(params, lr=torch.tensor(float("nan"), device="cuda"))
    opt.step()
    (masters,), (state,) = opt.master_buffers(), opt.state_buffers()
    assert masters[:5].isnan().all() and masters[256:556].isnan().all()
    for flat in (masters, state["remainder"]):
        assert not flat[5:256].any() and not flat[556:].any()


def test_grad_norm_of_what_requires_a_gradient():
    w = torch.randn(1000, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="has no gradient"):
        grad_norm([g])
    with torch.no_grad():
        got = grad_norm([g])
    assert torch.equal(got, grad_norm([g.detach()])) and not got.requires_grad


def test_hooks_around_loading_a_state():
    """As around torch.optim.AdamW's: in their order, what the first ones return is loaded, the caller's dict stays."""
    p = make([300], F32)[0]
    for kind in (torch.optim.AdamW, FusedAdamW):
        opt, ran = kind([p], lr=1e-3), []
        opt.step()
        state = opt.state_dict()

        def other_rate(o, d):
            assert o is opt and d["param_groups"][0]["lr"] == 1e-3
            ran.append("pre")
            return {"state": d["state"], "param_groups": [{**d["param_groups"][0], "lr": 0.5}]}

        def without_state(o, d):
            assert d["param_groups"][0]["lr"] == 0.5
            ran.append("pre 2")
            d["state"] = {}

        opt.register_load_state_dict_pre_hook(other_rate)
        removed = opt.register_load_state_dict_pre_hook(lambda o, d: ran.append("removed"))
        opt.register_load_state_dict_pre_hook(without_state)
        opt.register_load_state_dict_post_hook(lambda o: ran.append(("post", o.param_groups[0]["lr"])))
        removed.remove()
        opt.load_state_dict(state)
        assert ran == ["pre", "pre 2", ("post", 0.5)]
        assert not opt.state[p] or int(opt.state[p]["step"]) == 0
        assert state["state"] and state["param_groups"][0]["lr"] == 1e-3


@pytest.mark.parametrize("option", ["amsgrad", "maximize", "differentiable"])
def test_options_that_make_another_step_are_refused(option):
    """From a checkpoint too, before anything of it is loaded; where they are off it is."""
    p, q = make([300, 5], F32)
    other = torch.optim.AdamW([q], lr=0.5)
    other.step()
    state = other.state_dict()
    opt = FusedAdamW([q], lr=1e-3)
    state["param_groups"][0][option] = True
    with pytest.raises(ValueError, match=option):
        opt.load_state_dict(state)
    assert opt.param_groups[0]["lr"] == 1e-3 and int(opt.state[q]["step"]) == 0
    state["param_groups"][0][option] = False
    opt.load_state_dict(state)
    assert opt.param_groups[0]["lr"] == 0.5 and int(opt.state[q]["step"]) == 1
    with pytest.raises(ValueError, match=option):
        opt.add_param_group({"params": [p], option: True})
    assert len(opt.param_groups) == 1
    opt.param_groups[0][option] = True
    with pytest.raises(ValueError, match=option):
        opt.step()
    assert int(opt.state[q]["step"]) == 1
    opt.param_groups[0][option] = False
    opt.step()
    assert int(opt.state[q]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_to_be_negated(bits):
    """A single value is contiguous as imag() of a conjugate: its memory holds the opposite of it."""
    params = [torch.zeros(n, device="cuda", requires_grad=True) for n in (1, 300)]
    params[0].grad = torch.complex(torch.zeros(1), torch.full((1,), 2.0)).cuda().conj().imag
    params[1].grad = torch._neg_view(torch.full((300,), 2.0, device="cuda"))
    assert params[0].grad.is_neg() and params[0].grad.is_contiguous() and params[1].grad.is_neg()
    opt = FusedAdamW(params, lr=1e-2, state_bits=bits, max_norm=1e6)
    opt.step()
    assert (params[0] > 0).all() and (params[1] > 0).all()
    assert float(grad_norm([p.grad for p in params])) == pytest.approx(2 * 301 ** 0.5, rel=1e-6) == float(opt.grad_norm)
    with pytest.raises(ValueError, match="negated"):
        FusedAdamW([torch._neg_view(torch.zeros(8, device="cuda")).requires_grad_()])
    params[1].grad = None
    params[1].data = torch._neg_view(torch.zeros(300, device="cuda"))
    params[1].grad = torch.ones(300, device="cuda")
    with pytest.raises(RuntimeError):
        opt.step()


def test_masters_of_empty_tensors():
    opt = FusedAdamW([torch.empty(0, 3, device="cuda", requires_grad=True)])
    junk = torch.full((256,), 5.0, device="cuda")
    del junk  # (its memory is what comes next)
    assert not opt.master_buffers()[0].any()


def test_a_group_that_could_not_be_added_leaves_nothing():
    params = make([10, 300], F32)
    opt = FusedAdamW(params[:1])
    native = opt._native

    class Full:
        def add_group(self, *args):
            raise torch.OutOfMemoryError("no room")

    opt._native = Full()
    with pytest.raises(torch.OutOfMemoryError):
        opt.add_param_group({"params": params[1:]})
    opt._native = native
    assert len(opt.param_groups) == 1 and list(opt.state_dict()["state"]) == [0]
    opt.step()
    opt.add_param_group({"params": params[1:]})
    opt.step()
    assert [int(s["step"]) for s in opt.state_dict()["state"].values()] == [2, 1]


def test_lazy_clones_of_a_parameter_stay_as_they_are():
    p, q = make([300, 40], F32)
    kept, before = torch._lazy_clone(p.detach()), p.detach().clone()
    opt = FusedAdamW([p, q])
    opt.step()
    assert torch.equal(kept, before) and not torch.equal(p, before)
    moments = opt.state[p]["exp_avg"]
    for t in (p.detach(), moments):
        kept = torch._lazy_clone(t)
        before = kept.clone()
        opt.step()
        assert torch.equal(kept, before) and not torch.equal(t, before)
