"""What a training step does around its aggregated gradients, as cases that can be timed.

Three kinds of work, each through the public Python interface:

``layer_norm``  ``ops.layer_norm.layer_norm``: the normalisation of a residual sum, its forward pass alone
                or with its backward pass (gradients of the input, the residual, weight and bias)
``adamw``       ``ops.adamw.FusedAdamW``: one step of all tensors of a model, moments in 32 or in 8 bits,
                with or without clipping by the norm of all gradients
``grad_norm``   ``ops.adamw.grad_norm``: the 2-norm over all gradients

Sizes come from BERT-large (16 x 512 tokens, hidden 1024; 298 tensors, 335 M parameters), from ResNet-50's
161 tensors and from 25 MB gradient buckets; the others are generic.

Moments in 8 bits. 32 consecutive values share a scale, a power of two: with e the exponent field of the
largest magnitude among them (at least 8), the scale is 2^(e-134), which puts the largest into [128, 256). A
value over its scale is rounded to 4 bits of significand (e4m3: exponents down to -6, below that steps of
2^-9), up or down at random, so that an average that moves by less than a step per update still moves as
far as it should in the mean; a second moment above zero stays above zero. The random bits are a function
of the seed, the step and the place of the value.
"""
import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "bfloat16": 2}
_PAD = 256  # every tensor begins at a multiple of this many values in the flat buffers
_LR, _BETA1, _BETA2, _EPS, _DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01
_STEP = 1000  # steps that the moments have behind them


def listed():
    return [
        # Evaluation of one short sentence: nothing but latency.
        _norm("norm_16_tokens", 16, 1024, "bfloat16", train=False),
        # Evaluation of a batch of 16 x 512 tokens.
        _norm("norm_bert_forward", 8192, 1024, "bfloat16", train=False),
        # Every normalisation of BERT-large in training, 16 x 512 tokens.
        _norm("norm_bert_train", 8192, 1024, "bfloat16", train=True),
        # The same without mixed precision, and with nothing to add: the head's normalisation.
        _norm("norm_head_fp32_train", 8192, 1024, "float32", train=True, residual=False),
        # Odd numbers of tokens and features; the sum goes on as the next block's residual.
        _norm("norm_ragged_train", 4099, 1021, "bfloat16", train=True, goes_on=True),
        # A wide layer on a large batch, weights in bf16 too.
        _norm("norm_wide_train", 16384, 8192, "bfloat16", train=True, goes_on=True, weights="bfloat16"),
        # One small layer with its embeddings: nothing but latency.
        _adamw("adamw_small", 32, "float32", _bert(512, 64, 1, 256)),
        # BERT-large as ddp_train.py trains it, with the usual clipping.
        _adamw("adamw_bert", 32, "float32", _bert(30522, 1024, 24, 4096), clip=True),
        # The same with a quarter of the memory for moments.
        _adamw("adamw8_bert", 8, "float32", _bert(30522, 1024, 24, 4096)),
        # Parameters and gradients in bf16, odd sizes, clipped. (The masters are put together as for a checkpoint.)
        _adamw("adamw8_ragged_bf16", 8, "bfloat16", _ragged(301, 400_000, 7), clip=True),
        # The gradients of one 25 MB bucket of BERT-large: many small tensors and a few large ones.
        {"name": "grad_norm_bucket", "kind": "grad_norm", "dtype": "float32", **_ragged(28, 1 << 22, 6)},
        # ResNet-50's 161 tensors.
        {"name": "grad_norm_resnet50", "kind": "grad_norm", "dtype": "float32", "model": "resnet50"},
    ]


def _norm(name, rows, features, dtype, train, residual=True, goes_on=False, weights="float32"):
    case = {"kind": "layer_norm", "rows": rows, "features": features, "dtype": dtype, "weights": weights, "train": train,
            "residual": residual, "goes_on": goes_on and residual}
    return dict(case, name=name) if name else case


def _adamw(name, bits, dtype, model, clip=False):
    case = {"kind": "adamw", "bits": bits, "dtype": dtype, "clip": clip, **model}
    return dict(case, name=name) if name else case


def _bert(vocab, hidden, layers, ffn):
    return {"model": "bert", "vocab": vocab, "hidden": hidden, "layers": layers, "ffn": ffn}


def _ragged(tensors, largest, mix):
    return {"model": "ragged", "tensors": tensors, "largest": largest, "mix": mix}


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["layer_norm"] * 3 + ["adamw"] * 3 + ["grad_norm"])
    if kind == "layer_norm":
        while True:
            rows, features = _log_uniform(rng, 1, 65536), _log_uniform(rng, 16, 16384)
            if rng.random() < 0.5:
                features = features // 8 * 8
            if rows * features <= 1 << 27:
                break
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        residual = rng.random() < 0.7
        return _norm("", rows, features, dtype, train=rng.random() < 0.7, residual=residual, goes_on=rng.random() < 0.5,
                     weights=rng.choice(["float32", dtype]))
    if rng.random() < 0.5:
        hidden = 8 * _log_uniform(rng, 4, 128)
        model = _bert(_log_uniform(rng, 100, 30522), hidden, rng.randint(1, 24), 4 * hidden)
    else:
        model = _ragged(rng.randint(1, 600), _log_uniform(rng, 1 << 8, 1 << 22), rng.randint(0, 1 << 20))
        if sum(_sizes(model)) > 300_000_000:
            model["tensors"] = 60
    dtype = rng.choice(["float32", "float32", "bfloat16"])
    if kind == "grad_norm":
        return {"kind": kind, "dtype": dtype, **model}
    return _adamw("", rng.choice([32, 8]), dtype, model, clip=rng.random() < 0.5)


def _sizes(case):
    """Number of values of every parameter tensor."""
    if case["model"] == "bert":
        h, f, v = case["hidden"], case["ffn"], case["vocab"]
        layer = [3 * h * h, 3 * h, h * h, h, h, h, f * h, f, h * f, h, h, h]
        return [v, v * h, 512 * h, 2 * h, h, h] + layer * case["layers"] + [h * h, h, h, h]
    if case["model"] == "resnet50":
        sizes, c = [64 * 3 * 49, 64, 64], 64
        for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for b in range(blocks):
                sizes += [c * width, width, width, width * width * 9, width, width, width * width * 4, width * 4, width * 4]
                if b == 0:
                    sizes += [c * width * 4, width * 4, width * 4]
                c = width * 4
        return sizes + [2048 * 1000, 1000]
    rng = random.Random(case["mix"])
    return [case["largest"]] + [_log_uniform(rng, 1, case["largest"]) for _ in range(case["tensors"] - 1)]


def _places(sizes):
    """Where each tensor begins in the flat buffers, and their length."""
    places, total = [], 0
    for n in sizes:
        places.append(total)
        total += -(-n // _PAD) * _PAD
    return places, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["kind"] == "layer_norm":
        rows, n, dtype, wtype = case["rows"], case["features"], _DTYPES[case["dtype"]], _DTYPES[case["weights"]]
        train = case["train"]
        # Features of a trained model have scales and means of their own.
        spread = torch.exp(0.5 * normal(n))
        state = {"kind": "layer_norm", "train": train, "eps": 1e-12,
                 "x": (normal(rows, n) * spread).add_(0.3 * normal(n)).to(dtype).requires_grad_(train),
                 "weight": (1 + 0.1 * normal(n)).to(wtype).requires_grad_(train),
                 "bias": (0.1 * normal(n)).to(wtype).requires_grad_(train), "residual": None, "dy": None, "ds": None}
        if case["residual"]:
            state["residual"] = normal(rows, n).to(dtype).requires_grad_(train)
        if train:
            state["dy"] = (1e-3 * normal(rows, n) * torch.exp(normal(rows, 1))).to(dtype)
            if case["goes_on"]:
                state["ds"] = (1e-3 * normal(rows, n)).to(dtype)
        return state
    sizes = _sizes(case)
    places, total = _places(sizes)
    dtype = _DTYPES[case["dtype"]]
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    scale = torch.empty(total, device="cuda")
    host = random.Random(seed)
    for n, at in zip(sizes, places):
        used[at:at + n] = True
        scale[at:at + n] = 10.0 ** host.uniform(-6, -2)  # layers' gradients differ by orders of magnitude
    scale = torch.where(used, scale, 0.0)
    scale *= torch.exp(normal(total))
    grad = (normal(total) * scale).to(dtype)
    grads = [grad[at:at + n] for n, at in zip(sizes, places)]
    if case["kind"] == "grad_norm":
        return {"kind": "grad_norm", "grad": grad, "grads": grads}
    master = torch.where(used, 0.02 * normal(total), 0.0)
    m = 0.3 * normal(total) * scale
    v = scale.square_().mul_(torch.rand(total, device="cuda", generator=gen) + 0.5)
    state = {"kind": "adamw", "bits": case["bits"], "clip": 1.0 if case["clip"] else None, "seed": seed & 0x7FFFFFFF, "step": _STEP,
             "param": master, "grad": grad}
    if dtype == torch.bfloat16:
        state["master"], state["param"] = master, _to_bf16(master)
        state["remainder"] = master.view(torch.int32).to(torch.int16)  # the low half
    if case["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = m, v
    else:
        for key, x in (("exp_avg", m), ("exp_avg_sq", v)):
            exponent = (x.abs().view(-1, 32).amax(1).view(torch.int32) >> 23).clamp_(min=8)
            state[key] = torch.ldexp(x.view(-1, 32), (134 - exponent).unsqueeze(1)).to(torch.float8_e4m3fn).view(-1)
            state[key + "_scale"] = (exponent - 7).to(torch.uint8).view(torch.float8_e8m0fnu)
    if own:
        from switchml_b200.ops.adamw import FusedAdamW
        params = []
        for n, at, g in zip(sizes, places, grads):
            params.append(state["param"][at:at + n].requires_grad_())
            params[-1].grad = g
        optimizer = FusedAdamW(params, lr=_LR, betas=(_BETA1, _BETA2), eps=_EPS, weight_decay=_DECAY, state_bits=case["bits"],
                               max_norm=state["clip"], seed=state["seed"])
        kept = optimizer.state_dict()
        for i, (n, at) in enumerate(zip(sizes, places)):
            kept["state"][i] = {"step": torch.tensor(_STEP), **{
                k: state[k][at:at + n] if not k.endswith("_scale") else state[k][at // 32:at // 32 + -(-n // 32)]
                for k in ("remainder", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale") if k in state}}
        optimizer.load_state_dict(kept)
        return {"kind": "adamw", "optimizer": optimizer, "param": state["param"]}
    return state


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "layer_norm":
        return _layer_norm(state)
    if state["kind"] == "grad_norm":
        return _grad_norm(state["grad"])
    return _adamw_step(state)


def _run_own(state):
    if state["kind"] == "grad_norm":
        from switchml_b200.ops.adamw import grad_norm
        return grad_norm(state["grads"])
    if state["kind"] == "adamw":
        optimizer = state["optimizer"]
        optimizer.step()
        out = {"param": state["param"], **optimizer.state_buffers()[0]}
        if out.pop("remainder", None) is not None:
            out["master"] = optimizer.master_buffers()[0]
        if optimizer.grad_norm is not None:
            out["norm"] = optimizer.grad_norm
        return out
    from switchml_b200.ops.layer_norm import layer_norm
    x, residual, weight, bias = state["x"], state["residual"], state["weight"], state["bias"]
    if residual is None:
        outputs = (layer_norm(x, weight, bias, state["eps"]),)
    else:
        outputs = layer_norm(x, weight, bias, state["eps"], residual=residual)
    out = {"y": outputs[0]}
    if residual is not None:
        out["sum"] = outputs[1]
    if state["train"]:
        gradients = (state["dy"],) if state["ds"] is None else (state["dy"], state["ds"])
        leaves = [t for t in (x, weight, bias, residual) if t is not None]
        got = torch.autograd.grad(outputs[:len(gradients)], leaves, gradients)
        out |= dict(zip(("dx", "dweight", "dbias", "dresidual"), got))
    return out


@torch.no_grad()
def _layer_norm(state):
    x, residual, wtype = state["x"], state["residual"], state["weight"].dtype
    out = {}
    total = x
    if residual is not None:
        total = (x.float() + residual.float()).to(x.dtype)  # the sum in the type that it goes on in
        out["sum"] = total
    s, w, b = total.float(), state["weight"].float(), state["bias"].float()
    centred = s - s.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + state["eps"])
    xhat = centred * rstd
    out["y"] = (xhat * w + b).to(x.dtype)
    if state["train"]:
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        if state["ds"] is not None:
            dx = dx + state["ds"].float()
        out["dx"] = dx.to(x.dtype)
        out["dweight"], out["dbias"] = (dy * xhat).sum(0).to(wtype), dy.sum(0).to(wtype)
        if residual is not None:
            out["dresidual"] = out["dx"]
    return out


def _grad_norm(grad):
    return torch.sqrt(grad.double().square().sum()).float()


def _mix(x):
    """A bijection of the 32-bit numbers that leaves no pattern, on 64-bit integers."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(numel, seed, step, device):
    """32 random bits for every place (fewer than 2^32 of them): 16 for the first moment, 16 for the second."""
    key = _mix(_mix((_mix(seed) + step) & 0xFFFFFFFF))
    return _mix((torch.arange(numel, device=device) + key) & 0xFFFFFFFF)


def _to_8_bits(x, bits16, never_zero):
    """(values, scales) of x in 8 bits: see above."""
    magnitude = x.abs().view(-1, 32)
    exponent = (magnitude.amax(1, keepdim=True).view(torch.int32) >> 23).clamp(min=8)
    y = magnitude * ((261 - exponent) << 23).view(torch.float32)
    small = y < 2.0 ** -6
    t = torch.where(small, y + 2.0 ** -6, y)
    code = ((t.view(torch.int32) + ((bits16.int() << 4) | 8).view(-1, 32)) >> 20) - torch.where(small, 968, 960)
    if never_zero:
        code = torch.where(magnitude > 0, code.clamp(min=1), code)
    code = code | ((x.view(torch.int32) >> 24) & 0x80).view(-1, 32)
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn), (exponent - 7).to(torch.uint8).view(-1).view(torch.float8_e8m0fnu)


def _to_bf16(x):
    return ((x.view(torch.int32) + 0x8000) >> 16).to(torch.int16).view(torch.bfloat16)


def _from_8_bits(x, scale):
    return (x.float().view(-1, 32) * scale.float().unsqueeze(1)).view(-1)


@torch.no_grad()
def _adamw_step(state):
    state["step"] += 1
    step, eight = state["step"], state["bits"] == 8
    g = state["grad"].float()
    out = {}
    if state["clip"] is not None:
        out["norm"] = _grad_norm(state["grad"])
        g = g * torch.clamp(state["clip"] / (out["norm"] + 1e-6), max=1.0)
    m, v = state["exp_avg"], state["exp_avg_sq"]
    if eight:
        m, v = _from_8_bits(m, state["exp_avg_scale"]), _from_8_bits(v, state["exp_avg_sq_scale"])
    m = m * _BETA1 + g * (1 - _BETA1)
    v = v * _BETA2 + g * (1 - _BETA2) * g
    denominator = torch.sqrt(v) / math.sqrt(1 - _BETA2 ** step) + _EPS
    master = state.get("master", state["param"])
    master.copy_(master * (1 - _LR * _DECAY) - _LR / (1 - _BETA1 ** step) * (m / denominator))
    if master is not state["param"]:
        state["param"] = _to_bf16(master)
        out["master"] = master
    if eight:
        bits = _random_bits(m.numel(), state["seed"], step, m.device)
        for key, x, b in (("exp_avg", m, bits & 0xFFFF), ("exp_avg_sq", v, bits >> 16)):
            state[key], state[key + "_scale"] = _to_8_bits(x, b, key == "exp_avg_sq")
            out[key + "_scale"] = state[key + "_scale"]
    else:
        state["exp_avg"].copy_(m)
        state["exp_avg_sq"].copy_(v)
    return {**out, "param": state["param"], "exp_avg": state["exp_avg"], "exp_avg_sq": state["exp_avg_sq"]}


def work(case):
    if case["kind"] == "layer_norm":
        n, row, size = case["features"], case["rows"] * case["features"], _BYTES[case["dtype"]]
        tensors = 4 if case["residual"] else 2  # x, residual; y, sum
        parameters, flops = 2, 9 * row
        if case["train"]:
            tensors += 3 if case["goes_on"] else 2  # dy and dx, the sum's gradient; dx is the residual's gradient too
            parameters, flops = 5, 25 * row
        return {"bytes": tensors * row * size + parameters * n * _BYTES[case["weights"]], "flops": flops}
    n, size = sum(_sizes(case)), _BYTES[case["dtype"]]
    if case["kind"] == "grad_norm":
        return {"bytes": n * size + 4, "flops": 2 * n}
    values = 8 + size  # the parameter (with its remainder) there and back, the gradient
    values += 16 if case["bits"] == 32 else 4 * (1 + 1 / 32)
    return {"bytes": n * values, "flops": n * (14 if case["bits"] == 32 else 40)}


def exact(case, seed):
    """The same from the definitions, in 64 bits."""
    with torch.no_grad():
        state = _inputs(case, seed)
        if case["kind"] == "layer_norm":
            return _exact_layer_norm(state)
        norm = torch.linalg.vector_norm(state["grad"].double())
        if case["kind"] == "grad_norm":
            return norm
        return _exact_adamw(state, norm)


def _inputs(case, seed):
    global own
    mine, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = mine


def _exact_layer_norm(state):
    s = state["x"].double()
    out = {}
    if state["residual"] is not None:
        out["sum"] = (s + state["residual"].double()).to(state["x"].dtype)
        s = out["sum"].double()
        out["sum"] = s
    w = state["weight"].double()
    var, mean = torch.var_mean(s, 1, correction=0, keepdim=True)
    xhat = (s - mean) / torch.sqrt(var + state["eps"])
    out["y"] = torch.addcmul(state["bias"].double(), xhat, w)
    if state["train"]:
        dy, n = state["dy"].double(), s.shape[1]
        g = dy * w
        along = torch.einsum("ij,ij->i", g, xhat).unsqueeze(1) / n
        dx = (g - g.sum(1, keepdim=True) / n - along * xhat) / torch.sqrt(var + state["eps"])
        out["dx"] = dx if state["ds"] is None else dx + state["ds"].double()
        out["dweight"], out["dbias"] = torch.einsum("ij,ij->j", dy, xhat), torch.einsum("ij->j", dy)
        if state["residual"] is not None:
            out["dresidual"] = out["dx"]
    return out


def _exact_adamw(state, norm):
    step = _STEP + 1
    g = state["grad"].double()
    out = {}
    if state["clip"] is not None:
        out["norm"] = norm
        g *= min(1.0, state["clip"] / (float(norm) + 1e-6))
    m, v = state["exp_avg"].double(), state["exp_avg_sq"].double()
    if state["bits"] == 8:
        m = (m.view(-1, 32) * state["exp_avg_scale"].double()[:, None]).flatten()
        v = (v.view(-1, 32) * state["exp_avg_sq_scale"].double()[:, None]).flatten()
    m.lerp_(g, 1 - _BETA1)
    v.lerp_(g * g, 1 - _BETA2)
    mhat, vhat = m / (1 - _BETA1 ** step), v / (1 - _BETA2 ** step)
    start = state.get("master", state["param"]).double()
    out["param"] = start - _LR * _DECAY * start - _LR * mhat / (vhat.sqrt() + _EPS)
    if "master" in state:
        out["master"] = out["param"]
    if state["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    one = torch.ones((), dtype=torch.float64, device=m.device)
    bits = _random_bits(m.numel(), state["seed"], step, m.device)
    for key, x, b in (("exp_avg", m, bits % 65536), ("exp_avg_sq", v, bits // 65536)):
        scale = torch.ldexp(one, torch.frexp(x.abs().view(-1, 32).amax(1).clamp(min=2.0 ** -119)).exponent - 8)
        y = (x.abs().view(-1, 32) / scale[:, None]).flatten()
        width = torch.ldexp(one, torch.frexp(y.clamp(min=2.0 ** -6)).exponent - 4)
        y = torch.floor(y / width + (b.double() + 0.5) / 65536) * width
        if key == "exp_avg_sq":
            y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
        out[key], out[key + "_scale"] = torch.copysign(y, x), scale
    return out
