"""AdamW over many tensors at once, and the norm of all their gradients (csrc/kernels/adamw.cu).

    optimizer = FusedAdamW(model.parameters(), lr=1e-4, state_bits=8, max_norm=1.0)
    loss.backward(); optimizer.step()

All tensors of a group take their step in one launch (in one per 384 tensors), gradients are read where they lie, in
the buckets of ``parallel.ddp`` too. Parameters are float32, or bfloat16 with 16 bits of remainder in the
state, which make the parameter a float32 value. The moments are float32, or with ``state_bits=8`` e4m3 numbers of
which 32, neighbours in memory, share a scale that is a power of two (e8m0). Those are rounded up or down at
random, with the distance as the chance: a second moment moves by a thousandth per step while its codes lie 6 to 12 %
apart, so rounding to the nearest would hold it where it is. The random bits are a function of ``seed``, the step and
the place of the value: the same run gives the same bits. A tracer (``torch.jit.trace``, ``make_fx``, ``torch.export``) would
not see the kernels: calls under one are refused.
"""
import torch

from .._native import native_extension

_MOMENTS = ("exp_avg", "exp_avg_sq")
_SCALED = 32  # values that share a scale
# Options of torch.optim.AdamW that would make another step: a group that has one, from a checkpoint say, is refused. (The others
# choose between ways to the same result, or, as decoupled_weight_decay, are set right by torch.optim.AdamW too.)
_OTHER_STEPS = ("amsgrad", "maximize", "differentiable")


def _ops():
    return native_extension("torch_switchml_train")


def grad_norm(tensors):
    """The 2-norm over all values of `tensors` (float32, bfloat16; of one CUDA device) as a float32 tensor without
    dimensions on that device: summed in float64 and in a fixed order. It has no gradient: tensors that require one are
    refused while gradients are recorded, so that none is lost (a penalty on gradients that were made with ``create_graph``)."""
    return _ops().grad_norm(list(tensors))


class FusedAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` for CUDA parameters in float32 or bfloat16, see above.

    `lr` may be a float32 tensor without dimensions on the parameters' device: a captured step then follows its value.
    With `max_norm` the gradients of all groups are scaled down to that norm where theirs is larger; ``grad_norm``
    then holds the norm before that, and a step whose norm is infinite or NaN changes nothing.
    Without it such values go where the formulas take them; with 8 bits they take the 32 values
    that share their scale with them. The ``.grad`` of the parameters stays as it is.

    State is allocated when a group is added, and ``load_state_dict`` copies into it, so that captured steps
    stay valid. It lies as the parameters do then: a memory format is chosen before the optimizer is made, and a
    parameter that has changed its own is refused. Counts of steps are kept on the device, one per parameter: a parameter without a gradient
    takes no step. One step at a time: steps of one optimizer on several streams have to be ordered by the caller.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is %r: 8 or 32 is wanted" % (state_bits,))
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm is %r: a positive number or None is wanted" % (max_norm,))
        if not 0 <= seed < 1 << 32:
            raise ValueError("seed is %r: a number of 32 bits is wanted" % (seed,))
        self._bits, self._max_norm = state_bits, max_norm
        self._native = _ops().Adamw(state_bits, seed)
        self._buffers = []   # of every group: flat tensors
        self._steps = []     # of every group: the parameters' counts of steps
        self._values = 0     # in the flat buffers of all groups
        self._device = None
        self._checked = []   # settings that have been found in order
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    @property
    def grad_norm(self):
        """The norm of the last step's gradients, None without `max_norm`: always the same tensor on the device, which every step
        and every replay of a captured one writes anew. ``.clone()`` keeps a value."""
        return self._native.norm if self._max_norm is not None else None

    def add_param_group(self, group):
        first = len(self.param_groups)
        super().add_param_group(group)
        try:
            self._allocate(self.param_groups[first])
        except Exception:
            del self.param_groups[first:]
            raise

    def __getstate__(self):
        raise TypeError("FusedAdamW is neither copied nor pickled: take its state_dict()")

    @staticmethod
    def _check_options(group):
        for name in _OTHER_STEPS:
            if group.get(name):
                raise ValueError("FusedAdamW has no %s" % name)

    def _check(self, group, device):
        lr, betas = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.dim() != 0 or lr.device != device:
                raise ValueError("lr as a tensor has to be a float32 without dimensions on %s" % device)
        elif not 0 <= lr < float("inf"):
            raise ValueError("lr is %r" % (lr,))
        if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
            raise ValueError("betas are %r: two numbers from 0 to below 1 are wanted" % (betas,))
        if not group["eps"] >= 0 or not group["weight_decay"] >= 0:
            raise ValueError("eps is %r, weight_decay %r" % (group["eps"], group["weight_decay"]))

    def _allocate(self, group):
        params = group["params"]
        device = self._device
        if not params:
            raise ValueError("a group has no parameters")
        self._check_options(group)
        for p in params:
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError("a parameter is %s: float32 or bfloat16 is wanted" % p.dtype)
            if p.layout != torch.strided or not p.is_cuda or (device or p.device) != p.device:
                raise ValueError("a parameter is %s on %s: strided on one CUDA device is wanted" % (p.layout, p.device))
            if not torch.ops.aten.is_non_overlapping_and_dense(p) or p.is_neg():
                raise ValueError("a parameter of the shape %s has gaps or overlaps in memory, or is a negated view" % (tuple(p.shape),))
            device = p.device
        # Tensors are taken side by side: two that share memory would be written by both.
        ends = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                      for g in self.param_groups for p in g["params"] if p.numel())
        if any(a[1] > b[0] for a, b in zip(ends, ends[1:])):
            raise ValueError("two parameters share memory")
        self._check(group, device)
        align = _ops().ALIGN
        places, total = [], 0
        for p in params:
            places.append(total)
            total += -(-p.numel() // align)
        total = max(total, 1)
        if total >= 1 << 32:
            raise ValueError("a group of %d values is too large" % (total * align))
        values = total * align
        flat = {}
        with torch.no_grad():
            for name in _MOMENTS:
                flat[name] = torch.zeros(values, dtype=torch.float32 if self._bits == 32 else torch.uint8, device=device)
                if self._bits == 8:
                    flat[name] = flat[name].view(torch.float8_e4m3fn)
                    flat[name + "_scale"] = torch.ones(values // _SCALED, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
            if any(p.dtype == torch.bfloat16 for p in params):
                flat["remainder"] = torch.zeros(values, dtype=torch.int16, device=device)
            steps = torch.zeros(len(params), dtype=torch.int32, device=device)
            states = {}
            for i, (p, place) in enumerate(zip(params, places)):
                at, n = place * align, p.numel()
                state = states[p] = {"step": steps[i]}
                for name in _MOMENTS:
                    state[name] = flat[name][at:at + n].as_strided(p.shape, p.stride())
                    if self._bits == 8:
                        state[name + "_scale"] = flat[name + "_scale"][at // _SCALED:at // _SCALED + -(-n // _SCALED)]
                if p.dtype == torch.bfloat16:
                    state["remainder"] = flat["remainder"][at:at + n].as_strided(p.shape, p.stride())
        self._native.add_group(params, places, flat["exp_avg"], flat["exp_avg_sq"], flat.get("exp_avg_scale"),
                               flat.get("exp_avg_sq_scale"), flat.get("remainder"), steps, self._values)
        self.state.update(states)
        self._device = device
        self._values += values
        self._buffers.append(flat)
        self._steps.append(steps)

    def state_buffers(self):
        """What the optimizer keeps, for every group as a dict of few flat tensors (``exp_avg``, ``exp_avg_sq``, their
        ``_scale`` with 8 bits, ``remainder`` with bf16 parameters): each parameter's state begins at a multiple of 256
        values. They are the state itself, not copies."""
        return [dict(b) for b in self._buffers]

    def master_buffers(self):
        """The parameters in float32, remainders included: for every group one new flat tensor in the layout of
        ``state_buffers``."""
        return [self._native.masters(i) for i in range(len(self._buffers))]

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        settings, tensors = [], []
        for group in self.param_groups:
            if "amsgrad" in group or "maximize" in group or "differentiable" in group:
                self._check_options(group)
            lr, (beta1, beta2), eps, decay = group["lr"], group["betas"], group["eps"], group["weight_decay"]
            tensor = isinstance(lr, torch.Tensor)
            now = (0.0 if tensor else lr, beta1, beta2, eps, decay)
            if tensor or now not in self._checked:
                self._check(group, self._device)
                self._checked = self._checked[-15:] + [now]
            tensors.append(lr if tensor else None)
            settings.append(now)
        self._native.step(settings, tensors, self._max_norm)
        return loss

    def load_state_dict(self, state_dict):
        """Copies `state_dict` into the state. Moments may come in the other form (those of
        ``torch.optim.AdamW`` among them): they are converted, to 8 bits by rounding to the nearest. A parameter
        that it says nothing about starts anew."""
        state_dict = dict(state_dict)  # hooks may change it, not the caller's
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            changed = hook(self, state_dict)
            if changed is not None:
                state_dict = changed
        self._load_all(state_dict)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    @torch.no_grad()
    def _load_all(self, state_dict):
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state is that of other groups of parameters")
        for group in groups:
            self._check_options(group)
        plans = []
        for saved, group in zip(groups, self.param_groups):
            for key, p in zip(saved["params"], group["params"]):
                entry = state_dict["state"].get(key) or {}
                for name in _MOMENTS:
                    if entry and (name not in entry or entry[name].shape != p.shape):
                        raise ValueError("the state of a parameter of the shape %s has no %s of that shape" % (tuple(p.shape), name))
                    if entry and entry[name].dtype == torch.float8_e4m3fn and entry[name + "_scale"].numel() != -(-p.numel() // _SCALED):
                        raise ValueError("the state of a parameter of the shape %s has another number of scales" % (tuple(p.shape),))
                plans.append((entry, p))
        for saved, group in zip(groups, self.param_groups):
            for key, value in saved.items():
                if key == "params":
                    continue
                if isinstance(group.get(key), torch.Tensor):
                    group[key].copy_(torch.as_tensor(value))  # a captured step reads it
                else:
                    group[key] = value.clone().to(self._device) if isinstance(value, torch.Tensor) else value
        copies, fills = ([], []), []
        for entry, p in plans:
            state = self.state[p]
            fills.append(int(entry.get("step", 0)))
            if "remainder" in state:
                if "remainder" in entry:
                    copies[0].append(state["remainder"])
                    copies[1].append(entry["remainder"])
                else:
                    state["remainder"].zero_()
            for name in _MOMENTS:
                self._load(entry, state, name, p, copies)
        if copies[0]:
            torch._foreach_copy_(*copies)
        for steps in self._steps:
            n = steps.numel()
            steps.copy_(torch.tensor(fills[:n], dtype=torch.int32))
            del fills[:n]

    def _load(self, entry, state, name, p, copies):
        new, scale = state[name], state.get(name + "_scale")
        old = entry.get(name)
        if old is None:
            new.view(torch.uint8 if self._bits == 8 else new.dtype).zero_()
            if scale is not None:
                scale.view(torch.uint8).fill_(1)
            return
        eight = old.dtype == torch.float8_e4m3fn
        if eight and self._bits == 8 and old.stride() == new.stride():
            copies[0].extend((new.view(torch.uint8), scale.view(torch.uint8)))
            copies[1].extend((old.view(torch.uint8), entry[name + "_scale"].view(torch.uint8)))
            return
        if eight:
            old = dequantized(old, entry[name + "_scale"])
        if self._bits == 32:
            copies[0].append(new)
            copies[1].append(old)
            return
        flat = torch.empty_strided(new.shape, new.stride(), dtype=torch.float32, device=p.device).copy_(old).as_strided((p.numel(),), (1,))
        blocks = torch.nn.functional.pad(flat, (0, -p.numel() % _SCALED)).view(-1, _SCALED)
        exponent = (blocks.abs().amax(1).view(torch.int32) >> 23).clamp_(min=8)
        codes = (blocks * ((261 - exponent).clamp_(min=1) << 23).view(torch.float32).unsqueeze(1)).to(torch.float8_e4m3fn).view(torch.uint8)
        if name == "exp_avg_sq":
            codes = torch.where(blocks > 0, codes.clamp(min=1), codes)
        lost = exponent == 255
        codes = torch.where(lost.unsqueeze(1), 0x7F, codes)
        new.view(torch.uint8).as_strided((p.numel(),), (1,)).copy_(codes.view(-1)[:p.numel()])
        scale.view(torch.uint8).copy_(torch.where(lost, 255, exponent - 7))


def dequantized(values, scale):
    """float32 values of moments in 8 bits: ``state[p]["exp_avg"]`` with ``state[p]["exp_avg_scale"]``, or the like."""
    n = values.numel()
    flat = values.view(torch.uint8).as_strided((n,), (1,)).view(torch.float8_e4m3fn).float()
    flat *= scale.float().repeat_interleave(_SCALED)[:n]
    return flat.as_strided(values.shape, values.stride())
