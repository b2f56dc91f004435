"""PyTorch modules over the C ABI for what stands between and behind the convolutions of a
training step: group norm with an activation, products grouped by row blocks, the AdamW step.

    x = SubMConv3d(16, 64, 3)(x)
    x = GroupNormAct(8, 64, activation="relu")(x)          # per sample of the sparse tensor
    y = GroupedLinear(num_groups, 64, 128)(rows, ends)      # one matrix for each block of rows
    AdamW(model.parameters(), lr=1e-3, state_bits=8).step()

Every tensor stays on the GPU.  Nothing is read back, but for one check of the row order of a SparseConvTensor whose
indices came from outside (SparseConvTensor.sample_ends).  There is no CPU path.
"""
import math
import sys

import torch
from torch import nn

from .torch_sparse import SparseConvTensor, _handle

ops = sys.modules[__package__]


class _GroupedMatMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, group_ends):
        input, weight = input.contiguous(), weight.contiguous()
        ctx.save_for_backward(input, weight, group_ends)
        return ops.grouped_matmul_forward(_handle(input.device), input, weight, group_ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        input, weight, group_ends = ctx.saved_tensors
        grad = grad.contiguous()
        h = _handle(input.device)
        grad_input = grad_weight = None
        if ctx.needs_input_grad[0]:
            grad_input = ops.grouped_matmul_backward_input(h, grad, weight, group_ends)
        if ctx.needs_input_grad[1]:
            grad_weight = ops.grouped_matmul_backward_weight(h, input, grad, group_ends)
        return grad_input, grad_weight, None


def grouped_matmul(input, weight, group_ends):
    """output[r] = input[r] @ weight[g] for the rows r of group g, differentiable in input and weight
    (mluOpGroupedMatMul*).  input [rows,Ci], weight [G,Ci,Co]; group_ends int32 [G] on the device: group
    g's rows end there and the next group's begin.  Rows behind the last end give zeros and get zeros."""
    return _GroupedMatMul.apply(input, weight, group_ends)


class GroupedLinear(nn.Module):
    """A linear layer with a matrix of its own for each block of rows (experts, classes, levels)."""

    def __init__(self, num_groups, in_channels, out_channels, dtype=torch.float32):
        super().__init__()
        self.weight = nn.Parameter(torch.empty(int(num_groups), int(in_channels), int(out_channels), dtype=dtype))
        bound = 1.0 / math.sqrt(in_channels)
        nn.init.uniform_(self.weight, -bound, bound)

    def forward(self, input, group_ends):
        return grouped_matmul(input, self.weight, group_ends)


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, num_groups, epsilon, activation, sample_ends):
        input = input.contiguous()
        out, mean, rstd = ops.group_norm_act_forward(_handle(input.device), input, weight, bias, num_groups, epsilon,
                                                     activation, sample_ends)
        ctx.save_for_backward(input, weight, bias, mean, rstd, sample_ends)
        ctx.num_groups, ctx.activation = num_groups, activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        input, weight, bias, mean, rstd, sample_ends = ctx.saved_tensors
        affine = weight is not None and (ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        grad_input, grad_weight, grad_bias = ops.group_norm_act_backward(
            _handle(input.device), grad.contiguous(), input, weight, bias, mean, rstd, ctx.num_groups, ctx.activation,
            sample_ends, affine_grad=affine, affine_grad_dtype=weight.dtype if affine else None)
        needs = ctx.needs_input_grad
        return (grad_input if needs[0] else None, grad_weight if needs[1] else None, grad_bias if needs[2] else None, None,
                None, None, None)


def group_norm_act(input, num_groups, weight=None, bias=None, epsilon=1e-5, activation="none", sample_ends=None):
    """Group norm over channels-last values with an activation ("none", "relu", "silu"), differentiable
    in input, weight and bias (mluOpGroupNormAct*).  input [N, ..., C], each index of the first dimension a
    sample; or [rows, C] with sample_ends int32 [N] on the device, where each sample's rows end."""
    return _GroupNormAct.apply(input, weight, bias, num_groups, epsilon, activation, sample_ends)


class GroupNormAct(nn.Module):
    """group_norm_act as a module, for tensors [N, ..., C] and for a SparseConvTensor, whose samples are
    normalised one by one (its rows in ascending order of the batch index)."""

    def __init__(self, num_groups, num_channels, epsilon=1e-5, affine=True, activation="none", dtype=torch.float32):
        super().__init__()
        self.num_groups, self.epsilon, self.activation = int(num_groups), float(epsilon), activation
        self.weight = nn.Parameter(torch.ones(num_channels, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels, dtype=dtype)) if affine else None

    def forward(self, x):
        if not isinstance(x, SparseConvTensor):
            return group_norm_act(x, self.num_groups, self.weight, self.bias, self.epsilon, self.activation)
        out = SparseConvTensor(group_norm_act(x.features, self.num_groups, self.weight, self.bias, self.epsilon,
                                              self.activation, x.sample_ends()),
                               x.indices, x.spatial_shape, x.batch_size, x.indice_dict)
        out._ends = x._ends
        return out


class AdamW(torch.optim.Optimizer):
    """AdamW with one launch for up to 480 tensors (mluOpMultiTensorAdamW).

    state_bits: 32, or 8 for states of one byte an element and one scale for 256 elements (first moment
    and square root of the second in e4m3, rounded stochastically from the step and the element, so that
    small changes of a moment are not lost; a resumed run repeats them).  Parameters are dense CUDA tensors, in
    any order of dimensions, in float32, float16 or bfloat16; states are held in float or 8 bits whatever the
    parameter's type.  capturable=True keeps the step count and the learning rate of each parameter group on the
    device, so that a captured step can be
    replayed (lr may then be a CUDA tensor, a number is captured as it is; one step count for the whole group).  step(grad_scale=t)
    multiplies every gradient by the float32 CUDA tensor t of one element.  Before a step is captured, run one
    outside of the capture, which allocates the states and the handles, and let go of its loss: autograd cannot capture
    a backward pass while an earlier graph of the same parameters is alive.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32")
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError("lr must not be negative")
        if torch.is_tensor(lr) and not capturable:
            raise ValueError("a tensor as lr needs capturable=True")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError("0 <= beta < 1, eps >= 0 and weight_decay >= 0 are required")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.state_bits, self.capturable = state_bits, bool(capturable)
        self._plans = {}      # the tensors of each bucket, checked and laid out for the call
        self._schedules = {}  # capturable: per group (step count, {1, beta1, beta2}, the betas it holds)

    def _new_state(self, p):
        state = {"step": 0}
        for key in ("exp_avg", "exp_avg_sq"):  # (in the parameter's order)
            state[key] = torch.zeros_like(p, dtype=torch.float32 if self.state_bits == 32 else torch.uint8, requires_grad=False)
            if self.state_bits == 8:
                state[key + "_scale"] = torch.zeros(-(-p.numel() // ops.SCALE_BLOCK), dtype=torch.float32, device=p.device)
        return state

    @staticmethod
    def _gradient(p):
        """The gradient in the parameter's order."""
        if p.is_contiguous():
            return p.grad.contiguous()
        return p.grad if ops.same_order(p, p.grad) else torch.empty_like(p, dtype=p.grad.dtype).copy_(p.grad)

    def _bucket(self, key, params):
        """The plan for these parameters, built anew where a parameter or state lies elsewhere than before."""
        states = [self.state[p] for p in params]
        keys = ["exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if self.state_bits == 8 else [])
        tensors = [params] + [[s[k] for s in states] for k in keys]
        at = [list(map(torch.Tensor.data_ptr, v)) for v in tensors] + [p.is_contiguous() or p.stride() for p in params]
        known = self._plans.get(key)
        if known is None or known[0] != at:
            if len(self._plans) >= 64:  # the set of parameters that have gradients changes from step to step
                self._plans.clear()
            known = self._plans[key] = (at, ops.MultiTensorAdamW(*tensors))
        return known[1]

    @staticmethod
    def _refuse_capture(device):
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("run one step before the capture: replays would clear states that the graph makes")

    def _new_schedule(self, index, device, step):
        self._schedules[index] = (torch.full((), step, dtype=torch.int64, device=device), None, None)

    def _schedule(self, index, group, device):
        """Capturable: counts the group's step on the device and returns its schedule tensor."""
        if index not in self._schedules:
            self._refuse_capture(device)
            self._new_schedule(index, device, 0)
        count, base, made_for = self._schedules[index]
        betas = tuple(group["betas"])
        if made_for != betas:
            base = torch.ones(3, dtype=torch.float64, device=device)
            for i, beta in enumerate(betas):
                base[i + 1].fill_(beta)  # (on the device: nothing is copied from the host, which a capture forbids)
            # what a graph fills is not kept for other calls
            if device.type != "cuda" or not torch.cuda.is_current_stream_capturing():
                self._schedules[index] = (count, base, betas)
        count += 1
        powers = 1.0 - base ** count
        lr = group["lr"]
        if torch.is_tensor(lr):
            powers[0].copy_(lr)
        else:
            powers[0].fill_(float(lr))
        return powers.to(torch.float32)

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []  # every refusal comes before the first update
        for index, group in enumerate(self.param_groups):
            buckets = {}
            for i, p in enumerate(group["params"]):
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("sparse gradients are not supported")
                state = self.state[p]
                if not state:
                    self._refuse_capture(p.device)
                    state.update(self._new_state(p))
                count = 0 if self.capturable else state["step"] + 1
                buckets.setdefault((p.device, p.dtype, p.grad.dtype, count), []).append((i, p))
            if self.capturable and len({key[0] for key in buckets}) > 1:
                raise ValueError("capturable: the parameters of a group lie on one device")
            for (device, dtype, grad_dtype, count), members in buckets.items():
                plan = self._bucket((index, device, dtype, grad_dtype, tuple(i for i, _ in members)), [p for _, p in members])
                calls.append((index, group, device, count, plan, [p for _, p in members]))
        if (not self.capturable and any(device.type == "cuda" for _, _, device, *_ in calls)
                and torch.cuda.is_current_stream_capturing()):
            raise RuntimeError("capturable=True is needed to capture a step: a graph would repeat this one's count and rate")
        schedules = {}
        for index, group, device, count, plan, members in calls:
            more = {}
            if self.capturable:
                if index not in schedules:
                    schedules[index] = self._schedule(index, group, device)
                more["schedule"] = schedules[index]
            if self.state_bits == 8:
                more["rounding"] = "stochastic"
                if self.capturable:
                    more["step_count"] = self._schedules[index][0]
            lr = 0.0 if self.capturable else float(group["lr"])
            plan.step(_handle(device), list(map(self._gradient, members)), lr, group["betas"], group["eps"],
                      group["weight_decay"], max(count, 1), grad_scale=grad_scale, **more)
            for p in members:
                self.state[p]["step"] += 1
        return loss

    def __getstate__(self):  # (copies and pickles; what is laid out for the calls is not part of it)
        return {**super().__getstate__(), "state_bits": self.state_bits, "capturable": self.capturable,
                "_schedules": self._schedules}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans = {}
        self._schedules = {i: (entry[0].to(torch.int64), None, None) for i, entry in self._schedules.items()}

    def state_dict(self):
        """As Optimizer.state_dict.  A capturable optimiser's step counts are read from the device, where replays count too."""
        out = super().state_dict()
        states = out["state"] = dict(out["state"])
        for index, (count, *_) in self._schedules.items():
            for i in out["param_groups"][index]["params"]:
                if i in states:
                    states[i] = {**states[i], "step": int(count)}
        return out

    def _loaded_state(self, p, state):
        """A saved state of parameter `p` as this optimiser keeps it."""
        out = {"step": int(state["step"])}
        for key in ("exp_avg", "exp_avg_sq"):
            value, numel = state[key], p.numel()
            if self.state_bits == 32 and value.is_floating_point() and value.dtype != torch.float8_e4m3fn:
                value = value.to(torch.float32)
            elif self.state_bits == 32 or value.dtype not in (torch.uint8, torch.float8_e4m3fn):
                raise ValueError("%s is %s, which is no state of %d bits" % (key, value.dtype, self.state_bits))
            if value.numel() != numel:
                raise ValueError("%s has %d elements, its parameter %d" % (key, value.numel(), numel))
            if not ops.same_order(p, value):
                if self.state_bits == 8:
                    raise ValueError("8-bit states lie in the order that their parameter had in memory")
                value = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(value.reshape(p.shape))
            out[key] = value
            if self.state_bits == 8:
                out[key + "_scale"] = state[key + "_scale"].to(torch.float32)
                if out[key + "_scale"].numel() != -(-numel // ops.SCALE_BLOCK):
                    raise ValueError("%s has another number of scales" % key)
        return {key: v.detach().clone().to(p.device) if torch.is_tensor(v) else v for key, v in out.items()}

    def load_state_dict(self, state_dict):
        """As Optimizer.load_state_dict, with the states in this class's types (the base class would cast them to the
        parameters'); a state of torch.optim.AdamW is taken over.  Capturable: the parameters of a group must have
        been saved at one step.  Graphs that were captured before update what was there before: capture again."""
        state_dict = dict(state_dict)
        counts = {i: int(pair[0]) for i, pair in state_dict.pop("schedules", {}).items()}  # (kept apart by earlier versions)
        if any(("exp_avg_scale" in s) != (self.state_bits == 8) for s in state_dict["state"].values()):
            raise ValueError("the saved states have another number of bits")
        groups = state_dict["param_groups"]
        for key in ("amsgrad", "maximize"):
            if any(g.get(key) for g in groups):
                raise ValueError("%s is not supported" % key)
        params = dict(zip([i for g in groups for i in g["params"]], [p for g in self.param_groups for p in g["params"]]))
        states = {i: self._loaded_state(params[i], s) for i, s in state_dict["state"].items() if i in params}
        for index, g in enumerate(groups):
            own = [states[i] for i in g["params"] if i in states]
            for s in own:
                s["step"] = counts.get(index, s["step"])
            steps = {s["step"] for s in own}
            if self.capturable and len(steps) > 1:
                raise ValueError("capturable: one step count for a group, the saved ones are %s" % sorted(steps))
            counts[index] = max(steps, default=counts.get(index, 0))
        super().load_state_dict(state_dict)
        for i, s in states.items():
            self.state[params[i]] = s
        self._schedules, self._plans = {}, {}
        for index, group in enumerate(self.param_groups):
            if self.capturable and counts[index] and group["params"]:
                self._new_schedule(index, group["params"][0].device, counts[index])
            if not self.capturable and torch.is_tensor(group["lr"]):
                group["lr"] = float(group["lr"])
