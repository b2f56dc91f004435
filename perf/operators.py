"""Cases of the training-step operators that stand next to the sparse convolutions: matrix
products grouped by ragged row blocks (and their gradients), group norm with an activation on
channels-last rows (and its gradients), and the AdamW step over many tensors.

Every case runs in two forms on the same inputs: elementary torch operations, and the library's
own entry points (`own`).
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"half": torch.float16, "bfloat16": torch.bfloat16, "float": torch.float32}
EPSILON = 1e-5        # group norm
BETAS, ADAM_EPSILON, WEIGHT_DECAY, LEARNING_RATE, STEP = (0.9, 0.999), 1e-8, 0.01, 1e-3, 137
BLOCK = 256           # elements that share a scale in an 8-bit state
E4M3_MAX = 448.0


def listed():
    return [
        # a decoding step's worth of rows: every group's weight is read for a handful of rows
        {"name": "product_few_rows", "op": "product", "rows": 48, "spare": 0, "groups": 8, "ci": 1024, "co": 512,
         "skew": 0.7, "dtype": "bfloat16"},
        # 27 groups as in a 3x3x3 rulebook, the channels of the backbone's middle levels, in float
        {"name": "product_float_27", "op": "product", "rows": 120000, "spare": 640, "groups": 27, "ci": 64, "co": 64,
         "skew": 0.5, "dtype": "float"},
        # a wide expert layer over a whole batch: bound by the tensor cores
        {"name": "product_wide", "op": "product", "rows": 65536, "spare": 0, "groups": 32, "ci": 2048, "co": 4096,
         "skew": 0.3, "dtype": "bfloat16"},
        # both gradients of a layer with odd row counts and channel counts off the powers of two
        {"name": "product_grad_odd", "op": "product_grad", "rows": 4999, "spare": 37, "groups": 13, "ci": 200, "co": 328,
         "skew": 1.2, "dtype": "half"},
        # both gradients of a training batch
        {"name": "product_grad_wide", "op": "product_grad", "rows": 32768, "spare": 0, "groups": 16, "ci": 2048,
         "co": 2048, "skew": 0.4, "dtype": "bfloat16"},
        # a small feature map, where the call's latency counts
        {"name": "norm_small", "op": "norm", "samples": 2, "rows": 256, "spare": 0, "ragged": False, "channels": 128,
         "groups": 32, "activation": "silu", "dtype": "bfloat16"},
        # the backbone's first level: four clouds of about 120,000 voxels with 16 channels
        {"name": "norm_voxels", "op": "norm", "samples": 4, "rows": 120000, "spare": 1001, "ragged": True,
         "channels": 16, "groups": 4, "activation": "relu", "dtype": "half"},
        # gradients over feature maps of 64 x 64
        {"name": "norm_grad_maps", "op": "norm_grad", "samples": 8, "rows": 4096, "spare": 0, "ragged": False,
         "channels": 512, "groups": 32, "activation": "silu", "dtype": "bfloat16"},
        # gradients over eight clouds of about 200,000 voxels with 128 channels
        {"name": "norm_grad_voxels", "op": "norm_grad", "samples": 8, "rows": 200000, "spare": 0, "ragged": True,
         "channels": 128, "groups": 8, "activation": "relu", "dtype": "half"},
        # the parameters of a small sparse backbone
        {"name": "adamw_backbone", "op": "adamw", "tensors": 24, "elements": 500000, "bits": 32, "dtype": "float"},
        # a wide model, states in 32 bits
        {"name": "adamw_wide", "op": "adamw", "tensors": 200, "elements": 100000000, "bits": 32, "dtype": "float"},
        # the same in bfloat16, states in 8 bits
        {"name": "adamw_wide_8bit", "op": "adamw", "tensors": 200, "elements": 100000000, "bits": 8,
         "dtype": "bfloat16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["product", "product_grad", "norm", "norm_grad", "adamw"])
    if op in ("product", "product_grad"):
        dtype = rng.choice(["half", "bfloat16", "half", "bfloat16", "float"])
        odd = rng.random() < 0.25
        top = 256 if dtype == "float" or odd else 4096
        while True:
            rows, groups = _log_int(rng, 1, 65536), _log_int(rng, 1, 128)
            ci, co = _log_int(rng, 8, top), _log_int(rng, 8, top)
            if not odd:
                ci, co = (ci + 7) // 8 * 8, (co + 7) // 8 * 8
            if rows * ci * co <= 1 << 36 and groups * ci * co <= 1 << 27:
                break
        return {"op": op, "rows": rows, "spare": rng.choice([0, 0, rows // 10]), "groups": groups, "ci": ci, "co": co,
                "skew": round(rng.uniform(0.0, 1.5), 2), "dtype": dtype}
    if op in ("norm", "norm_grad"):
        while True:
            samples, rows = _log_int(rng, 1, 16), _log_int(rng, 1, 200000)
            groups, per = rng.choice([1, 4, 8, 16, 32]), _log_int(rng, 1, 64)
            if samples * rows * groups * per <= 1 << 27:
                break
        ragged = rng.random() < 0.5
        return {"op": op, "samples": samples, "rows": rows, "spare": rng.choice([0, rows // 7]) if ragged else 0,
                "ragged": ragged, "channels": groups * per, "groups": groups,
                "activation": rng.choice(["none", "relu", "silu"]), "dtype": rng.choice(["half", "bfloat16", "float"])}
    tensors = _log_int(rng, 1, 300)
    return {"op": op, "tensors": tensors, "elements": max(tensors, _log_int(rng, 1000, 100000000)),
            "bits": rng.choice([8, 32]), "dtype": rng.choice(["half", "bfloat16", "float"])}


def _row_ends(rng, rows, parts, skew):
    """int32 [parts]: where each block of rows ends; block sizes from a log-normal, some of them empty."""
    share = np.exp(skew * rng.standard_normal(parts))
    counts = rng.multinomial(rows, share / share.sum())
    return np.cumsum(counts).astype(np.int32)


def prepare(case, seed):
    rng = np.random.default_rng([seed, 11])
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    state = {"case": dict(case)}
    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("product", "product_grad"):
        rows, groups, ci, co = case["rows"], case["groups"], case["ci"], case["co"]
        ends = _row_ends(rng, rows - case["spare"], groups, case["skew"])
        state["capacity"] = int(np.diff(ends, prepend=0).max(initial=0)) or 1
        state["ends"] = torch.from_numpy(ends).cuda()
        state["input"] = normal(rows, ci).to(dtype)
        state["weight"] = normal(groups, ci, co, scale=1.0 / math.sqrt(ci)).to(dtype)
        if case["op"] == "product_grad":
            state["output_grad"] = normal(rows, co).to(dtype)
    elif case["op"] in ("norm", "norm_grad"):
        samples, channels, groups = case["samples"], case["channels"], case["groups"]
        rows = samples * case["rows"] + case["spare"]
        x = normal(rows, channels) * (0.5 + torch.rand(channels, generator=gen, device="cuda")) + normal(channels)
        x = x.to(dtype)
        state["capacity"], state["ends"] = case["rows"], None
        if case["ragged"]:
            ends = _row_ends(rng, samples * case["rows"], samples, 0.1)
            state["capacity"] = int(np.diff(ends, prepend=0).max(initial=0)) or 1
            state["ends"] = torch.from_numpy(ends).cuda()
        else:
            x = x.view(samples, case["rows"], channels)
        state["input"] = x
        state["weight"], state["bias"] = 1.0 + normal(channels, scale=0.1), normal(channels, scale=0.1)
        if case["op"] == "norm_grad":
            state["output_grad"] = normal(*x.shape).to(dtype)
            state["mean"], state["rstd"] = _statistics(_padded(state, x), _counts(state), groups)
    else:
        state.update(_prepare_adamw(case, gen, dtype))
    return state


def _tensor_sizes(case):
    """Sizes of the tensors of an optimiser step: log-normal shares of the elements, at least one each."""
    rng = random.Random("%d %d" % (case["tensors"], case["elements"]))
    share = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    left = case["elements"] - case["tensors"]
    return [1 + int(left * s / sum(share)) for s in share]


def _starts(sizes):
    """Each tensor begins on a block of its own in the flat buffers of the program."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return starts, at


def _prepare_adamw(case, gen, dtype):
    sizes = _tensor_sizes(case)
    starts, total = _starts(sizes)
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for s, n in zip(starts, sizes):
        inside[s:s + n] = True

    def normal(scale):
        return torch.randn(total, generator=gen, device="cuda").mul_(scale).mul_(inside)

    grad = normal(1e-3)
    params = normal(0.05).to(dtype)
    first = normal(2e-4)
    second = (grad * 0.7 + normal(1e-3)).square_()
    state = {"sizes": sizes, "starts": starts, "params": params, "grads": grad.to(dtype),
             "grad_scale": torch.rand(1, generator=gen, device="cuda") * 0.5 + 0.5}
    if case["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = first, second
    else:
        state["exp_avg"], state["exp_avg_scale"] = _to_8bit(first)
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = _to_8bit(second.sqrt())
    # what the program hands to a step: one view of the flat buffers for each tensor
    for key in ("params", "grads", "exp_avg", "exp_avg_sq"):
        state[key + "_list"] = [state[key][s:s + n] for s, n in zip(starts, sizes)]
    if case["bits"] == 8:
        for key in ("exp_avg_scale", "exp_avg_sq_scale"):
            state[key + "_list"] = [state[key][s // BLOCK:(s + n + BLOCK - 1) // BLOCK] for s, n in zip(starts, sizes)]
    return state


# ---------------------------------------------------------------- plain forms

def _slots(ends, rows, parts, capacity):
    """For each row its place in [parts * capacity] padded rows; rows of no part go to one place behind them."""
    row = torch.arange(rows, device=ends.device)
    part = torch.searchsorted(ends, row.to(torch.int32), right=True)
    starts = torch.cat([ends.new_zeros(1), ends])
    return torch.where(part < parts, part * capacity + row - starts[part], parts * capacity)


def _pad(values, slots, parts, capacity):
    out = values.new_zeros((parts * capacity + 1, values.shape[1]), dtype=torch.float32)
    out[slots] = values.float()
    return out[:-1].view(parts, capacity, values.shape[1])


def _unpad(padded, slots):
    flat = padded.reshape(-1, padded.shape[2])
    return torch.cat([flat, flat.new_zeros((1, flat.shape[1]))])[slots]


def _plain_product(state):
    x, w, parts, cap = state["input"], state["weight"], state["case"]["groups"], state["capacity"]
    slots = _slots(state["ends"], x.shape[0], parts, cap)
    return _unpad(torch.bmm(_pad(x, slots, parts, cap), w.float()), slots).to(x.dtype)


def _plain_product_grad(state):
    x, w, dy, parts, cap = (state["input"], state["weight"], state["output_grad"], state["case"]["groups"],
                            state["capacity"])
    slots = _slots(state["ends"], x.shape[0], parts, cap)
    padded = _pad(dy, slots, parts, cap)
    dx = _unpad(torch.bmm(padded, w.float().transpose(1, 2)), slots).to(x.dtype)
    dw = torch.bmm(_pad(x, slots, parts, cap).transpose(1, 2), padded).to(w.dtype)
    return dx, dw


def _counts(state):
    case = state["case"]
    if state["ends"] is None:
        return torch.full((case["samples"],), case["rows"], dtype=torch.int32, device="cuda")
    return torch.diff(state["ends"], prepend=state["ends"].new_zeros(1))


def _padded(state, values):
    """[samples, capacity, channels] in 32 bits."""
    if state["ends"] is None:
        return values.float()
    slots = _slots(state["ends"], values.shape[0], state["case"]["samples"], state["capacity"])
    return _pad(values, slots, state["case"]["samples"], state["capacity"])


def _unpadded(state, padded):
    if state["ends"] is None:
        return padded
    return _unpad(padded, _slots(state["ends"], state["input"].shape[0], state["case"]["samples"], state["capacity"]))


def _mask(x, counts):
    return (torch.arange(x.shape[1], device=x.device)[None, :] < counts[:, None])[:, :, None, None]


def _statistics(x, counts, groups):
    """mean and 1 / sqrt(variance + epsilon) of each sample's groups, [samples, groups] each; the sums in 64 bits."""
    x = x.view(x.shape[0], x.shape[1], groups, -1)
    n = (counts * x.shape[3]).clamp(min=1)[:, None]
    mean = x.sum((1, 3), dtype=torch.float64) / n
    off = (x - mean.float()[:, None, :, None]) * _mask(x, counts)
    var = off.square().sum((1, 3), dtype=torch.float64) / n
    return mean.float(), (1.0 / torch.sqrt(var + EPSILON)).float()


def _affine(state, x, mean, rstd):
    """(normalised, before the activation), [samples, capacity, groups, channels of a group]."""
    groups = state["case"]["groups"]
    x = x.view(x.shape[0], x.shape[1], groups, -1)
    xhat = (x - mean[:, None, :, None]) * rstd[:, None, :, None]
    return xhat, xhat * state["weight"].view(groups, -1) + state["bias"].view(groups, -1)


def _plain_norm(state):
    x, act = state["input"], state["case"]["activation"]
    padded = _padded(state, x)
    mean, rstd = _statistics(padded, _counts(state), state["case"]["groups"])
    _, u = _affine(state, padded, mean, rstd)
    y = u.clamp(min=0) if act == "relu" else u / (1 + torch.exp(-u)) if act == "silu" else u
    return _unpadded(state, y.reshape(padded.shape)).to(x.dtype), mean, rstd


def _plain_norm_grad(state):
    x, act, groups = state["input"], state["case"]["activation"], state["case"]["groups"]
    padded, counts = _padded(state, x), _counts(state)
    xhat, u = _affine(state, padded, state["mean"], state["rstd"])
    du = _padded(state, state["output_grad"]).view(xhat.shape)
    if act == "relu":
        du = du * (u > 0)
    elif act == "silu":
        s = 1 / (1 + torch.exp(-u))
        du = du * (s * (1 + u * (1 - s)))
    dbeta = du.sum((0, 1), dtype=torch.float64)
    dgamma = (du * xhat).sum((0, 1), dtype=torch.float64)
    dxhat = du * state["weight"].view(groups, -1)
    n = (counts * xhat.shape[3]).clamp(min=1)[:, None]
    c1 = (dxhat.sum((1, 3), dtype=torch.float64) / n).float()
    c2 = ((dxhat * xhat).sum((1, 3), dtype=torch.float64) / n).float()
    dx = (dxhat - c1[:, None, :, None] - xhat * c2[:, None, :, None]) * state["rstd"][:, None, :, None]
    return (_unpadded(state, dx.reshape(padded.shape)).to(x.dtype), dgamma.float().reshape(-1),
            dbeta.float().reshape(-1))


def _to_8bit(x):
    """e4m3 values and one scale for each block of BLOCK elements."""
    blocks = x.view(-1, BLOCK)
    largest = blocks.abs().amax(1)
    fits = largest >= 1e-30
    inverse = torch.where(fits, E4M3_MAX / largest, torch.zeros_like(largest))
    scale = torch.where(fits, largest * (1 / E4M3_MAX), torch.zeros_like(largest))
    return (blocks * inverse[:, None]).to(torch.float8_e4m3fn).view(-1), scale


def _roots_to_8bit(x):
    """The same for values that are not negative; one that is not zero stays off zero."""
    blocks = x.view(-1, BLOCK)
    largest = blocks.amax(1)
    fits = largest >= 1e-30
    inverse = torch.where(fits, E4M3_MAX / largest, torch.zeros_like(largest))[:, None]
    scale = torch.where(fits, largest * (1 / E4M3_MAX), torch.zeros_like(largest))
    codes = torch.where((blocks > 0) & (inverse > 0), (blocks * inverse).clamp(min=2.0 ** -9), blocks * inverse)
    return codes.to(torch.float8_e4m3fn).view(-1), scale


def _from_8bit(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _plain_adamw(state):
    (b1, b2), bits = BETAS, state["case"]["bits"]
    g = state["grads"].float() * state["grad_scale"]
    if bits == 32:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    else:
        m = _from_8bit(state["exp_avg"], state["exp_avg_scale"])
        v = _from_8bit(state["exp_avg_sq"], state["exp_avg_sq_scale"]).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    change = m / (root * (1 / math.sqrt(1 - b2 ** STEP)) + ADAM_EPSILON)
    p = state["params"].float() * (1 - LEARNING_RATE * WEIGHT_DECAY) - change * (LEARNING_RATE / (1 - b1 ** STEP))
    state["params"].copy_(p)
    if bits == 32:
        state["exp_avg"].copy_(m)
        state["exp_avg_sq"].copy_(v)
    else:
        for key, pair in (("exp_avg", _to_8bit(m)), ("exp_avg_sq", _roots_to_8bit(root))):
            state[key].copy_(pair[0])
            state[key + "_scale"].copy_(pair[1])
    return _adamw_outputs(state)


def _adamw_outputs(state):
    keys = ["params", "exp_avg", "exp_avg_sq"]
    return {k: state[k] for k in keys + (["exp_avg_scale", "exp_avg_sq_scale"] if state["case"]["bits"] == 8 else [])}


# ---------------------------------------------------------------- the library's calls

_loaded = {}


def _library():
    """The harness package and a handle on the current stream."""
    if not _loaded:
        import __graft_entry__
        _loaded["ops"] = __graft_entry__.load_package()[0]
        _loaded["handle"] = _loaded["ops"].Handle(0)
    _loaded["handle"].set_queue(torch.cuda.current_stream().cuda_stream)
    return _loaded["ops"], _loaded["handle"]


def _own_pass(state):
    ops, handle = _library()
    case = state["case"]
    if case["op"] == "product":
        return ops.grouped_matmul_forward(handle, state["input"], state["weight"], state["ends"])
    if case["op"] == "product_grad":
        return (ops.grouped_matmul_backward_input(handle, state["output_grad"], state["weight"], state["ends"]),
                ops.grouped_matmul_backward_weight(handle, state["input"], state["output_grad"], state["ends"]))
    if case["op"] == "norm":
        return ops.group_norm_act_forward(handle, state["input"], state["weight"], state["bias"], case["groups"],
                                          EPSILON, case["activation"], state["ends"])
    if case["op"] == "norm_grad":
        return ops.group_norm_act_backward(handle, state["output_grad"], state["input"], state["weight"], state["bias"],
                                           state["mean"], state["rstd"], case["groups"], case["activation"],
                                           state["ends"])
    if "optimizer" not in state:  # a program makes it once for its parameters and states
        scales = ([state["exp_avg_scale_list"], state["exp_avg_sq_scale_list"]] if case["bits"] == 8 else [])
        state["optimizer"] = ops.MultiTensorAdamW(state["params_list"], state["exp_avg_list"], state["exp_avg_sq_list"],
                                                  *scales)
    state["optimizer"].step(handle, state["grads_list"], LEARNING_RATE, BETAS, ADAM_EPSILON, WEIGHT_DECAY, STEP,
                            grad_scale=state["grad_scale"])
    return _adamw_outputs(state)


def run(state):
    if own:
        return _own_pass(state)
    return {"product": _plain_product, "product_grad": _plain_product_grad, "norm": _plain_norm,
            "norm_grad": _plain_norm_grad, "adamw": _plain_adamw}[state["case"]["op"]](state)


# ---------------------------------------------------------------- 64 bits

def _blocks_of(ends, rows):
    ends = [rows] if ends is None else ends.tolist()
    return list(zip([0] + ends[:-1], ends))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("product", "product_grad"):
        x, w = state["input"], state["weight"]
        if case["op"] == "product":
            y = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device="cuda")
            for g, (a, b) in enumerate(_blocks_of(state["ends"], x.shape[0])):
                y[a:b] = x[a:b].double() @ w[g].double()
            return y
        dy = state["output_grad"]
        dx, dw = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros_like(w, dtype=torch.float64)
        for g, (a, b) in enumerate(_blocks_of(state["ends"], x.shape[0])):
            dx[a:b] = dy[a:b].double() @ w[g].double().T
            dw[g] = x[a:b].double().T @ dy[a:b].double()
        return dx, dw
    if case["op"] in ("norm", "norm_grad"):
        return _exact_norm(case, state)
    return _exact_adamw(case, state)


def _exact_norm(case, state):
    channels, groups, act = case["channels"], case["groups"], case["activation"]
    x = state["input"].reshape(-1, channels)
    ends = state["ends"] if case["ragged"] else torch.arange(1, case["samples"] + 1) * case["rows"]
    gamma, beta = state["weight"].double(), state["bias"].double()
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    means, rstds = [], []
    dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)

    def spread(v):  # [groups] -> [channels]
        return v.repeat_interleave(channels // groups)

    def by_group(v):  # mean over the rows and a group's channels
        return v.reshape(v.shape[0], groups, -1).mean((0, 2)) if v.shape[0] else v.new_zeros(groups)

    for i, (a, b) in enumerate(_blocks_of(ends, x.shape[0])):
        rows = x[a:b].double()
        if case["op"] == "norm":
            mean = by_group(rows)
            rstd = (by_group((rows - spread(mean)) ** 2) + EPSILON) ** -0.5
        else:
            mean, rstd = state["mean"][i].double(), state["rstd"][i].double()
        means.append(mean)
        rstds.append(rstd)
        xhat = (rows - spread(mean)) * spread(rstd)
        u = xhat * gamma + beta
        if case["op"] == "norm":
            out[a:b] = u.relu() if act == "relu" else u * u.sigmoid() if act == "silu" else u
            continue
        du = state["output_grad"].reshape(-1, channels)[a:b].double()
        if act == "relu":
            du = torch.where(u > 0, du, torch.zeros_like(du))
        elif act == "silu":
            du = du * u.sigmoid() * (1 + u * (-u).sigmoid())
        dbeta += du.sum(0)
        dgamma += (du * xhat).sum(0)
        dxhat = du * gamma
        out[a:b] = spread(rstd) * (dxhat - spread(by_group(dxhat)) - xhat * spread(by_group(dxhat * xhat)))
    out = out.view(state["input"].shape)
    return (out, torch.stack(means), torch.stack(rstds)) if case["op"] == "norm" else (out, dgamma, dbeta)


def _exact_adamw(case, state):
    b1, b2 = BETAS
    g = state["grads"].double() * state["grad_scale"].double()
    m, v = state["exp_avg"].double(), state["exp_avg_sq"].double()
    if case["bits"] == 8:
        m = m * state["exp_avg_scale"].double().repeat_interleave(BLOCK)
        v = (v * state["exp_avg_sq_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    step = LEARNING_RATE / (1 - b1 ** STEP) * m / (v.sqrt() / (1 - b2 ** STEP) ** 0.5 + ADAM_EPSILON)
    out = {"params": state["params"].double() * (1 - LEARNING_RATE * WEIGHT_DECAY) - step}
    if case["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    for key, values in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
        blocks = values.view(-1, BLOCK)
        largest = blocks.abs().amax(1)
        out[key + "_scale"] = largest / E4M3_MAX
        codes = blocks / torch.where(largest > 0, out[key + "_scale"], torch.ones_like(largest))[:, None]
        if key == "exp_avg_sq":
            codes = torch.where(codes > 0, codes.clamp(min=2.0 ** -9), codes)
        out[key] = codes.to(torch.float8_e4m3fn).float().view(-1)
    return out


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] in ("product", "product_grad"):
        size = 4 if case["dtype"] == "float" else 2
        rows, ci, co = case["rows"], case["ci"], case["co"]
        weights = min(case["groups"], case["rows"] - case["spare"]) * ci * co
        flops = 2.0 * (rows - case["spare"]) * ci * co
        if case["op"] == "product":
            return {"bytes": size * (rows * ci + weights + rows * co), "flops": flops}
        return {"bytes": size * (rows * co + rows * ci + weights + rows * ci + case["groups"] * ci * co),
                "flops": 2 * flops}
    if case["op"] in ("norm", "norm_grad"):
        size = 4 if case["dtype"] == "float" else 2
        elements = (case["samples"] * case["rows"] + case["spare"]) * case["channels"]
        small = 8 * case["channels"] + 8 * case["samples"] * case["groups"]
        if case["op"] == "norm":
            return {"bytes": 2 * size * elements + small, "flops": 10.0 * elements}
        return {"bytes": 3 * size * elements + 2 * small, "flops": 25.0 * elements}
    size = 4 if case["dtype"] == "float" else 2
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    elements = sum(_tensor_sizes(case))
    return {"bytes": (3 * size + state) * elements, "flops": 15.0 * elements}
