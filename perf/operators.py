"""Cases of the layer norm and of the many-tensor AdamW step: their inputs, plain forms, calls and exact values.

With ``own`` false ``run`` computes the plain form in elementary torch operations; with ``own`` true it calls the
framework (include/xdfm.h, recommenders_amd/models/deeprec/models/adamw.py).  Both take the same state.
"""

import ctypes
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_DTYPE_CODE = {"fp32": 0, "bf16": 1, "fp16": 2}
_ACT_CODE = {"identity": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "elu": 4}

# the dense variables of two of this framework's models, matrices as rows x columns
_TOWER = "1,1521x20,390x10,20,1,624x20,20,20,20,20x20,20,20,20,20,1"  # CIN [20, 10], DNN [20, 20], dim 16
_WIDE = "1,1521x256,4992x256,4992x256,512,1,2496x1024,1024,1024,1024,1024x512,512,512,512,512,1"  # dim 64
_TABLE = "2300000x10,2300000"  # a table of 2.3 M rows and its linear weights under the dense update


def listed():
    return [
        # one sample scored: the norm of one row of the wide tower, where the launch is what counts
        {"name": "norm fwd, one row", "op": "norm_fwd", "rows": 1, "cols": 1024, "dtype": "fp32", "act": "relu",
         "pad": 0},
        # the first layer of the wide tower in training, batch 65536
        {"name": "norm fwd, wide tower", "op": "norm_fwd", "rows": 65536, "cols": 1024, "dtype": "fp32", "act": "relu",
         "pad": 0},
        # rows of an odd length out of a wider buffer, 16-bit activations
        {"name": "norm fwd, odd rows", "op": "norm_fwd", "rows": 4099, "cols": 1001, "dtype": "fp16", "act": "tanh",
         "pad": 6},
        # the narrow tower of the Criteo-shaped workload, batch 8192
        {"name": "norm bwd, narrow tower", "op": "norm_bwd", "rows": 8192, "cols": 20, "dtype": "fp32", "act": "relu",
         "pad": 0},
        # the second layer of the wide tower, batch 65536
        {"name": "norm bwd, wide tower", "op": "norm_bwd", "rows": 65536, "cols": 512, "dtype": "fp32", "act": "relu",
         "pad": 0},
        # a sample's 39 embeddings of 64 side by side, 16-bit activations
        {"name": "norm bwd, embeddings", "op": "norm_bwd", "rows": 16384, "cols": 2496, "dtype": "bf16",
         "act": "identity", "pad": 0},
        # the dense variables of the Criteo-shaped model: launch-bound
        {"name": "adamw, narrow model", "op": "adamw", "bits": 32, "tensors": _TOWER, "grad": "fp32"},
        # the dense variables of the wide model
        {"name": "adamw, wide model", "op": "adamw", "bits": 32, "tensors": _WIDE, "grad": "fp32"},
        # the embedding table under the dense update
        {"name": "adamw, table", "op": "adamw", "bits": 32, "tensors": _TABLE, "grad": "fp32"},
        # the same three with states of 8 bits
        {"name": "adamw8, narrow model", "op": "adamw", "bits": 8, "tensors": _TOWER, "grad": "fp32"},
        {"name": "adamw8, wide model", "op": "adamw", "bits": 8, "tensors": _WIDE, "grad": "bf16"},
        {"name": "adamw8, table", "op": "adamw", "bits": 8, "tensors": _TABLE, "grad": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "adamw"])
    if op != "adamw":
        cols = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(65536, (1 << 25) // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "act": rng.choice(["identity", "relu", "sigmoid", "tanh", "elu"]), "pad": rng.choice([0, 0, 1, 4, 13])}
    left, sizes = 1 << 24, []
    for _ in range(_log_int(rng, 1, 300)):
        n = min(_log_int(rng, 1, 1 << 20), left)
        if n < 1:
            break
        left -= n
        sizes.append("%dx%d" % (n // 2 + 1, 2) if n > 64 and rng.random() < 0.5 else str(n))
    return {"op": op, "bits": rng.choice([32, 8]), "tensors": ",".join(sizes), "grad": rng.choice(["fp32", "bf16"])}


def _sizes(case):
    """Elements and decay of each tensor: matrices decay, vectors (biases, the norms' weights) do not."""
    shapes = [[int(n) for n in t.split("x")] for t in case["tensors"].split(",")]
    return [math.prod(s) for s in shapes], [0.01 if len(s) == 2 else 0.0 for s in shapes]


def work(case):
    if case["op"] != "adamw":
        size = 4 if case["dtype"] == "fp32" else 2
        n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
        if case["op"] == "norm_fwd":
            return {"bytes": 2 * size * n + 8 * rows + 8 * cols, "flops": 8 * n}
        return {"bytes": 3 * size * n + 8 * rows + 16 * cols, "flops": 16 * n}
    sizes, _ = _sizes(case)
    n, blocks = sum(sizes), sum((s + 63) // 64 for s in sizes)
    g = 4 if case["grad"] == "fp32" else 2
    if case["bits"] == 32:
        return {"bytes": n * (8 + g + 16), "flops": 15 * n}
    # states read and written as codes and scales, and given out as values (16 bits hold them exactly)
    return {"bytes": n * (8 + g + 4 + 4) + 4 * blocks, "flops": 40 * n}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = {"case": case}
    if case["op"] != "adamw":
        rows, cols, dt = case["rows"], case["cols"], _DTYPES[case["dtype"]]

        def buffer():
            return torch.empty((rows, cols + case["pad"]), dtype=dt, device="cuda")[:, :cols]

        # pre-activations: samples differ in spread and level
        spread = 0.5 + torch.rand((rows, 1), generator=gen, device="cuda")
        state["x"] = buffer().copy_(normal(rows, cols) * spread + 0.3 * normal(rows, 1))
        state["gamma"] = 1.0 + 0.1 * normal(cols)
        state["beta"] = 0.1 * normal(cols)
        state["eps"] = 1e-5
        state["stats"] = torch.empty((2, rows), device="cuda")
        if case["op"] == "norm_fwd":
            state["y"] = buffer()
        else:
            # what the forward pass left
            _, mean, rstd = _norm_plain(state)
            state["stats"][0], state["stats"][1] = mean[:, 0], rstd[:, 0]
            state["dy"] = buffer().copy_(1e-2 * normal(rows, cols))
            state["dx"] = buffer()
            state["dgamma"], state["dbeta"] = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
            if own:
                from recommenders_amd import _lib

                need = ctypes.c_size_t()
                _lib.check(_lib.lib.xdfm_layer_norm_bwd_workspace_floats(rows, cols, ctypes.byref(need)))
                state["workspace"] = torch.empty(max(need.value, 1), device="cuda")
        return state
    sizes, decay = _sizes(case)
    n = sum(sizes)
    lengths = torch.tensor(sizes, device="cuda")
    state["sizes"], state["decay"], state["lengths"] = sizes, decay, lengths
    # gradients of the variables differ in scale; some of their elements (unused rows, dead units) are zero
    scale = torch.repeat_interleave(10.0 ** (-2 - 2 * torch.rand(len(sizes), generator=gen, device="cuda")), lengths)
    live = torch.rand(n, generator=gen, device="cuda") > 0.05
    state["p"] = 0.05 * normal(n)
    state["g"] = (scale * normal(n) * live).to(_DTYPES[case["grad"]])
    m = 0.3 * scale * normal(n) * live
    v = (scale * normal(n)).square() * live
    state.update(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=57, seed=seed)
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
    else:
        state["block"] = _blocks(state)
        half = torch.full((n,), 1 << 19, device="cuda")
        state["m8"], state["ms"] = _encode(m, state["block"], 16, half)
        state["v8"], state["vs"] = _encode(v, state["block"], 32, half)
        state["m_out"] = torch.empty(n, dtype=torch.bfloat16, device="cuda")
        state["v_out"] = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    if own:
        from recommenders_amd.models.deeprec.models.adamw import AdamW

        def split(flat):
            return list(torch.split(flat, sizes))

        if case["bits"] == 32:
            slots = dict(slot_m=split(state["m"]), slot_v=split(state["v"]))
        else:
            blocks = [(s + 63) // 64 for s in sizes]
            slots = dict(slot_m=split(state["m8"]), slot_v=split(state["v8"]),
                         scale_m=list(torch.split(state["ms"], blocks)), scale_v=list(torch.split(state["vs"], blocks)))
        state["plan"] = AdamW(split(state["p"]), split(state["g"]), weight_decay=decay, state_bits=case["bits"], **slots)
    return state


# ------------------------------------------------------------------ layer norm, plain
def _activate(u, act):
    if act == "relu":
        return torch.where(u > 0, u, 0.0)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-u))
    if act == "tanh":
        return torch.tanh(u)
    if act == "elu":
        return torch.where(u > 0, u, torch.expm1(u))
    return u


def _slope(u, act):
    if act == "relu":
        return (u > 0).to(u.dtype)
    if act == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-u))
        return s * (1.0 - s)
    if act == "tanh":
        return 1.0 - torch.tanh(u).square()
    if act == "elu":
        return torch.where(u > 0, 1.0, torch.exp(u))
    return torch.ones_like(u)


def _norm_plain(state):
    x = state["x"].float()
    mean = x.mean(1, keepdim=True)
    off = x - mean
    rstd = 1.0 / torch.sqrt((off * off).mean(1, keepdim=True) + state["eps"])
    return off * rstd, mean, rstd


def _norm_fwd_plain(state):
    xhat, mean, rstd = _norm_plain(state)
    state["y"].copy_(_activate(xhat * state["gamma"] + state["beta"], state["case"]["act"]))
    state["stats"][0], state["stats"][1] = mean[:, 0], rstd[:, 0]
    return state["y"], state["stats"]


def _norm_bwd_plain(state):
    mean, rstd = state["stats"][0][:, None], state["stats"][1][:, None]
    xhat = (state["x"].float() - mean) * rstd
    u = xhat * state["gamma"] + state["beta"]
    if state["case"]["act"] == "relu":  # a unit is on or off by the exact sign: 32 bits miss it next to zero
        u = (state["x"].double() - mean) * rstd * state["gamma"].double() + state["beta"]
    du = state["dy"].float() * _slope(u, state["case"]["act"]).float()
    t = du * state["gamma"]
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    state["dx"].copy_(dx)
    state["dgamma"].copy_((du * xhat).sum(0))
    state["dbeta"].copy_(du.sum(0))
    return state["dx"], state["dgamma"], state["dbeta"]


# ------------------------------------------------------------------ AdamW, plain
def _blocks(state):
    """The number of the 64-element block that each element of the flat buffers lies in: blocks begin anew with
    every tensor."""
    per = (state["lengths"] + 63) // 64
    first = torch.repeat_interleave(per.cumsum(0) - per, state["lengths"])
    return first + _within(state) // 64


def _within(state):
    """Each element's place in its tensor."""
    lengths = state["lengths"]
    start = torch.repeat_interleave(lengths.cumsum(0) - lengths, lengths)
    return torch.arange(int(start.numel()), device=start.device) - start


def _encode(x, block, span, r20):
    """Values -> (codes, scales) of the 8-bit states: 3 bits under the leading one, 4 (span 16, signed) or 5 (span 32)
    bits of exponent, a power of two per block; r20 in [0, 2^20) is added below the last kept bit."""
    top = torch.zeros(int(block[-1]) + 1, dtype=x.dtype, device=x.device)
    top.scatter_reduce_(0, block, x.abs(), "amax")
    scale = torch.clamp(top.float().view(torch.int32) >> 23, min=48)
    q = torch.ldexp(x.abs().double(), (127 + span - scale)[block])
    low = torch.clamp(torch.frexp(q).exponent - 4, min=0)  # of the last kept bit
    k = (torch.round(torch.ldexp(q, 20 - low)).long() + r20) >> 20
    if span == 32:
        k = torch.where((x > 0) & (k == 0), 1, k)  # a second moment that is not zero stays so
    code = k + 8 * low
    if span == 16:
        code = code + 128 * (x < 0)
    return code.to(torch.uint8), scale.to(torch.uint8)


def _decode(code, scale, block, span):
    c = code.long()
    size = c & 127 if span == 16 else c
    e, f = size >> 3, size & 7
    units = torch.where(e > 0, (8 + f) << torch.clamp(e - 1, min=0), f).double()
    value = torch.ldexp(units, scale.int()[block] - 127 - span).float()
    return torch.where(c >= 128, -value, value) if span == 16 else value


def _random(state):
    """32 random bits for each element, out of its place, its tensor, the step and the seed."""
    def mix(a, b):
        return ((a ^ (a >> 15)) * 0x9E3779B1 + b) & 0xFFFFFFFF

    seed, step = state["seed"], state["step"]
    tensor = torch.repeat_interleave(torch.arange(len(state["sizes"]), device="cuda"), state["lengths"])
    key = mix(mix(mix(seed & 0xFFFFFFFF, seed >> 32), step & 0xFFFFFFFF), tensor)
    at = _within(state)
    a = ((at & 0xFFFFFFFF) + mix(key, 1)) * 0x9E3779B1 & 0xFFFFFFFF
    a = (a ^ (a >> 15) ^ mix(key, 2 + (at >> 32))) * 0x6A09E667 & 0xFFFFFFFF
    return a ^ (a >> 16)


def _adamw_plain(state):
    case, lr, b1, b2 = state["case"], state["lr"], state["beta1"], state["beta2"]
    g = state["g"].float()
    if case["bits"] == 32:
        m, v = state["m"], state["v"]
    else:
        block = state["block"]
        m, v = _decode(state["m8"], state["ms"], block, 16), _decode(state["v8"], state["vs"], block, 32)
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    root = torch.sqrt(v) / math.sqrt(1.0 - b2 ** state["step"]) + state["eps"]
    shrink = torch.repeat_interleave(torch.tensor(state["decay"], device="cuda"), state["lengths"]) * lr
    p = state["p"] - shrink * state["p"] - (lr / (1.0 - b1 ** state["step"])) * m / root
    state["p"].copy_(p)
    if case["bits"] == 32:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return {"p": state["p"], "m": state["m"], "v": state["v"]}
    bits = _random(state)
    for_m, for_v = ((bits & 0xFFFF) << 4) + 8, ((bits >> 16) << 4) + 8
    for name, x, span, r in (("m", m, 16, for_m), ("v", v, 32, for_v)):
        code, scale = _encode(x, block, span, r)
        state[name + "8"].copy_(code)
        state[name + "s"].copy_(scale)
        state[name + "_out"].copy_(_decode(code, scale, block, span))
    return {"p": state["p"], "m": state["m_out"], "v": state["v_out"]}


# ------------------------------------------------------------------ the framework's calls
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own(state):
    from recommenders_amd import _lib

    case = state["case"]
    if case["op"] == "norm_fwd":
        x, y = state["x"], state["y"]
        _lib.check(_lib.lib.xdfm_layer_norm_fwd(
            x.data_ptr(), x.stride(0), _DTYPE_CODE[case["dtype"]], case["rows"], case["cols"],
            state["gamma"].data_ptr(), state["beta"].data_ptr(), state["eps"], _ACT_CODE[case["act"]], y.data_ptr(),
            y.stride(0), state["stats"].data_ptr(), _stream()))
        return y, state["stats"]
    if case["op"] == "norm_bwd":
        x, dy, dx = state["x"], state["dy"], state["dx"]
        _lib.check(_lib.lib.xdfm_layer_norm_bwd(
            x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), _DTYPE_CODE[case["dtype"]], case["rows"],
            case["cols"], state["gamma"].data_ptr(), state["beta"].data_ptr(), state["stats"].data_ptr(),
            _ACT_CODE[case["act"]], dx.data_ptr(), dx.stride(0), state["dgamma"].data_ptr(),
            state["dbeta"].data_ptr(), state["workspace"].data_ptr(), _stream()))
        return dx, state["dgamma"], state["dbeta"]
    plan = state["plan"]
    plan.step(lr=state["lr"], beta1=state["beta1"], beta2=state["beta2"], eps=state["eps"], step=state["step"],
              seed=state["seed"])
    if case["bits"] == 32:
        return {"p": state["p"], "m": state["m"], "v": state["v"]}
    plan.read_state(state["m_out"], state["v_out"])
    return {"p": state["p"], "m": state["m_out"], "v": state["v_out"]}


def run(state):
    if own:
        return _own(state)
    return {"norm_fwd": _norm_fwd_plain, "norm_bwd": _norm_bwd_plain, "adamw": _adamw_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------ exact values
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adamw":
        return _adamw_exact(case, state)
    x, gamma, beta = state["x"].double(), state["gamma"].double(), state["beta"].double()
    act, n = case["act"], case["cols"]
    if case["op"] == "norm_fwd":
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = (var + state["eps"]).rsqrt()
        u = torch.addcmul(beta, gamma, (x - mean) * rstd)
        y = {"identity": lambda: u, "relu": lambda: u.clamp(min=0), "sigmoid": lambda: torch.sigmoid(u),
             "tanh": lambda: 1 - 2 / (torch.exp(2 * u) + 1), "elu": lambda: torch.nn.functional.elu(u)}[act]()
        return y, torch.stack([mean.flatten(), rstd.flatten()])
    # the statistics are inputs here, as the forward pass rounded them
    mean, rstd = state["stats"].double()[:, :, None]
    xhat = (x - mean) * rstd
    u = torch.addcmul(beta, gamma, xhat)
    if act == "sigmoid":
        slope = 0.25 / torch.cosh(u / 2).square()
    elif act == "tanh":
        slope = 1 / torch.cosh(u).square()
    elif act == "elu":
        slope = torch.exp(u.clamp(max=0))
    else:
        slope = (u > 0).double() if act == "relu" else torch.ones_like(u)
    du = state["dy"].double() * slope
    dgamma, dbeta = torch.einsum("rc,rc->c", du, xhat), du.sum(0)
    along = (du @ gamma)[:, None] / n
    across = torch.einsum("rc,rc,c->r", du, xhat, gamma)[:, None] / n
    return rstd * (du * gamma - along - xhat * across), dgamma, dbeta


def _adamw_exact(case, state):
    """Tensor by tensor, the definition in 64 bits; the codes' values by the distance to the next lower multiple."""
    t, lr, b1, b2 = state["step"], state["lr"], state["beta1"], state["beta2"]
    out = {"p": [], "m": [], "v": []}
    at = block_at = 0
    word = 1 << 32
    for index, (n, decay) in enumerate(zip(state["sizes"], state["decay"])):
        part = slice(at, at + n)
        p, g = state["p"][part].double(), state["g"][part].double()
        if case["bits"] == 32:
            m, v = state["m"][part].double(), state["v"][part].double()
        else:
            blocks = slice(block_at, block_at + (n + 63) // 64)
            m = _value(state["m8"][part], state["ms"][blocks], True)
            v = _value(state["v8"][part], state["vs"][blocks], False)
            block_at = blocks.stop
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + state["eps"])
        out["p"].append(p * (1 - lr * decay) - lr * step)
        if case["bits"] != 32:
            key = state["seed"] % word
            for more in (state["seed"] // word, t, index):
                key = ((key ^ key // 32768) * 0x9E3779B1 + more) % word
            keys = [((key ^ key // 32768) * 0x9E3779B1 + k) % word for k in (1, 2)]
            i = torch.arange(n, device="cuda")
            a = ((i + keys[0]) * 0x9E3779B1) % word
            a = ((a ^ a // 32768 ^ keys[1]) * 0x6A09E667) % word
            a = a ^ a // 65536
            m = _rounded(m, (a % 65536 + 0.5) / 65536, 16)
            v = _rounded(v, (a // 65536 + 0.5) / 65536, 32)
        out["m"].append(m)
        out["v"].append(v)
        at += n
    return {k: torch.cat(parts) for k, parts in out.items()}


def _padded(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 64)).view(-1, 64)


def _value(code, scale, signed):
    c = _padded(code.double())
    sign = torch.where(c >= 128, -1.0, 1.0) if signed else torch.ones_like(c)
    c = c % 128 if signed else c
    e = torch.floor(c / 8)
    units = torch.where(e < 1, c, (8 + c % 8) * 2.0 ** (e - 1))
    return (sign * units * 2.0 ** (scale.double() - (143 if signed else 159))[:, None]).flatten()[:code.numel()]


def _rounded(x, u, span):
    """x to a multiple of its last kept bit, up where u and what is cut off reach one together."""
    b = _padded(x)
    top = b.abs().amax(1, keepdim=True).clamp(min=2.0 ** -79)
    unit = 2.0 ** (torch.frexp(top).exponent - 1 - span).double()
    size = b.abs()
    last = torch.maximum(unit, 2.0 ** (torch.frexp(size).exponent - 4).double())
    k = torch.floor(size / last + _padded(u))
    if span == 32:
        k = torch.where((size > 0) & (k < 1), 1.0, k)
    return (torch.sign(b) * k * last).flatten()[:x.numel()]
