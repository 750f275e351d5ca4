"""Cases of the training and serving operators beside the array ops: group normalisation with an
activation (channels last), the gated linear recurrence, and the AdamW step over many tensors.

`run` computes a case in plain torch operations, or, where `own` is set, through the library's C ABI.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
ACTS = {"none": 0, "silu": 2, "gelu": 3}
SCANS = {"linear": 0, "sigmoid": 1}
EPS_NORM = 1e-5
#: elements of a tensor that share one scale in the 8-bit states
BLOCK = 256
#: hyperparameters of the optimiser, as the 32-bit floats that the entry points take
LR, BETA1, BETA2, EPS, DECAY = (float(np.float32(v)) for v in (1e-3, 0.9, 0.999, 1e-8, 0.01))
RNG_SEED = 0x51CED
_M64 = (1 << 64) - 1


def listed():
    return [
        # the six parameter tensors of the sine-fit network (1-64-64-1): nothing but launch latency
        {"name": "adamw sine fit", "op": "adamw", "bits": 32, "layers": "1-64-64-1"},
        # a deep model's list of weights, biases and norms, lengths from one element up, odd ones among them
        {"name": "adamw many tensors", "op": "adamw", "bits": 32, "count": 150, "elements": 40_000_000},
        # the classifier 784-2048-2048-10 with its moments in 8 bits
        {"name": "adamw8 classifier", "op": "adamw", "bits": 8, "layers": "784-2048-2048-10"},
        # a large model's share on one device: where 8-bit states are wanted for their size
        {"name": "adamw8 large", "op": "adamw", "bits": 8, "count": 40, "elements": 134_217_728},
        # the heads of one decoding step's tokens, normalised and gated: latency
        {"name": "norm tokens", "op": "norm", "dir": "fwd", "samples": 64, "positions": 1, "channels": 512, "groups": 8, "act": "silu"},
        # feature maps of odd width and group size, an ordinary convolution block
        {"name": "norm odd maps", "op": "norm", "dir": "fwd", "samples": 10, "positions": 961, "channels": 390, "groups": 13, "act": "gelu"},
        # the backward pass of a sequence block's norm: every token a row of its own
        {"name": "norm rows grad", "op": "norm", "dir": "bwd", "samples": 8192, "positions": 1, "channels": 2048, "groups": 16, "act": "silu"},
        # the backward pass over large feature maps
        {"name": "norm maps grad", "op": "norm", "dir": "bwd", "samples": 32, "positions": 4096, "channels": 512, "groups": 32, "act": "silu"},
        # one token for each of a batch of sequences, from the state that the last call left
        {"name": "scan one token", "op": "scan", "dir": "fwd", "mode": "sigmoid", "batch": 32, "steps": 1, "channels": 2048},
        # a training batch, forward
        {"name": "scan batch", "op": "scan", "dir": "fwd", "mode": "sigmoid", "batch": 8, "steps": 2048, "channels": 1024},
        # its backward pass at odd sizes
        {"name": "scan batch grad", "op": "scan", "dir": "bwd", "mode": "sigmoid", "batch": 4, "steps": 4099, "channels": 1001},
        # one long document: too few channels to fill the chip without a split of the time axis
        {"name": "scan long", "op": "scan", "dir": "fwd", "mode": "linear", "batch": 1, "steps": 65536, "channels": 1024},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("adamw", "norm", "scan"))
    if op == "adamw":
        return {"op": op, "bits": rng.choice((32, 8)), "count": _log(rng, 1, 200), "elements": _log(rng, 1000, 100_000_000)}
    if op == "norm":
        # (groups of eight values and more: of two, the gradient is what is left of a difference of equals)
        positions = rng.choice((1, _log(rng, 2, 8192)))
        groups, size = _log(rng, 1, 64), _log(rng, -(-8 // positions), 256)
        room = 50_000_000 // (groups * size * positions)
        samples = _log(rng, 1, min(8192 if positions == 1 else 64, max(1, room)))
        return {"op": op, "dir": rng.choice(("fwd", "bwd")), "samples": samples, "positions": positions, "channels": groups * size,
                "groups": groups, "act": rng.choice(("none", "silu", "gelu"))}
    steps, channels = rng.choice((1, _log(rng, 1, 65536), _log(rng, 64, 16384))), _log(rng, 1, 4096)
    room = 40_000_000 // (steps * channels)
    if room < 1:
        steps, room = max(1, 40_000_000 // channels), 1
    return {"op": op, "dir": rng.choice(("fwd", "bwd")), "mode": rng.choice(("linear", "sigmoid")), "batch": _log(rng, 1, min(64, room)),
            "steps": steps, "channels": channels}


def work(case):
    if case["op"] == "adamw":
        n = sum(_lens(case))
        blocks = sum(-(-k // BLOCK) for k in _lens(case))
        # parameter in and out, gradient in, both moments in and out (and two scales a block)
        return {"bytes": 28 * n if case["bits"] == 32 else 16 * n + 16 * blocks, "flops": 14 * n}
    if case["op"] == "norm":
        n, c = case["samples"] * case["positions"] * case["channels"], case["channels"]
        s = case["samples"] * case["groups"]
        if case["dir"] == "fwd":
            return {"bytes": 8 * n + 8 * c + 8 * s, "flops": 12 * n}
        return {"bytes": 12 * n + 16 * c + 8 * s, "flops": 24 * n}
    n, s = case["batch"] * case["steps"] * case["channels"], case["batch"] * case["channels"]
    if case["dir"] == "fwd":
        return {"bytes": 12 * n + 8 * s, "flops": (2 if case["mode"] == "linear" else 8) * n}
    # linear: gate, h and its gradient in, two gradients out; sigmoid: the input as well
    return {"bytes": (20 if case["mode"] == "linear" else 24) * n + 12 * s, "flops": (4 if case["mode"] == "linear" else 14) * n}


# ---------------------------------------------------------------- inputs
def _lens(case):
    """Lengths of the parameter tensors: a network's weights and biases, or `count` lengths that differ
    widely and add up to about `elements`."""
    if case.get("layers"):
        d = [int(v) for v in case["layers"].split("-")]
        return [k for i, o in zip(d, d[1:]) for k in (i * o, o)]
    r = random.Random(case["count"] * 1_000_003 + case["elements"])
    shares = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["count"])]
    total = sum(shares)
    return [max(1, int(case["elements"] * s / total)) for s in shares]


def _starts(lens):
    """Each tensor starts on the next multiple of BLOCK elements of one slab, as a pool hands them out."""
    at, starts = 0, []
    for n in lens:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _pointers(flat, starts, size):
    base = flat.data_ptr()
    return (ctypes.c_void_p * len(starts))(*[base + size * s for s in starts])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = {"case": dict(case, stream=(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream))}
    if case["op"] == "adamw":
        lens = _lens(case)
        starts, total = _starts(lens)
        # 1 inside a tensor, 0 in the slab's gaps behind it
        edge = torch.zeros(total + 1, device=DEV)
        edge.index_add_(0, torch.tensor(starts, device=DEV), torch.ones(len(lens), device=DEV))
        edge.index_add_(0, torch.tensor([a + n for a, n in zip(starts, lens)], device=DEV), -torch.ones(len(lens), device=DEV))
        inside = edge[:-1].cumsum(0).round()
        # gradients whose size differs over blocks, the moments that such gradients leave, a step well into the run
        size = torch.exp(2 * normal(total // BLOCK)).repeat_interleave(BLOCK) * 1e-3 * inside
        s["p"] = normal(total) * 0.05 * inside
        s["g"] = normal(total) * size
        m, v = normal(total) * 0.3 * size, (0.2 + uniform(total)) * size * size
        s["t"] = 200 + seed % 50
        s["lens"], s["count"] = (ctypes.c_size_t * len(lens))(*lens), len(lens)
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
            s["args"] = [_pointers(s[k], starts, 4) for k in "pgmv"]
            return s
        s["scales"] = torch.zeros(2 * (total // BLOCK), device=DEV)
        s["m8"], s["v8"] = (torch.zeros(total, dtype=torch.uint8, device=DEV) for _ in range(2))
        zero = torch.zeros(total, dtype=torch.int64, device=DEV)
        _store8(s, m, v, zero)
        blocks = [-(-n // BLOCK) for n in lens]
        counts = torch.tensor(blocks, device=DEV)
        first = torch.tensor([a // BLOCK for a in starts], device=DEV)
        s["ordinal"] = torch.arange(len(lens), device=DEV).repeat_interleave(counts)  # of each block's tensor
        s["within"] = torch.arange(total // BLOCK, device=DEV) - first.repeat_interleave(counts)  # block's place in it
        s["args"] = [_pointers(s["p"], starts, 4), _pointers(s["g"], starts, 4), _pointers(s["m8"], starts, 1), _pointers(s["v8"], starts, 1),
                     _pointers(s["scales"], [2 * a // BLOCK for a in starts], 4)]
        return s
    if case["op"] == "norm":
        n, p, c, k = case["samples"], case["positions"], case["channels"], case["groups"]
        # every channel with an offset and a size of its own
        s["x"] = normal(n, p, c) * torch.exp(0.3 * normal(c)) + 0.5 * normal(c)
        s["weight"], s["bias"] = 1 + 0.2 * normal(c), 0.2 * normal(c)
        s["mean"], s["rstd"] = torch.empty(n, k, device=DEV), torch.empty(n, k, device=DEV)
        if case["dir"] == "fwd":
            s["out"] = torch.empty_like(s["x"])
            return s
        x = s["x"].view(n, p, k, c // k)
        mean = x.mean(dim=(1, 3), keepdim=True)
        s["mean"] = mean.reshape(n, k).contiguous()
        s["rstd"] = torch.rsqrt((x - mean).square().mean(dim=(1, 3)) + EPS_NORM)
        s["dy"] = normal(n, p, c)
        s["dx"], s["dw"], s["db"] = torch.empty_like(s["x"]), torch.empty(c, device=DEV), torch.empty(c, device=DEV)
        return s
    b, t, d = case["batch"], case["steps"], case["channels"]
    # gates that forget at very different rates over the channels
    s["gate"] = normal(b, t, d) + 2 * normal(d) + 1
    if case["mode"] == "linear":
        s["gate"] = torch.sigmoid(s["gate"])
    s["x"], s["h0"] = normal(b, t, d), normal(b, d)
    if case["dir"] == "fwd":
        s["h"], s["h_last"] = torch.empty(b, t, d, device=DEV), torch.empty(b, d, device=DEV)
        return s
    s["h"] = _scan_plain(case["mode"], s["gate"], s["x"], s["h0"])
    s["dh"], s["dh_last"] = normal(b, t, d), normal(b, d)
    s["dgate"], s["dx"], s["dh0"] = torch.empty_like(s["gate"]), torch.empty_like(s["x"]), torch.empty_like(s["h0"])
    return s


# ---------------------------------------------------------------- plain forms
def _act(name, u):
    if name == "silu":
        return u / (1 + torch.exp(-u))
    if name == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u


def _act_grad(name, u):
    if name == "silu":
        q = 1 / (1 + torch.exp(-u))
        return q * (1 + u * (1 - q))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(u)


def _norm_fwd(s):
    c = s["case"]
    n, p, k = c["samples"], c["positions"], c["groups"]
    x = s["x"].view(n, p, k, -1)
    mean = x.mean(dim=(1, 3), keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + EPS_NORM)
    u = (centred * rstd).view(n, p, -1) * s["weight"] + s["bias"]
    return {"out": _act(c["act"], u), "mean": mean.reshape(n, k), "rstd": rstd.reshape(n, k)}


def _norm_bwd(s):
    c = s["case"]
    n, p, k = c["samples"], c["positions"], c["groups"]
    mean, rstd = s["mean"].view(n, 1, k, 1), s["rstd"].view(n, 1, k, 1)
    hat = (s["x"].view(n, p, k, -1) - mean) * rstd
    flat = hat.view(n, p, -1)
    gu = s["dy"] * _act_grad(c["act"], flat * s["weight"] + s["bias"])
    dw, db = (gu * flat).sum(dim=(0, 1)), gu.sum(dim=(0, 1))
    gx = (gu * s["weight"]).view(n, p, k, -1)
    a, b = gx.mean(dim=(1, 3), keepdim=True), (gx * hat).mean(dim=(1, 3), keepdim=True)
    return {"dx": (rstd * (gx - a - hat * b)).view(n, p, -1), "dw": dw, "db": db}


def _coefficients(mode, gate, x):
    if mode == "linear":
        return gate.clone(), x.clone()
    return 1 / (1 + torch.exp(-gate)), x / (1 + torch.exp(gate))


def _scan_plain(mode, gate, x, h0):
    a, h = _coefficients(mode, gate, x)
    h[:, 0] += a[:, 0] * h0
    k = 1
    while k < h.shape[1]:  # runs of k steps are joined in pairs
        h[:, k:] = h[:, k:] + a[:, k:] * h[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return h


def _scan_bwd(s):
    mode = s["case"]["mode"]
    a, _ = _coefficients(mode, s["gate"], s["x"])
    g = s["dh"].clone()
    g[:, -1] += s["dh_last"]
    c = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), dim=1)
    k = 1
    while k < g.shape[1]:
        g[:, :-k] = g[:, :-k] + c[:, :-k] * g[:, k:]
        c[:, :-k] = c[:, :-k] * c[:, k:]
        k *= 2
    before = torch.cat((s["h0"].unsqueeze(1), s["h"][:, :-1]), dim=1)
    dh0 = a[:, 0] * g[:, 0]
    if mode == "linear":
        return {"dgate": g * before, "dx": g, "dh0": dh0}
    rest = 1 / (1 + torch.exp(s["gate"]))
    return {"dgate": g * (before - s["x"]) * a * rest, "dx": g * rest, "dh0": dh0}


def _splitmix(z):
    """splitmix64 on int64 tensors: the same bits as on unsigned ones."""
    z = z + (0x9E3779B97F4A7C15 - (1 << 64))
    z = (z ^ ((z >> 30) & 0x3FFFFFFFF)) * (0xBF58476D1CE4E5B9 - (1 << 64))
    z = (z ^ ((z >> 27) & 0x1FFFFFFFFF)) * (0x94D049BB133111EB - (1 << 64))
    return z ^ ((z >> 31) & 0x1FFFFFFFF)


def _splitmix_int(z):
    z = (z + 0x9E3779B97F4A7C15) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return z ^ (z >> 31)


def _signed(z):
    return z - (1 << 64) if z >> 63 else z


def _random16(s, t):
    """16 random bits for every element: a word for four neighbours, from seed, step, tensor and place."""
    key = _splitmix(s["ordinal"] + _signed(_splitmix_int((RNG_SEED + t) & _M64)))
    quad = torch.arange(BLOCK // 4, device=DEV)
    word = _splitmix((key + s["within"] * (BLOCK // 4)).unsqueeze(1) + quad)
    shift = 16 * torch.arange(4, device=DEV)
    return ((word.unsqueeze(2) >> shift) & 0xFFFF).reshape(-1)


def _scale(x, top):
    """A power of two for each block that takes its largest magnitude into [2^top, 2^(top+1))."""
    most = x.view(-1, BLOCK).abs().amax(dim=1)
    e = torch.clamp((most.view(torch.int32) >> 23), min=top + 1) - top
    return (e << 23).view(torch.float32)


def _load8(s):
    scale = s["scales"].view(-1, 2)
    m = s["m8"].view(torch.float8_e4m3fn).float().view(-1, BLOCK) * scale[:, :1]
    v = s["v8"].view(torch.float8_e5m2).float().view(-1, BLOCK) * scale[:, 1:]
    return m.view(-1), v.view(-1)


def _store8(s, m, v, random16):
    sm, sv = _scale(m, 7), _scale(v, 14)
    x = (m.view(-1, BLOCK) / sm.unsqueeze(1)).view(-1)
    s["m8"].copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
    y = (v.view(-1, BLOCK) / sv.unsqueeze(1)).view(-1)
    y = ((y.view(torch.int32) + (random16 << 5).to(torch.int32)) & ~0x1FFFFF).view(torch.float32)
    code = y.to(torch.float8_e5m2).view(torch.uint8)
    s["v8"].copy_(torch.where((v > 0) & (code == 0), 1, code))  # what is not zero stays so
    s["scales"].copy_(torch.stack((sm, sv), dim=1).view(-1))


def _adamw(s):
    t = s["t"]
    m, v = (s["m"], s["v"]) if s["case"]["bits"] == 32 else _load8(s)
    g, p = s["g"], s["p"]
    rest1, rest2 = float(np.float32(1) - np.float32(BETA1)), float(np.float32(1) - np.float32(BETA2))
    m = m * BETA1 + g * rest1
    v = v * BETA2 + (g * rest2) * g
    size, root = LR / (1 - BETA1 ** t), 1 / math.sqrt(1 - BETA2 ** t)
    p.copy_(p * (1 - LR * DECAY) - size * (m / (torch.sqrt(v) * root + EPS)))
    if s["case"]["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        _store8(s, m, v, _random16(s, t))


def _adamw_outputs(s):
    if s["case"]["bits"] == 32:
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    # the states are 8-bit floats, each block's in units of its scale
    return {"p": s["p"], "m": s["m8"].view(torch.float8_e4m3fn), "v": s["v8"].view(torch.float8_e5m2), "scales": s["scales"]}


# ---------------------------------------------------------------- the library's calls
_contexts = {}


def _ctx(stream):
    """The library's context for a device's stream, the one that a state's inputs were made on: calls come behind them."""
    if stream not in _contexts:
        from sliced_amd.device import Context
        _contexts[stream] = Context(stream[0], stream=stream[1])
    return _contexts[stream]


def _run_own(s):
    c = s["case"]
    ctx = _ctx(c["stream"])
    if c["op"] == "adamw":
        if c["bits"] == 32:
            ctx.call("slhip_adamw_step_multi", s["count"], *s["args"], s["lens"], LR, BETA1, BETA2, EPS, DECAY, s["t"], None)
        else:
            ctx.call("slhip_adamw8_step_multi", s["count"], *s["args"], s["lens"], LR, BETA1, BETA2, EPS, DECAY, s["t"], None, RNG_SEED)
        return _adamw_outputs(s)
    at = {k: v.data_ptr() for k, v in s.items() if k != "case"}
    if c["op"] == "norm":
        shape = (c["samples"], c["positions"], c["channels"], c["groups"], ACTS[c["act"]])
        if c["dir"] == "fwd":
            ctx.call("slhip_group_norm", *shape, EPS_NORM, at["x"], at["weight"], at["bias"], at["mean"], at["rstd"], at["out"])
            return {k: s[k] for k in ("out", "mean", "rstd")}
        ctx.call("slhip_group_norm_grad", *shape, at["x"], at["weight"], at["bias"], at["mean"], at["rstd"], at["dx"], at["dw"], at["db"],
                 at["dy"], 0.0)
        return {k: s[k] for k in ("dx", "dw", "db")}
    shape = (SCANS[c["mode"]], c["batch"], c["steps"], c["channels"])
    if c["dir"] == "fwd":
        ctx.call("slhip_gated_scan", *shape, at["gate"], at["x"], at["h0"], at["h"], at["h_last"])
        return {k: s[k] for k in ("h", "h_last")}
    ctx.call("slhip_gated_scan_grad", *shape, at["gate"], at["x"], at["h0"], at["h"], at["dgate"], at["dx"], at["dh0"], at["dh"],
             at["dh_last"], 0.0)
    return {k: s[k] for k in ("dgate", "dx", "dh0")}


def run(state):
    c = state["case"]
    if c["op"] == "adamw":
        state["t"] += 1
    if own:
        return _run_own(state)
    if c["op"] == "adamw":
        _adamw(state)
        return _adamw_outputs(state)
    if c["op"] == "norm":
        return _norm_fwd(state) if c["dir"] == "fwd" else _norm_bwd(state)
    if c["dir"] == "bwd":
        return _scan_bwd(state)
    h = _scan_plain(c["mode"], state["gate"], state["x"], state["h0"])
    return {"h": h, "h_last": h[:, -1].clone()}


# ---------------------------------------------------------------- 64 bits
def _exact_adamw(s):
    t = s["t"] + 1
    f = torch.float64
    g, p = s["g"].to(f), s["p"].to(f)
    if s["case"]["bits"] == 32:
        m, v = s["m"].to(f), s["v"].to(f)
    else:
        per = s["scales"].to(f).view(-1, 2).repeat_interleave(BLOCK, dim=0)
        m = s["m8"].view(torch.float8_e4m3fn).to(f) * per[:, 0]
        v = s["v8"].view(torch.float8_e5m2).to(f) * per[:, 1]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    step = (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    p = (1 - LR * DECAY) * p - LR * step
    if s["case"]["bits"] == 32:
        return {"p": p, "m": m, "v": v}

    def exponent(x):
        return ((x.view(torch.int64) >> 52) & 0x7FF) - 1023

    def by_blocks(x, top):
        blocks = x.view(-1, BLOCK)
        e = torch.clamp(exponent(blocks.abs().amax(dim=1)) - top, min=-126).to(f)
        scale = torch.exp2(e)
        return (blocks / scale.unsqueeze(1)).view(-1), scale

    def grid(x, bits, lowest):
        """The distance of the format's neighbours at x."""
        e = torch.clamp(exponent(x), min=lowest)
        return torch.exp2((e - bits).to(f))

    x, sm = by_blocks(m, 7)
    u = grid(x, 3, -6)
    m8 = torch.round(x / u) * u
    y, sv = by_blocks(v, 14)
    u = torch.exp2((exponent(y) - 2).to(f))  # two bits behind the leading one, whatever its place
    r = _random16(s, t).to(f) / 65536
    y = torch.where(y > 0, torch.floor(y / u + r) * u, y)
    u = grid(y, 2, -14)
    v8 = torch.where(y > 0, torch.clamp(torch.round(y / u) * u, min=2.0 ** -16), y)
    return {"p": p, "m": m8, "v": v8, "scales": torch.stack((sm, sv), dim=1).view(-1)}


def _exact_norm(s):
    c, f = s["case"], torch.float64
    n, p, d, k = c["samples"], c["positions"], c["channels"], c["groups"]
    x = s["x"].to(f).view(n, p, k, d // k).transpose(1, 2).reshape(n, k, -1)
    w, b = (s[q].to(f).view(1, k, 1, -1).expand(n, k, p, -1).reshape(n, k, -1) for q in ("weight", "bias"))

    def back(y):
        return y.view(n, k, p, -1).transpose(1, 2).reshape(n, p, d)

    if c["dir"] == "fwd":
        mean = x.sum(dim=2, keepdim=True) / x.shape[2]
        rstd = ((x - mean).square().sum(dim=2, keepdim=True) / x.shape[2] + EPS_NORM) ** -0.5
        u = (x - mean) * rstd * w + b
        y = {"none": lambda: u, "silu": lambda: u * torch.sigmoid(u),
             "gelu": lambda: u * 0.5 * torch.erfc(-u / math.sqrt(2))}[c["act"]]()
        return {"out": back(y), "mean": mean[..., 0], "rstd": rstd[..., 0]}
    mean, rstd = s["mean"].to(f).unsqueeze(2), s["rstd"].to(f).unsqueeze(2)
    hat = (x - mean) * rstd
    u = hat * w + b
    q = torch.sigmoid(u)
    slope = {"none": lambda: torch.ones_like(u), "silu": lambda: q + u * q * (1 - q),
             "gelu": lambda: 0.5 * torch.erfc(-u / math.sqrt(2)) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)}[c["act"]]()
    gu = s["dy"].to(f).view(n, p, k, d // k).transpose(1, 2).reshape(n, k, -1) * slope
    gx = gu * w
    dx = rstd * (gx - gx.sum(2, keepdim=True) / x.shape[2] - hat * ((gx * hat).sum(2, keepdim=True) / x.shape[2]))
    dw, db = (back(q).sum(dim=(0, 1)) for q in (gu * hat, gu))
    return {"dx": back(dx), "dw": dw, "db": db}


def _exact_scan(s):
    c, f = s["case"], torch.float64
    gate, x, h = s["gate"].to(f), s["x"].to(f), s["h0"].to(f)
    a = gate if c["mode"] == "linear" else torch.sigmoid(gate)
    steps = c["steps"]
    if c["dir"] == "fwd":
        b = x if c["mode"] == "linear" else x * torch.sigmoid(-gate)
        out = torch.empty_like(x)
        for t in range(steps):
            h = torch.addcmul(b[:, t], a[:, t], h)
            out[:, t] = h
        return {"h": out, "h_last": h}
    dh, g = s["dh"].to(f), s["dh_last"].to(f)
    sums = torch.empty_like(dh)
    for t in range(steps - 1, -1, -1):
        g = dh[:, t] + g
        sums[:, t] = g
        g = a[:, t] * g
    before = torch.cat((h.unsqueeze(1), s["h"].to(f)[:, :-1]), dim=1)
    if c["mode"] == "linear":
        return {"dgate": sums * before, "dx": sums, "dh0": g}
    return {"dgate": sums * (before - x) * a * torch.sigmoid(-gate), "dx": sums * torch.sigmoid(-gate), "dh0": g}


def exact(case, seed):
    s = prepare(case, seed)
    return {"adamw": _exact_adamw, "norm": _exact_norm, "scan": _exact_scan}[case["op"]](s)
