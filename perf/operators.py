"""Measured cases of the linear, grouped linear and group norm operators.

With `own` false, run() computes them in elementary torch operations in 32 bits; with `own` true it calls the
library through its Python bindings.
"""
import math

import torch

own = False

ACTS = ("none", "silu", "gelu_tanh", "gelu_erf")
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

_contexts = {}


def _context():
    """The library context of the current device, on torch's current stream."""
    from seedvr2_ncnn_b200 import abi

    dev = torch.cuda.current_device()
    if dev not in _contexts:
        _contexts[dev] = abi.Context(dev)
    ctx = _contexts[dev]
    ctx.set_stream(torch.cuda.current_stream(dev))
    return abi, ctx


# ------------------------------------------------------------------ cases
def listed():
    return [
        # The timestep MLP's second layer: one row, so the weight's bytes and the launch are all there is.
        {"name": "linear one row", "op": "linear", "m": 1, "n": 2560, "k": 2560, "pad": 0, "act": "silu", "bias": True,
         "gate": False, "residual": False, "out": "bf16"},
        # MLP up of the text rows alone.
        {"name": "linear text mlp up", "op": "linear", "m": 58, "n": 10240, "k": 2560, "pad": 0, "act": "gelu_tanh",
         "bias": True, "gate": False, "residual": False, "out": "bf16"},
        # A residual block's 1x1 shortcut over five 180 x 320 frames, added to the convolution's output.
        {"name": "linear vae shortcut", "op": "linear", "m": 288000, "n": 256, "k": 512, "pad": 0, "act": "none",
         "bias": True, "gate": False, "residual": True, "out": "bf16"},
        # MLP down of a 720p step: 21,600 video and 58 text rows onto the fp32 residual stream.
        {"name": "linear mlp down", "op": "linear", "m": 21658, "n": 2560, "k": 10240, "pad": 0, "act": "none",
         "bias": True, "gate": True, "residual": True, "out": "f32"},
        # Separate weights for the video and the text stream: two groups of very unequal size.
        {"name": "grouped two streams qkv", "op": "grouped", "rows": 21658, "groups": 2, "split": "streams", "n": 7680,
         "k": 2560, "act": "none", "bias": True, "gate": False, "residual": False, "out": "bf16"},
        # Eight ragged groups, some empty, as a router leaves them; rows behind the last group stay.
        {"name": "grouped eight ragged", "op": "grouped", "rows": 4101, "groups": 8, "split": "ragged", "n": 2560,
         "k": 2560, "act": "gelu_tanh", "bias": True, "gate": False, "residual": False, "out": "bf16"},
        # Many groups with a few rows each: every group's weight is read for hardly any rows.
        {"name": "grouped few rows each", "op": "grouped", "rows": 128, "groups": 64, "split": "ragged", "n": 2048,
         "k": 1024, "act": "silu", "bias": False, "gate": False, "residual": False, "out": "bf16"},
        # Widths off every tile, a gate and an fp32 residual.
        {"name": "grouped odd widths", "op": "grouped", "rows": 3001, "groups": 16, "split": "ragged", "n": 1001,
         "k": 1283, "act": "gelu_erf", "bias": True, "gate": True, "residual": True, "out": "f32"},
        # One small tile of the mid block: latency.
        {"name": "group norm small", "op": "norm", "i": 1, "r": 256, "c": 512, "g": 32, "act": "silu", "affine": True,
         "in": "bf16", "out": "bf16"},
        # The mid block at 720p: six latent frames of 90 x 160.
        {"name": "group norm mid", "op": "norm", "i": 6, "r": 14400, "c": 512, "g": 32, "act": "silu", "affine": True,
         "in": "bf16", "out": "bf16"},
        # The decoder's last level: two frames of 720 x 1280.
        {"name": "group norm full frame", "op": "norm", "i": 2, "r": 921600, "c": 128, "g": 32, "act": "silu",
         "affine": True, "in": "bf16", "out": "bf16"},
        # Ten channels a group and odd rows, fp32 as the attention layer takes it.
        {"name": "group norm odd", "op": "norm", "i": 3, "r": 3555, "c": 320, "g": 32, "act": "none", "affine": True,
         "in": "f32", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "grouped", "norm"])
    if op == "norm":
        while True:
            g = rng.choice([1, 8, 20, 32, 32, 32])
            c = g * _log(rng, 1, 48)
            i, r = _log(rng, 1, 24), _log(rng, 1, 921600)
            if c <= 2048 and 64 <= i * r * c <= 2 * 921600 * 128:
                break
        kind = rng.choice(["bf16", "f32"])
        if kind == "f32" and i * r * c > 921600 * 128:
            kind = "bf16"
        return {"op": op, "i": i, "r": r, "c": c, "g": g, "act": rng.choice(["none", "silu", "gelu_tanh", "gelu_erf"]),
                "affine": rng.random() < 0.8, "in": kind, "out": rng.choice(["bf16", kind])}
    while True:
        rows, n, k = _log(rng, 1, 60000), _log(rng, 8, 10240), _log(rng, 8, 10240)
        groups = _log(rng, 1, 64) if op == "grouped" else 1
        if rows * n * k <= 21658 * 2560 * 10240 and groups * n * k <= 300_000_000 and rows * (n + k) <= 300_000_000:
            break
    rest = {"n": n, "k": k, "act": rng.choice(ACTS), "bias": rng.random() < 0.7, "gate": rng.random() < 0.3,
            "residual": rng.random() < 0.5, "out": rng.choice(["bf16", "f32"])}
    if op == "linear":
        return {"op": op, "m": rows, "pad": rng.choice([0, 0, 8, 24]), **rest}
    return {"op": op, "rows": rows, "groups": groups, "split": "ragged", **rest}


# ------------------------------------------------------------------ inputs
def _offsets(case):
    """Row offsets of the groups, on the host: fixed by the case, so that work() knows which groups are empty."""
    rows, groups = case["rows"], case["groups"]
    if case["split"] == "streams":
        return [0, rows - 58, rows]
    gen = torch.Generator().manual_seed(rows * 131 + groups)
    share = torch.rand(groups, generator=gen).pow(2.0)
    share[torch.rand(groups, generator=gen) < 0.15] = 0.0
    if float(share.sum()) == 0.0:
        share[0] = 1.0
    used = rows - rows // 50  # the last rows belong to no group
    ends = torch.round(torch.cumsum(share.double(), 0) / float(share.double().sum()) * used).long().tolist()
    ends[-1] = used
    return [0] + ends


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pitch(k):
    return (k + 7) // 8 * 8


def _rows(gen, rows, k, pad=0):
    """Activations: normal values with a few large channels, bf16, in rows of a pitch of 16 bytes' multiple."""
    full = torch.empty(rows, _pitch(k) + pad, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    scale = torch.ones(full.shape[1], device="cuda")
    scale[:: max(1, full.shape[1] // 7)] = 6.0
    return full.mul_(scale.bfloat16())[:, :k]


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case)
    if case["op"] == "norm":
        shape = (case["i"], case["r"], case["c"])
        x = torch.empty(shape, device="cuda", dtype=DTYPES[case["in"]]).normal_(generator=gen)
        spread = torch.rand(case["c"], device="cuda", generator=gen) * 2 + 0.2
        shift = torch.randn(case["c"], device="cuda", generator=gen) * 1.5
        s["x"] = x.mul_(spread.to(x.dtype)).add_(shift.to(x.dtype))
        s["gamma"] = torch.randn(case["c"], device="cuda", generator=gen) * 0.2 + 1 if case["affine"] else None
        s["beta"] = torch.randn(case["c"], device="cuda", generator=gen) * 0.2 if case["affine"] else None
        s["out_buffer"] = torch.zeros(shape, device="cuda", dtype=DTYPES[case["out"]])
        return s
    rows, n, k = case.get("m", case.get("rows")), case["n"], case["k"]
    groups = case.get("groups", 1)
    s["a"] = _rows(gen, rows, k, case.get("pad", 0))
    w = torch.empty(groups, n, _pitch(k), device="cuda", dtype=torch.bfloat16)
    s["w"] = w.normal_(generator=gen).mul_(1.0 / math.sqrt(k))[:, :, :k]
    s["b"] = torch.randn(groups, n, device="cuda", generator=gen) * 0.1 if case["bias"] else None
    s["gate_v"] = torch.randn(groups, n, device="cuda", generator=gen) * 0.5 if case["gate"] else None
    dtype = DTYPES[case["out"]]
    s["res"] = torch.empty(rows, n, device="cuda", dtype=dtype).normal_(generator=gen) if case["residual"] else None
    s["out_buffer"] = torch.zeros(rows, n, device="cuda", dtype=dtype)
    if case["op"] == "grouped":
        s["host_offsets"] = _offsets(case)
        s["offsets"] = torch.tensor(s["host_offsets"], dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def _act(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "gelu_erf":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _plain_rows(s, a, w, b, gate, res):
    y = a @ w.t()
    if b is not None:
        y = y + b
    y = _act(y, s["act"])
    if gate is not None:
        y = y * gate
    return y if res is None else y + res.float()


def run(s):
    if own:
        abi, ctx = _context()
        act = {"none": abi.S2_ACT_NONE, "silu": abi.S2_ACT_SILU, "gelu_tanh": abi.S2_ACT_GELU_TANH,
               "gelu_erf": abi.S2_ACT_GELU_ERF}[s["act"]]
        if s["op"] == "norm":
            return abi.group_norm(ctx, s["x"], s["g"], s["gamma"], s["beta"], eps=1e-6, act=act, out=s["out_buffer"])
        if s["op"] == "linear":
            return abi.linear(ctx, s["a"], s["w"][0], None if s["b"] is None else s["b"][0], act=act,
                              gate=None if s["gate_v"] is None else s["gate_v"][0], residual=s["res"],
                              out=s["out_buffer"])
        return abi.grouped_linear(ctx, s["a"], s["w"], s["offsets"], s["b"], act=act, gate=s["gate_v"],
                                  residual=s["res"], out=s["out_buffer"])
    out = s["out_buffer"]
    if s["op"] == "norm":
        i, r, c, g = s["i"], s["r"], s["c"], s["g"]
        x = s["x"].float().view(i, r, g, c // g)
        d = x - x.mean(dim=(1, 3), keepdim=True)
        y = (d * torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + 1e-6)).view(i, r, c)
        if s["affine"]:
            y = y * s["gamma"] + s["beta"]
        return out.copy_(_act(y, s["act"]))
    a, w, b, gate, res = s["a"].float(), s["w"].float(), s["b"], s["gate_v"], s["res"]
    if s["op"] == "linear":
        return out.copy_(_plain_rows(s, a, w[0], None if b is None else b[0], None if gate is None else gate[0], res))
    at = s["host_offsets"]
    for g in range(s["groups"]):  # one product a group: its rows and its weight are its own
        lo, hi = at[g], at[g + 1]
        if lo < hi:
            out[lo:hi] = _plain_rows(s, a[lo:hi], w[g], None if b is None else b[g], None if gate is None else gate[g],
                                     None if res is None else res[lo:hi])
    return out


# ------------------------------------------------------------------ work and exact values
def work(case):
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "norm":
        n = case["i"] * case["r"] * case["c"]
        return {"bytes": n * (size[case["in"]] + size[case["out"]]) + (8 * case["c"] if case["affine"] else 0), "flops": 10 * n}
    n, k, o = case["n"], case["k"], size[case["out"]]
    if case["op"] == "linear":
        rows, weights, extra = case["m"], 1, 0
    else:
        at = _offsets(case)
        rows, weights, extra = at[-1], sum(b > a for a, b in zip(at, at[1:])), 4 * len(at)
    vectors = weights * n * 4 * (int(case["bias"]) + int(case["gate"]))
    return {"bytes": rows * k * 2 + weights * n * k * 2 + vectors + extra + rows * n * o * (1 + int(case["residual"])),
            "flops": 2 * rows * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64

    def activate(v):
        if case["act"] == "silu":
            return v * torch.sigmoid(v)
        if case["act"] == "gelu_tanh":
            return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
        if case["act"] == "gelu_erf":
            return v * 0.5 * torch.special.erfc(-v / math.sqrt(2))
        return v

    if case["op"] == "norm":
        i, r, c, g = case["i"], case["r"], case["c"], case["g"]
        out = torch.empty(i, r, c, device="cuda", dtype=f64)
        for n in range(i):
            x = s["x"][n].to(f64).view(r, g, c // g)
            var, mean = torch.var_mean(x, dim=(0, 2), unbiased=False, keepdim=True)
            y = ((x - mean) / torch.sqrt(var + 1e-6)).view(r, c)
            if case["affine"]:
                y = torch.addcmul(s["beta"].to(f64), y, s["gamma"].to(f64))
            out[n] = activate(y)
        return out
    rows = s["a"].shape[0]
    at = s.get("host_offsets", [0, rows])
    out = torch.zeros(rows, case["n"], device="cuda", dtype=f64)
    for g, (lo, hi) in enumerate(zip(at, at[1:])):
        v = torch.mm(s["a"][lo:hi].to(f64), s["w"][g].to(f64).t())
        if case["bias"]:
            v += s["b"][g].to(f64)
        v = activate(v)
        if case["gate"]:
            v *= s["gate_v"][g].to(f64)
        if case["residual"]:
            v += s["res"][lo:hi].to(f64)
        out[lo:hi] = v
    return out
