"""Linear layers of group-scaled 4-bit weights, and the norm and rotation of attention heads, as measurable cases.

A weight is (code - zero) * scale: codes 0..15, one scale and one zero point (8 where there are none) per group of consecutive
values of K.  Activations stay what they are, 16-bit floating point.  A case is one of

  linear  `layers` projections (rk_npu_g4_run_device);
  swiglu  `layers` gate / up projections with silu(gate) * up behind them (rk_npu_g4_run_swiglu_device);
  heads   queries and keys of a joint projection's rows, each head normed (or not) and rotated by its token's position, which may
          have several axes (rk_npu_heads_norm_rotate_device).

Several layers are used where few rows meet the weights: each has weights of its own, as in a model.

In the plain form a product's weights are decoded in the call: codes, scales and zero points are what a program holds.
"""
import ctypes
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_BASE = 1e6  # of the rotation's frequencies

# The largest drawn case costs what the largest listed one does.
_MOST_PRODUCTS = 4096 * 4096 * 14336
_MOST_VALUES = 8192 * 40 * 128


def _linear(name, M, K, N, group, zeros, type, out, layers=1, kind="linear"):
    return {"name": name, "kind": kind, "M": M, "K": K, "N": N, "group": group, "zeros": zeros, "type": type, "out": out, "layers": layers}


def _heads(name, M, q_heads, k_heads, D, R, type, norm, axes, pairs):
    return {"name": name, "kind": "heads", "M": M, "q_heads": q_heads, "k_heads": k_heads, "D": D, "R": R, "type": type, "norm": norm, "axes": axes, "pairs": pairs}


def listed():
    return [
        # One token through a small projection, the finest groups: latency.
        _linear("linear_1row_small", 1, 512, 384, 32, True, "bf16", "bf16"),
        # One token of one sequence through the up projection of four layers: the weights' bytes.
        _linear("linear_1row", 1, 4096, 14336, 128, False, "f16", "f16", layers=4),
        # Eight sequences decoded together, the down projection of four layers: long K, few rows.
        _linear("linear_8rows_down", 8, 14336, 4096, 128, True, "bf16", "bf16", layers=4),
        # A short prompt on a small model, no size a multiple of anything, fp32 out.
        _linear("linear_61rows_ragged", 61, 2050, 1999, 64, True, "f16", "f32"),
        # Many decoding sequences, or a short prompt.
        _linear("linear_128rows", 128, 4096, 11008, 128, False, "f16", "f16"),
        # A long prompt through the widest projection: the largest product.
        _linear("linear_4096rows", 4096, 4096, 14336, 128, False, "bf16", "bf16"),
        # One token through the gate / up projection of two layers.
        _linear("swiglu_1row", 1, 4096, 14336, 128, False, "bf16", "bf16", layers=2, kind="swiglu"),
        # A chunk of a prompt through one, finer groups with zero points.
        _linear("swiglu_512rows", 512, 4096, 14336, 64, True, "f16", "f16", kind="swiglu"),
        # One token behind its QKV projection: latency.
        _heads("heads_1row", 1, 32, 8, 128, 128, "bf16", True, 1, "halves"),
        # A long prompt behind it.
        _heads("heads_8192rows", 8192, 32, 8, 128, 128, "bf16", True, 1, "halves"),
        # Frames of a video among text: time, height and width, no norm.
        _heads("heads_video", 2521, 28, 4, 128, 128, "f16", False, 3, "halves"),
        # Patches of an image, two axes, small odd-sized heads, neighbouring values turned, in fp32.
        _heads("heads_image_ragged", 1521, 15, 5, 90, 60, "f32", True, 2, "neighbours"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """A size of lo..hi: mostly a multiple of `step`, now and then any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 0.3 else max(-(-lo // step), round(v / step)) * step


def _layers(rows, weights):
    """Layers of a drawn case: few rows meet weights that come from memory (up to four layers, about 64 MB)."""
    return 1 if rows > 64 else max(1, min(4, int(120e6 / weights)))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "swiglu", "heads", "heads"])
    type = rng.choice(["f16", "bf16"])
    if kind == "heads":
        D = rng.choice([64, 80, 96, 128, 128, 256, 2 * rng.randint(16, 128)])
        axes = rng.choice([1, 1, 2, 3, 4])
        R = D if rng.random() < 0.6 else 2 * rng.randint(axes, D // 2)
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 4, 7, 8])
        M = _log_int(rng, 1, min(16384, _MOST_VALUES // ((q_heads + k_heads) * D)))
        return {"kind": kind, "M": M, "q_heads": q_heads, "k_heads": k_heads, "D": D, "R": R, "type": rng.choice([type, type, "f32"]),
                "norm": rng.random() < 0.6, "axes": axes, "pairs": rng.choice(["halves", "halves", "neighbours"])}
    while True:
        M = _log_int(rng, 1, 4096)
        K, N = _size(rng, 512, 14336, 128), _size(rng, 512, 14336, 128)
        both = 2 if kind == "swiglu" else 1
        if M * K * N * both <= _MOST_PRODUCTS:
            return {"kind": kind, "M": M, "K": K, "N": N, "group": rng.choice([32, 64, 128, 128]), "zeros": rng.random() < 0.5, "type": type,
                    "out": rng.choice([type, type, "f32"]), "layers": _layers(M, K * N * both)}


def work(case):
    M = case["M"]
    if case["kind"] == "heads":
        values = M * (case["q_heads"] + case["k_heads"]) * case["D"]
        return {"bytes": 2 * values * _SIZE[case["type"]] + 4 * case["axes"] * M, "flops": 10 * values}
    K, N, rows = case["K"], case["N"], case["N"] * (2 if case["kind"] == "swiglu" else 1)
    weights = rows * (-(-K // 2)) + rows * (-(-K // case["group"])) * (3 if case["zeros"] else 2)
    one = M * K * _SIZE[case["type"]] + M * N * _SIZE[case["out"]] + weights
    return {"bytes": case["layers"] * one, "flops": case["layers"] * 2 * M * K * rows}


# ---- what a program holds before the call --------------------------------------------------

_sessions = []


def _session():
    """The process's one context and domain, as a program opens them once."""
    if not _sessions:
        from rknpu2_matmul_open_amd import ops
        _sessions.append(ops.Session())
    return _sessions[0]


class _State:
    """A case's inputs and, for the framework's calls, its handles and outputs; the handles are given back with it."""

    def __init__(self, case):
        self.case, self.layers, self.handles = case, [], []

    def __del__(self):
        for h in self.handles:
            h.close()


def _rows(gen, M, K, type):
    """N(0, 1) rows with the outliers that activations show (0.5 % of the values, twenty times larger)."""
    x = torch.randn((M, K), generator=gen, device="cuda")
    far = torch.rand((M, K), generator=gen, device="cuda") < 0.005
    return torch.where(far, x * 20, x).to(_TYPES[type])


def _weights(gen, N, K, group, zeros):
    """N(0, 0.02) weights of a projection as a checkpoint holds them: codes by output channel, two a byte, the first in the low half;
    scales in fp16 and zero points by output channel and group.  Without zero points the range is symmetric about 8."""
    groups = -(-K // group)
    w = torch.randn((N, K), generator=gen, device="cuda").mul_(0.02)
    w = torch.nn.functional.pad(w, (0, groups * group - K)).view(N, groups, group)
    if zeros:
        low, high = w.amin(dim=2).clamp(max=0), w.amax(dim=2).clamp(min=0)
        scale = ((high - low) / 15).clamp(min=1e-6).half()
        zero = torch.round(-low / scale.float()).clamp(0, 15)
    else:
        scale = (w.abs().amax(dim=2) / 7.5).clamp(min=1e-6).half()
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    code = torch.round(w / scale.float()[:, :, None] + zero[:, :, None]).clamp_(0, 15).view(N, -1)[:, :K].to(torch.uint8)
    code = torch.nn.functional.pad(code, (0, K % 2))
    return {"codes": code[:, 0::2] | code[:, 1::2] << 4, "scales": scale, "zeros": zero.to(torch.uint8) if zeros else None}


def _positions(gen, M, axes):
    """Positions by axis and token: a text's far into a long context, or grids of patches one behind the other, with a time axis or without."""
    start = int(torch.randint(0, 500000, (1,), generator=gen, device="cuda"))
    t = torch.arange(M, device="cuda")
    if axes == 1:
        return (start + t).to(torch.int32)[None].contiguous()
    width = max(1, int(math.sqrt(M / 4)))
    grid = [t // width % width, t % width]  # height, width
    if axes > 2:
        grid.insert(0, t // (width * width))
    if axes > 3:
        grid.append(t)
    return torch.stack([start % 4096 + g for g in grid]).to(torch.int32)


def _pair_axis(case):
    """Which axis turns which pair: sections of (nearly) one length, the first one the smallest."""
    pairs, axes = case["R"] // 2, case["axes"]
    return [min(axes - 1, (i * axes + axes - 1) // max(1, pairs)) for i in range(pairs)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state, M = _State(case), case["M"]
    if case["kind"] == "heads":
        q, k, D = case["q_heads"], case["k_heads"], case["D"]
        channel = lambda: 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")  # noqa: E731
        joint = _rows(gen, M, (q + 2 * k) * D, case["type"]).view(M, q + 2 * k, D)  # queries, keys and values of a token
        i = torch.arange(case["R"] // 2, device="cuda", dtype=torch.float64)
        layer = {"q": joint[:, :q], "k": joint[:, q:q + k], "q_weight": channel(), "k_weight": channel(),
                 "positions": _positions(gen, M, case["axes"]), "inv_freq": (_BASE ** (-2 * i / max(1, case["R"]))).float(), "axis": _pair_axis(case),
                 "q_out": torch.empty((M, q, D), dtype=_TYPES[case["type"]], device="cuda"),
                 "k_out": torch.empty((M, k, D), dtype=_TYPES[case["type"]], device="cuda")}
        layer["axis_of_pair"] = torch.tensor(layer["axis"], device="cuda")
        state.layers.append(layer)
    else:
        rows = case["N"] * (2 if case["kind"] == "swiglu" else 1)
        for _ in range(case["layers"]):
            layer = _weights(gen, rows, case["K"], case["group"], case["zeros"])
            layer.update(x=_rows(gen, M, case["K"], case["type"]), y=torch.empty((M, case["N"]), dtype=_TYPES[case["out"]], device="cuda"))
            state.layers.append(layer)
    torch.cuda.synchronize()
    if own:
        _hold(state)
    return state


def _address(x):
    return ctypes.c_void_p(x.data_ptr() if x is not None else None)


def _hold(state):
    """What a program keeps: handles (weights of each layer, one workspace for all layers of a shape) and its calls' arguments."""
    from rknpu2_matmul_open_amd import capi, ops
    s, case, M = _session(), state.case, state.case["M"]
    lib, kind = s.lib, {"f32": capi.MX4_F32, "f16": capi.MX4_F16, "bf16": capi.MX4_BF16}

    def held(handle):
        state.handles.append(handle)
        return handle

    if case["kind"] == "heads":
        layer = state.layers[0]
        a = layer["args"] = ops.heads_args(s, layer["q"], layer["k"], layer["q_out"], layer["k_out"], norm=case["norm"], eps=_EPS,
                                           q_weight=layer["q_weight"] if case["norm"] else None, k_weight=layer["k_weight"] if case["norm"] else None,
                                           positions=layer["positions"], inv_freq=layer["inv_freq"], pair_axis=layer["axis"], neighbours=case["pairs"] == "neighbours")
        layer["call"] = (lib.rk_npu_heads_norm_rotate_device, (s.ctx, ctypes.byref(a)))
        return
    K, N, swiglu = case["K"], case["N"], case["kind"] == "swiglu"
    rows = 2 * N if swiglu else N
    ws = held(ops.G4Workspace(s, M, K, rows))
    for layer in state.layers:
        w = held(ops.G4Weights.from_device(s, K, rows, case["group"], layer["codes"], layer["scales"], layer["zeros"], gate_up=swiglu))
        layer["call"] = (lib.rk_npu_g4_run_swiglu_device if swiglu else lib.rk_npu_g4_run_device,
                         (ws.h, w.h, M, kind[case["type"]], _address(layer["x"]), K, kind[case["out"]], _address(layer["y"]), N))


# ---- one pass ------------------------------------------------------------------------------


def run(state):
    return [_run_layer(state.case, layer) for layer in state.layers]


def _run_layer(case, layer):
    if own:
        call, args = layer["call"]
        if call(*args):
            raise RuntimeError("%s failed" % call.__name__)
        return {"q": layer["q_out"], "k": layer["k_out"]} if case["kind"] == "heads" else layer["y"]
    return {"linear": _plain_linear, "swiglu": _plain_swiglu, "heads": _plain_heads}[case["kind"]](case, layer)


# ---- the plain forms -----------------------------------------------------------------------


def _decode(case, layer):
    codes, scales, zeros = layer["codes"], layer["scales"], layer["zeros"]
    code = torch.stack((codes & 15, codes >> 4), dim=2).flatten(1)[:, :case["K"]].float()
    wide = lambda x: x.float().repeat_interleave(case["group"], dim=1)[:, :case["K"]]  # noqa: E731
    return (code - (8 if zeros is None else wide(zeros))) * wide(scales)


def _plain_linear(case, layer):
    return (layer["x"].float() @ _decode(case, layer).t()).to(_TYPES[case["out"]])


def _plain_swiglu(case, layer):
    both = layer["x"].float() @ _decode(case, layer).t()
    gate, up = both[:, :case["N"]], both[:, case["N"]:]
    return (gate / (1 + torch.exp(-gate)) * up).to(_TYPES[case["out"]])


def _turned(case, layer, x, weight):
    x, R = x.float(), case["R"]
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + _EPS) * weight
    angle = layer["positions"].double()[layer["axis_of_pair"]].t() * layer["inv_freq"].double()  # [token, pair]: 64 bits, positions are far
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if case["pairs"] == "halves":
        a, b = x[:, :, :R // 2], x[:, :, R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=2)
    else:
        a, b = x[:, :, 0:R:2], x[:, :, 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=3).flatten(2)
    return torch.cat((turned, x[:, :, R:]), dim=2).to(_TYPES[case["type"]])


def _plain_heads(case, layer):
    return {"q": _turned(case, layer, layer["q"], layer["q_weight"]), "k": _turned(case, layer, layer["k"], layer["k_weight"])}


# ---- the definitions in 64 bits, apart from the above --------------------------------------


def _weights64(case, layer):
    N, K = layer["codes"].shape[0], case["K"]
    w = torch.empty((N, 2 * layer["codes"].shape[1]), dtype=torch.float64, device="cuda")
    w[:, 0::2] = (layer["codes"] % 16).double()
    w[:, 1::2] = (layer["codes"] // 16).double()
    w = w[:, :K]
    for g in range(layer["scales"].shape[1]):
        part = w[:, g * case["group"]:(g + 1) * case["group"]]
        part -= 8.0 if layer["zeros"] is None else layer["zeros"][:, g:g + 1].double()
        part *= layer["scales"][:, g:g + 1].double()
    return w


def _heads64(case, layer, x, weight):
    """Pairs as complex numbers, turned by a product with exp(i angle)."""
    x, R = x.double(), case["R"]
    if case["norm"]:
        x = x / torch.sqrt(x.square().sum(dim=2, keepdim=True) / case["D"] + _EPS) * weight.double()
    first = [i if case["pairs"] == "halves" else 2 * i for i in range(R // 2)]
    second = [i + (R // 2 if case["pairs"] == "halves" else 1) for i in first]
    found = x.clone()
    for i, axis in enumerate(layer["axis"]):
        angle = layer["positions"][axis].double() * float(layer["inv_freq"][i])
        turned = torch.complex(x[:, :, first[i]], x[:, :, second[i]]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        found[:, :, first[i]], found[:, :, second[i]] = turned.real, turned.imag
    return found


def exact(case, seed):
    found = []
    state = prepare(case, seed)
    for layer in state.layers:
        if case["kind"] == "heads":
            found.append({"q": _heads64(case, layer, layer["q"], layer["q_weight"]), "k": _heads64(case, layer, layer["k"], layer["k_weight"])})
            continue
        y = layer["x"].double() @ _weights64(case, layer).t()
        if case["kind"] == "swiglu":
            gate, up = y.split(case["N"], dim=1)
            y = gate * torch.sigmoid(gate) * up
        found.append(y)
    return found
