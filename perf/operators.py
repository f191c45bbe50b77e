"""The operators of microscaled 4-bit layers, as measurable cases.

MX4 data is e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in blocks of 32 along K that share a power of two:
a row of K values is ceil(K / 32) blocks of 16 bytes (first value in the low half of the first byte) and as many scale
bytes (exponent + 127; 255: not a number).  A case is one of

  quant   rows are quantized and read back (rk_npu_mx4_quantize_device, rk_npu_mx4_dequantize_device);
  linear  `layers` projections: the rows are quantized and multiplied with MX4 weights (rk_npu_mx4_run_device);
  norm    the norms after a block and before the next one, with the block's gate and the residual's scale
          (rk_npu_block_norm_device);
  block   `layers` gated FFN blocks on the residual stream: norm, gate / up product with SwiGLU, down product, norm, gate and
          residual (rk_npu_mx4_run_ffn_block_device).

Several layers are used where few rows meet the weights: each has weights of its own, as in a model, so that they come
from memory and not from a cache that the previous call filled.

In the plain form a product's weights are decoded in the call: the codes and scales are what a program holds.
"""
import ctypes
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_SCALE = 0.75  # of the residual stream

# The largest drawn case costs what the largest listed one does.
_MOST_PRODUCTS = 4096 * 4096 * 14336
_MOST_VALUES = 4096 * 14336


def _quant(name, M, K, type):
    return {"name": name, "kind": "quant", "M": M, "K": K, "type": type}


def _linear(name, M, K, N, type, out, layers=1):
    return {"name": name, "kind": "linear", "M": M, "K": K, "N": N, "type": type, "out": out, "layers": layers}


def _norm(name, M, D, stream, type, after, gate):
    return {"name": name, "kind": "norm", "M": M, "D": D, "stream": stream, "type": type, "after": after, "gate": gate}


def _block(name, M, H, I, type, after, gate, layers=1):
    return {"name": name, "kind": "block", "M": M, "H": H, "I": I, "type": type, "after": after, "gate": gate, "layers": layers}


def listed():
    return [
        # One token's row quantized on its own, and read back: latency.
        _quant("quant_1row", 1, 4096, "f16"),
        # The middle of a long prompt's FFN: the largest rows that a model quantizes.
        _quant("quant_4096rows", 4096, 14336, "bf16"),
        # One token of one sequence through the up projection of four layers: the weights' bytes.
        _linear("linear_1row", 1, 4096, 14336, "f16", "f16", layers=4),
        # Sixteen sequences decoded together, the down projection of two layers: long K, few rows.
        _linear("linear_16rows_down", 16, 14336, 4096, "bf16", "bf16", layers=2),
        # A short prompt on a small model, no size a multiple of anything, fp32 in and out.
        _linear("linear_61rows_ragged", 61, 2050, 1999, "f32", "f32"),
        # Many decoding sequences, or a short prompt.
        _linear("linear_128rows", 128, 4096, 11008, "f16", "f16"),
        # Prefill of 2048 tokens, a square projection.
        _linear("linear_2048rows", 2048, 4096, 4096, "f16", "f16"),
        # A long prompt through the widest projection: the largest product.
        _linear("linear_4096rows", 4096, 4096, 14336, "bf16", "bf16"),
        # Between two blocks of one token: norm after, channel gate, residual, norm before.
        _norm("norm_1row", 1, 4096, "bf16", "bf16", True, "channel"),
        # The same of a long prompt, the residual stream in fp32 and a gate value of its own for each value.
        _norm("norm_4096rows", 4096, 4096, "f32", "bf16", True, "full"),
        # One token through two whole FFN blocks.
        _block("block_1row", 1, 4096, 14336, "bf16", True, "channel", layers=2),
        # A chunk of a prompt through one.
        _block("block_512rows", 512, 4096, 14336, "bf16", False, "none"),
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
    kind = rng.choice(["quant", "linear", "linear", "linear", "norm", "block"])
    type = rng.choice(["f16", "bf16"])
    gate = rng.choice(["none", "channel", "full"])
    if kind == "quant":
        K = _size(rng, 64, 14336, 32)
        return {"kind": kind, "M": _log_int(rng, 1, min(65536, _MOST_VALUES // K)), "K": K, "type": rng.choice(["f32", "f16", "bf16"])}
    if kind == "norm":
        D = _size(rng, 256, 14336, 64)
        return {"kind": kind, "M": _log_int(rng, 1, min(16384, _MOST_VALUES // 4 // D)), "D": D, "stream": rng.choice([type, "f32"]), "type": type,
                "after": rng.random() < 0.5, "gate": gate}
    while True:
        M = _log_int(rng, 1, 4096)
        K, N = _size(rng, 512, 14336, 128), _size(rng, 512, 14336, 128)
        if kind == "linear" and M * K * N <= _MOST_PRODUCTS:
            return {"kind": kind, "M": M, "K": K, "N": N, "type": rng.choice([type, "f32"]), "out": rng.choice([type, "f32"]), "layers": _layers(M, K * N)}
        if kind == "block" and 3 * M * K * N <= _MOST_PRODUCTS:
            return {"kind": kind, "M": M, "H": K, "I": N, "type": type, "after": rng.random() < 0.5, "gate": gate, "layers": _layers(M, 3 * K * N)}


def _mx4_bytes(rows, K):
    return rows * (-(-K // 32)) * 17


def work(case):
    M = case["M"]
    if case["kind"] == "quant":  # values in, MX4 out; MX4 in, values (fp32) out
        return {"bytes": M * case["K"] * (_SIZE[case["type"]] + 4) + 2 * _mx4_bytes(M, case["K"]), "flops": 4 * M * case["K"]}
    if case["kind"] == "linear":
        K, N = case["K"], case["N"]
        one = M * K * _SIZE[case["type"]] + M * N * _SIZE[case["out"]] + _mx4_bytes(N, K)
        return {"bytes": case["layers"] * one, "flops": case["layers"] * 2 * M * K * N}
    gate = {"none": 0, "channel": 1, "full": M}[case["gate"]]
    if case["kind"] == "norm":
        D, s, t = case["D"], _SIZE[case["stream"]], _SIZE[case["type"]]
        return {"bytes": M * D * 2 * (s + t) + gate * D * t + 4 * D * (1 + case["after"]), "flops": 8 * M * D}
    H, I, t = case["H"], case["I"], _SIZE[case["type"]]
    one = _mx4_bytes(2 * I, H) + _mx4_bytes(H, I) + (2 * M + gate) * H * t + 4 * H * (1 + case["after"])
    return {"bytes": case["layers"] * one, "flops": case["layers"] * 6 * M * H * I}


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


def _weights(gen, N, K):
    """N(0, 0.02) weights of a projection as a checkpoint holds them: codes and scales by output channel."""
    return _encode(torch.randn((N, K), generator=gen, device="cuda").mul_(0.02))


def _channel(gen, D):
    return 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")


def _gate(gen, case, D):
    if case["gate"] == "none":
        return None
    shape = (D,) if case["gate"] == "channel" else (case["M"], D)
    return torch.rand(shape, generator=gen, device="cuda").to(_TYPES[case["type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state, M = _State(case), case["M"]
    empty = lambda shape, type: torch.empty(shape, dtype=type, device="cuda")  # noqa: E731
    if case["kind"] == "quant":
        K = case["K"]
        state.layers.append({"x": _rows(gen, M, K, case["type"]), "codes": empty((M, -(-K // 32) * 16), torch.uint8),
                             "scales": empty((M, -(-K // 32)), torch.uint8), "values": empty((M, K), torch.float32)})
    elif case["kind"] == "linear":
        for _ in range(case["layers"]):
            codes, scales = _weights(gen, case["N"], case["K"])
            state.layers.append({"x": _rows(gen, M, case["K"], case["type"]), "codes": codes, "scales": scales,
                                 "y": empty((M, case["N"]), _TYPES[case["out"]])})
    elif case["kind"] == "norm":
        D = case["D"]
        state.layers.append({"stream": _rows(gen, M, D, case["stream"]), "branch": _rows(gen, M, D, case["type"]),
                             "after": _channel(gen, D) if case["after"] else None, "gate": _gate(gen, case, D), "weight": _channel(gen, D),
                             "stream_out": empty((M, D), _TYPES[case["stream"]]), "y": empty((M, D), _TYPES[case["type"]])})
    else:
        H, I = case["H"], case["I"]
        for _ in range(case["layers"]):
            gu, gu_scales = _weights(gen, 2 * I, H)
            down, down_scales = _weights(gen, H, I)
            state.layers.append({"stream": _rows(gen, M, H, case["type"]), "gu": gu, "gu_scales": gu_scales, "down": down, "down_scales": down_scales,
                                 "weight": _channel(gen, H), "after": _channel(gen, H) if case["after"] else None, "gate": _gate(gen, case, H),
                                 "branch": empty((M, H), torch.float32), "stream_out": empty((M, H), _TYPES[case["type"]])})
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

    if case["kind"] == "quant":
        K = case["K"]
        for layer in state.layers:
            x, codes, scales, values = (_address(layer[k]) for k in ("x", "codes", "scales", "values"))
            layer["calls"] = [(lib.rk_npu_mx4_quantize_device, (s.ctx, kind[case["type"]], M, K, x, K, codes, scales)),
                              (lib.rk_npu_mx4_dequantize_device, (s.ctx, capi.MX4_F32, M, K, codes, scales, values, K))]
    elif case["kind"] == "linear":
        K, N = case["K"], case["N"]
        ws = held(ops.MX4Workspace(s, M, K, N))
        for layer in state.layers:
            w = held(ops.MX4Weights.from_device(s, K, N, layer["codes"].data_ptr(), layer["scales"].data_ptr()))
            layer["calls"] = [(lib.rk_npu_mx4_run_device, (ws.h, w.h, M, kind[case["type"]], _address(layer["x"]), K, kind[case["out"]],
                                                           _address(layer["y"]), N))]
    else:
        D = case["D"] if case["kind"] == "norm" else case["H"]
        if case["kind"] == "block":
            gu_ws, down_ws = held(ops.MX4Workspace(s, M, D, 2 * case["I"])), held(ops.MX4Workspace(s, M, case["I"], D))
        for layer in state.layers:
            a = layer["args"] = capi.BlockNormArgs()
            lib.rk_npu_block_norm_args_init(ctypes.byref(a), M, D)
            a.eps, a.residual_scale = _EPS, _SCALE
            a.residual_type = kind[case["stream"] if case["kind"] == "norm" else case["type"]]
            a.gate_type = kind[case["type"]]
            a.residual_ld = a.branch_ld = a.residual_out_ld = D
            a.gate_ld = D if case["gate"] == "full" else 0
            a.residual, a.gate, a.residual_out = _address(layer["stream"]), _address(layer["gate"]), _address(layer["stream_out"])
            a.weight, a.branch_weight = _address(layer["weight"]), _address(layer["after"])
            if case["kind"] == "norm":
                a.branch_type = a.y_type = kind[case["type"]]
                a.branch, a.y, a.y_ld = _address(layer["branch"]), _address(layer["y"]), D
                layer["calls"] = [(lib.rk_npu_block_norm_device, (s.ctx, ctypes.byref(a)))]
            else:
                a.branch_type = capi.MX4_F32
                gu = held(ops.MX4Weights.from_device(s, D, 2 * case["I"], layer["gu"].data_ptr(), layer["gu_scales"].data_ptr(), gate_up=True))
                down = held(ops.MX4Weights.from_device(s, case["I"], D, layer["down"].data_ptr(), layer["down_scales"].data_ptr()))
                layer["calls"] = [(lib.rk_npu_mx4_run_ffn_block_device, (gu_ws.h, gu.h, down_ws.h, down.h, ctypes.byref(a), _address(layer["branch"]), None))]


# ---- one pass ------------------------------------------------------------------------------


def run(state):
    return [_run_layer(state.case, layer) for layer in state.layers]


def _run_layer(case, layer):
    if own:
        for call, args in layer["calls"]:
            if call(*args):
                raise RuntimeError("%s failed" % call.__name__)
        return {"quant": lambda: {"scales": layer["scales"], "values": layer["values"]}, "linear": lambda: layer["y"],
                "norm": lambda: {"stream": layer["stream_out"], "y": layer["y"]}, "block": lambda: layer["stream_out"]}[case["kind"]]()
    return {"quant": _plain_quant, "linear": _plain_linear, "norm": _plain_norm, "block": _plain_block}[case["kind"]](case, layer)


# ---- the plain forms -----------------------------------------------------------------------

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _encode(x):
    """MX4 codes and scales of rows of any type."""
    rows, K = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(rows, -1, 32)
    most = x.abs().amax(dim=2)
    exponent = (torch.frexp(most).exponent - 3).clamp(min=-127)  # most = 0.5 .. 1 times 2^exponent of frexp
    exponent = torch.where(most == 0, -127, exponent)
    v = torch.ldexp(x, -exponent[:, :, None])
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6)
    code = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = torch.where(torch.signbit(x), code + 8, code)
    bad = ~torch.isfinite(most)
    code = torch.where(bad[:, :, None], 0, code).view(rows, -1, 2)
    scales = torch.where(bad, 255, exponent + 127).to(torch.uint8)
    return (code[:, :, 0] | code[:, :, 1] << 4).to(torch.uint8), scales


def _decode(codes, scales, K):
    """The values that MX4 rows stand for, in fp32."""
    rows = codes.shape[0]
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), dim=2).to(torch.int32)].view(rows, -1, 32)
    scale = torch.where(scales == 255, float("nan"), torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.to(torch.int32) - 127))
    return (v * scale[:, :, None]).view(rows, -1)[:, :K]


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS) * weight


def _residual(stream, branch, after, gate):
    branch = branch if after is None else _rms(branch, after)
    return _SCALE * stream + (branch if gate is None else branch * gate.float())


def _plain_quant(case, layer):
    codes, scales = _encode(layer["x"])
    return {"scales": scales, "values": _decode(codes, scales, case["K"])}


def _plain_linear(case, layer):
    x = _decode(*_encode(layer["x"]), case["K"])
    return (x @ _decode(layer["codes"], layer["scales"], case["K"]).t()).to(_TYPES[case["out"]])


def _plain_norm(case, layer):
    r = _residual(layer["stream"].float(), layer["branch"].float(), layer["after"], layer["gate"])
    return {"stream": r.to(_TYPES[case["stream"]]), "y": _rms(r, layer["weight"]).to(_TYPES[case["type"]])}


def _plain_block(case, layer):
    H, I = case["H"], case["I"]
    stream = layer["stream"].float()
    x = _decode(*_encode(_rms(stream, layer["weight"])), H)
    both = x @ _decode(layer["gu"], layer["gu_scales"], H).t()
    gate, up = both[:, :I], both[:, I:]
    middle = _decode(*_encode(gate / (1 + torch.exp(-gate)) * up), I)
    branch = middle @ _decode(layer["down"], layer["down_scales"], I).t()
    return _residual(stream, branch, layer["after"], layer["gate"]).to(_TYPES[case["type"]])


# ---- the definitions in 64 bits, apart from the above --------------------------------------


def _values64(x):
    """What each value of rows becomes as MX4: the nearest of the sixteen multiples of its block's scale, ties to an even code."""
    rows, K = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -K % 32)).reshape(rows, -1, 32)
    most = x.abs().amax(dim=2, keepdim=True)
    power = torch.floor(torch.log2(most))
    power = power + (torch.exp2(power + 1) <= most) - (torch.exp2(power) > most).double()  # a logarithm may be rounded over a border
    scale = torch.exp2(torch.where(most > 0, power - 2, -127.0).clamp(min=-127.0))
    v = x.abs() / scale
    # a border that belongs to the larger code is one where that code is even
    borders = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
    size = torch.zeros_like(v)
    for k, (border, up) in enumerate(borders):
        size += ((v >= border) if up else (v > border)) * (_VALUES[k + 1] - _VALUES[k])
    return (torch.copysign(size, x) * scale).view(rows, -1)[:, :K], scale[:, :, 0]


def _stored64(codes, scales, K):
    """The values of stored rows, from the fields of each code."""
    code = torch.stack((codes % 16, codes // 16), dim=2).flatten(1).long()
    e, m = code // 2 % 4, (code % 2).double()
    size = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.exp2(e.double() - 1))
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)
    return ((1 - 2 * (code // 8)).double() * size * scale)[:, :K]


def _normed64(x, weight):
    return x / torch.sqrt(x.square().sum(dim=1, keepdim=True) / x.shape[1] + _EPS) * weight.double()


def _joined64(layer, branch):
    if layer["after"] is not None:
        branch = _normed64(branch, layer["after"])
    if layer["gate"] is not None:
        branch = branch * layer["gate"].double()
    return layer["stream"].double() * _SCALE + branch


def exact(case, seed):
    found = []
    state = prepare(case, seed)
    for layer in state.layers:
        if case["kind"] == "quant":
            values, _ = _values64(layer["x"])
            found.append({"scales": None, "values": values})
        elif case["kind"] == "linear":
            found.append(_values64(layer["x"])[0] @ _stored64(layer["codes"], layer["scales"], case["K"]).t())
        elif case["kind"] == "norm":
            r = _joined64(layer, layer["branch"].double())
            found.append({"stream": r, "y": _normed64(r, layer["weight"])})
        else:
            H, I = case["H"], case["I"]
            both = _values64(_normed64(layer["stream"].double(), layer["weight"]))[0] @ _stored64(layer["gu"], layer["gu_scales"], H).t()
            gate, up = both.split(I, dim=1)
            middle = _values64(gate * torch.sigmoid(gate) * up)[0]
            found.append(_joined64(layer, middle @ _stored64(layer["down"], layer["down_scales"], I).t()))
    return found
