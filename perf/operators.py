"""The 8-bit row operators: real calls over their range, their plain forms, and their values in 64 bits.

A tensor in 8-bit rows is an int8 matrix ``q`` whose rows are ``ld`` bytes apart (a multiple of 16) and one fp32
scale per row; it stands for ``q * scale``. Five operators work on it: writing and reading it (``rows``), RMSNorm with
the residual's addition whose output is 8-bit rows (``norm``), the matrix product of two of them (``linear``), and the
backward passes of a linear layer and of the norm whose saved input is 8-bit rows (``linear_backward``,
``norm_backward``).
"""
import math

import torch

own = False

TINY = 2.0 ** -126   # smallest scale of a row
EPS = 1e-5


def listed():
    return [
        # one token of a decoding step enters a layer: latency is all that counts
        {"name": "norm_token", "op": "norm", "rows": 1, "features": 4096, "dtype": "bf16", "keep": False},
        # a training step's norm over a long batch: the 8-bit output and the 8-bit checkpoint of its input in one pass
        {"name": "norm_train", "op": "norm", "rows": 16384, "features": 4096, "dtype": "bf16", "keep": True},
        # one token through a square projection: the weights are read once
        {"name": "linear_token", "op": "linear", "rows": 1, "features": 4096, "out": 4096, "act": "none", "bias": False, "dtype": "bf16"},
        # odd everything, fp32 result
        {"name": "linear_ragged", "op": "linear", "rows": 333, "features": 1111, "out": 1001, "act": "relu", "bias": True, "dtype": "f32"},
        # the sentence encoder's first feed-forward product: 256 sentences of 128 tokens, 384 -> 1536 with GELU
        {"name": "linear_encoder", "op": "linear", "rows": 32768, "features": 384, "out": 1536, "act": "gelu", "bias": True, "dtype": "bf16"},
        # a prompt through a large projection: the tensor cores' rate counts
        {"name": "linear_large", "op": "linear", "rows": 8192, "features": 8192, "out": 8192, "act": "none", "bias": True, "dtype": "bf16"},
        # gradients of the encoder's first feed-forward product: a small weight under many tokens
        {"name": "linear_backward_encoder", "op": "linear_backward", "rows": 16384, "features": 384, "out": 1536},
        # gradients of a large projection
        {"name": "linear_backward_large", "op": "linear_backward", "rows": 16384, "features": 4096, "out": 4096},
        # odd width, fp32
        {"name": "norm_backward_ragged", "op": "norm_backward", "rows": 2049, "features": 1001, "dtype": "f32", "grad_h": False},
        # the training step's norm, with the residual stream's gradient added
        {"name": "norm_backward_train", "op": "norm_backward", "rows": 16384, "features": 4096, "dtype": "bf16", "grad_h": True},
        # a short checkpoint in fp32, odd width
        {"name": "rows_ragged", "op": "rows", "rows": 777, "features": 515, "dtype": "f32"},
        # a long batch's checkpoint: written and read back
        {"name": "rows_train", "op": "rows", "rows": 16384, "features": 4096, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]; half of them multiples of 16 where there is room."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 32 and rng.random() < 0.5:
        v = v // 16 * 16
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "linear_backward", "norm_backward", "rows"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("norm", "norm_backward", "rows"):
        features = _spread(rng, 8, 12000)
        rows = _spread(rng, 1, min(20000, (1 << 26) // features))
        case = {"op": op, "rows": rows, "features": features, "dtype": dtype}
        if op == "norm":
            case["keep"] = rng.random() < 0.5
        if op == "norm_backward":
            case["grad_h"] = rng.random() < 0.5
        return case
    features, out = _spread(rng, 16, 12000), _spread(rng, 8, 12000)
    most = (1 << 37) if op == "linear_backward" else (1 << 38)
    rows = _spread(rng, 1, max(1, min(40000, most // (features * out))))
    if op == "linear_backward":
        return {"op": op, "rows": rows, "features": features, "out": out}
    return {"op": op, "rows": rows, "features": features, "out": out, "act": rng.choice(["none", "gelu", "silu", "relu"]),
            "bias": rng.random() < 0.5, "dtype": dtype}


# ------------------------------------------------------------------------------------------------- inputs
def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _activations(g, rows, features):
    """Hidden states as a transformer has them: tokens of different size, a few channels far larger than the rest."""
    d = _device()
    x = torch.randn(rows, features, generator=g, device=d)
    x *= 0.5 + torch.rand(rows, 1, generator=g, device=d)
    loud = torch.rand(features, generator=g, device=d) < 0.01
    return x * torch.where(loud, 6.0, 1.0)


def _pack(x):
    """fp32 rows as 8-bit rows: (q with rows of a multiple of 16 bytes, scale)."""
    rows, features = x.shape
    scale = (x.abs().amax(1) / 127).clamp_min(TINY)
    q = torch.zeros(rows, (features + 15) // 16 * 16, dtype=torch.int8, device=x.device)
    q[:, :features] = torch.round(x / scale[:, None]).to(torch.int8)
    return q, scale


def prepare(case, seed):
    d = _device()
    g = torch.Generator(device=d)
    g.manual_seed(int(seed))
    rows, features, op = case["rows"], case["features"], case["op"]
    s = {"case": case}
    if op in ("norm", "rows"):
        s["x"] = _activations(g, rows, features).to(_dtype(case["dtype"]))
    if op == "norm":
        s["residual"] = torch.randn(rows, features, generator=g, device=d).to(_dtype(case["dtype"]))
        s["gamma"] = 1 + 0.2 * torch.randn(features, generator=g, device=d)
    if op == "norm_backward":
        h = _activations(g, rows, features)
        s["q"], s["scale"] = _pack(h)
        s["rstd"] = torch.rsqrt((h * h).mean(1) + EPS)
        s["gamma"] = 1 + 0.2 * torch.randn(features, generator=g, device=d)
        s["grad"] = (0.01 * torch.randn(rows, features, generator=g, device=d)).to(_dtype(case["dtype"]))
        s["grad_h"] = (0.01 * torch.randn(rows, features, generator=g, device=d)).to(_dtype(case["dtype"])) if case["grad_h"] else None
    if op in ("linear", "linear_backward"):
        s["q"], s["scale"] = _pack(_activations(g, rows, features))
        w = torch.randn(case["out"], features, generator=g, device=d) * features ** -0.5
    if op == "linear":
        s["wq"], s["wscale"] = _pack(w)
        s["bias"] = 0.1 * torch.randn(case["out"], generator=g, device=d) if case["bias"] else None
    if op == "linear_backward":
        s["w"] = w.to(torch.bfloat16)
        s["grad"] = (0.01 * torch.randn(rows, case["out"], generator=g, device=d)).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _quantize_plain(y):
    """8-bit rows of fp32 values: what they stand for, in bf16, and the scales."""
    scale = (y.abs().amax(1) / 127).clamp_min(TINY)
    q = torch.round(y / scale[:, None])
    return (q * scale[:, None]).to(torch.bfloat16), scale


def _activation_plain(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "relu":
        return y.clamp_min(0)
    return y


def _plain(s):
    case = s["case"]
    op, features = case["op"], case["features"]
    if op == "rows":
        values, scale = _quantize_plain(s["x"].float())
        return {"values": values, "scale": scale}
    if op == "norm":
        h = s["x"].float() + s["residual"].float()
        rstd = torch.rsqrt((h * h).mean(1) + EPS)
        values, scale = _quantize_plain(h * rstd[:, None] * s["gamma"])
        out = {"h": h.to(s["x"].dtype), "values": values, "scale": scale}
        if case["keep"]:
            out["h_values"], out["h_scale"] = _quantize_plain(h)
            out["rstd"] = rstd
        return out
    x = s["q"][:, :features].float()
    if op == "linear":
        y = x @ s["wq"][:, :features].float().T
        y = y * s["scale"][:, None] * s["wscale"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return _activation_plain(y, case["act"]).to(_dtype(case["dtype"]))
    x = x * s["scale"][:, None]
    grad = s["grad"].float()
    if op == "linear_backward":
        return {"grad_input": (grad @ s["w"].float()).to(torch.bfloat16), "grad_weight": (grad.T @ x).to(torch.bfloat16),
                "grad_bias": grad.sum(0)}
    normed = x * s["rstd"][:, None]
    scaled = grad * s["gamma"]
    dh = s["rstd"][:, None] * (scaled - normed * (scaled * normed).mean(1, keepdim=True))
    if s["grad_h"] is not None:
        dh = dh + s["grad_h"].float()
    return {"grad_input": dh.to(s["grad"].dtype), "grad_gamma": (grad * normed).sum(0)}


# ------------------------------------------------------------------------------------------------- the framework's calls
_backend = None


def _fnn():
    """The handle that a program keeps, working on torch's stream (the legacy default stream's handle is 1)."""
    global _backend
    if _backend is None:
        import grilly_b200

        _backend = grilly_b200.Compute(precision="bf16")
    stream = torch.cuda.current_stream().cuda_stream or 1
    if getattr(_backend, "_torch_stream", None) != stream:
        _backend.device.set_stream(stream)
        _backend._torch_stream = stream
    return _backend.fnn


_NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int8: "i8"}


def _view(t):
    from grilly_b200 import DeviceTensor

    return None if t is None else DeviceTensor(_backend.device, t.data_ptr(), t.shape, _NAMES[t.dtype], owned=False)


def _rows8(q, scale, features):
    from grilly_b200 import Rows8

    return Rows8(_view(q), _view(scale), (q.shape[0], features))


def _new_rows8(rows, features):
    """Room for 8-bit rows in torch's memory: (q, scale, the framework's view of the two)."""
    q = torch.empty(rows, (features + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    return scale, _rows8(q, scale, features), q


def _own(s):
    case, fnn = s["case"], _fnn()
    op, rows, features = case["op"], case["rows"], case["features"]
    if op in ("rows", "norm"):
        scale, y8, _q = _new_rows8(rows, features)
        values = torch.empty(rows, features, dtype=torch.bfloat16, device="cuda")
    if op == "rows":
        fnn.quantize_rows(_view(s["x"]), out=y8)
        fnn.dequantize_rows(y8, out=_view(values))
        return {"values": values, "scale": scale}
    if op == "norm":
        h = torch.empty_like(s["x"])
        out = {"h": h, "values": values, "scale": scale}
        h8 = rstd = None
        if case["keep"]:
            out["h_scale"], h8, _hq = _new_rows8(rows, features)
            out["h_values"] = torch.empty_like(values)
            out["rstd"] = rstd = torch.empty(rows, device="cuda")
        fnn.rmsnorm_residual_q8(_view(s["x"]), _view(s["residual"]), _view(s["gamma"]), eps=EPS, keep=case["keep"],
                                out=(y8, _view(h), h8, _view(rstd)))
        fnn.dequantize_rows(y8, out=_view(values))
        if case["keep"]:
            fnn.dequantize_rows(h8, out=_view(out["h_values"]))
        return out
    x8 = _rows8(s["q"], s["scale"], features)
    if op == "linear":
        y = torch.empty(rows, case["out"], dtype=_dtype(case["dtype"]), device="cuda")
        fnn.linear_q8(x8, _rows8(s["wq"], s["wscale"], features), _view(s["bias"]), act=case["act"], out=_view(y))
        return y
    if op == "linear_backward":
        gx = torch.empty(rows, features, dtype=torch.bfloat16, device="cuda")
        gw = torch.empty(case["out"], features, dtype=torch.bfloat16, device="cuda")
        gb = torch.empty(case["out"], device="cuda")
        fnn.linear_backward_q8(_view(s["grad"]), x8, _view(s["w"]), out=(_view(gx), _view(gw), _view(gb)))
        return {"grad_input": gx, "grad_weight": gw, "grad_bias": gb}
    gx = torch.empty_like(s["grad"])
    gg = torch.empty(features, device="cuda")
    fnn.rmsnorm_backward_q8(_view(s["grad"]), x8, _view(s["rstd"]), _view(s["gamma"]), grad_residual=_view(s["grad_h"]),
                            out=(_view(gx), _view(gg)))
    return {"grad_input": gx, "grad_gamma": gg}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, features, op = case["rows"], case["features"], case["op"]
    e = 2 if case.get("dtype", "bf16") == "bf16" else 4
    n = rows * features
    if op == "rows":
        return {"bytes": n * (e + 2) + 4 * rows, "flops": 4 * n}
    if op == "norm":
        keep = case["keep"]
        return {"bytes": n * (3 * e + 2 + (2 if keep else 0)) + 4 * features + rows * (12 if keep else 4), "flops": (14 if keep else 10) * n}
    if op == "norm_backward":
        return {"bytes": n * (2 * e + 1 + (e if case["grad_h"] else 0)) + 8 * features + 8 * rows, "flops": 10 * n}
    out = case["out"]
    if op == "linear":
        return {"bytes": n + out * features + 4 * (rows + 2 * out) + rows * out * e, "flops": 2 * n * out}
    return {"bytes": 2 * rows * out + n + 4 * rows + 2 * out * features + 2 * n + 2 * out * features + 4 * out, "flops": 4 * n * out}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: (v.double() if torch.is_tensor(v) and v.dtype != torch.int8 else v) for k, v in s.items()}
    op, k = case["op"], case["features"]

    def eight(t):
        step = torch.maximum(t.abs().max(dim=1, keepdim=True).values / 127, torch.tensor(TINY, dtype=torch.float64, device=t.device))
        return torch.round(t / step) * step, step[:, 0]

    if op in ("rows", "norm"):
        t = wide["x"]
        if op == "rows":
            values, scale = eight(t)
            return {"values": values, "scale": scale}
        t = t + wide["residual"]
        root = torch.sqrt(torch.linalg.vector_norm(t, dim=1) ** 2 / k + EPS)
        values, scale = eight(t / root[:, None] * wide["gamma"])
        out = {"h": t, "values": values, "scale": scale}
        if case["keep"]:
            out["h_values"], out["h_scale"] = eight(t)
            out["rstd"] = 1 / root
        return out
    x = s["q"][:, :k].double() * wide["scale"].unsqueeze(1)
    if op == "linear":
        y = torch.matmul(x, (s["wq"][:, :k].double() * wide["wscale"].unsqueeze(1)).t())
        if wide["bias"] is not None:
            y += wide["bias"]
        if case["act"] == "gelu":   # x sigmoid(2 u) is 0.5 x (1 + tanh u)
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "relu":
            y = torch.relu(y)
        return y
    grad = wide["grad"]
    if op == "linear_backward":
        return {"grad_input": torch.matmul(grad, wide["w"]), "grad_weight": torch.matmul(grad.t(), x), "grad_bias": grad.sum(dim=0)}
    normed = x * wide["rstd"].unsqueeze(1)
    dn = grad * wide["gamma"]
    dot = torch.einsum("rf,rf->r", dn, normed) / k
    dh = (dn - normed * dot.unsqueeze(1)) * wide["rstd"].unsqueeze(1)
    if wide["grad_h"] is not None:
        dh = dh + wide["grad_h"]
    return {"grad_input": dh, "grad_gamma": torch.einsum("rf,rf->f", grad, normed)}
