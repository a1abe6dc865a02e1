"""The 8-bit activation operators (include/bm_cuda_backend.h, "8-bit rows and their product") as cases to be timed and compared:
rows to 8 bits, RMSNorm with the residual's addition, SwiGLU, and the integer product with a scale per token and per channel.
Codes are returned as the values they stand for (code * scale, in bf16)."""
import math
import os

import torch

own = False

EPS = 1e-5
TINY = 2.0 ** -126     # a row whose scale would be below the smallest normal number is stored as zeros
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # attention output of one decode step of 64 sequences of the 360M configuration (15 heads x 64), before the O product
        {"name": "rows-decode", "op": "rows", "dtype": "f32", "rows": 64, "cols": 960, "pad": 0},
        # the same at prefill: 64 prompts of 512 tokens
        {"name": "rows-prefill", "op": "rows", "dtype": "f32", "rows": 32768, "cols": 960, "pad": 0},
        # single-token decode: fp32 residual stream, the branch's product in bf16
        {"name": "norm-decode-1", "op": "norm", "dtype": "f32", "add": "bf16", "rows": 1, "cols": 960, "pad": 0},
        # prefill of the 360M configuration
        {"name": "norm-prefill", "op": "norm", "dtype": "f32", "add": "bf16", "rows": 32768, "cols": 960, "pad": 0},
        # a wider model's bf16 stream with an odd width and a ragged number of rows
        {"name": "norm-odd", "op": "norm", "dtype": "bf16", "add": "bf16", "rows": 1021, "cols": 4099, "pad": 0},
        # gate | up of 64 sequences, and of a prefill
        {"name": "swiglu-decode", "op": "swiglu", "dtype": "bf16", "rows": 64, "cols": 2560},
        {"name": "swiglu-prefill", "op": "swiglu", "dtype": "bf16", "rows": 32768, "cols": 2560},
        # QKV of one token
        {"name": "product-decode-1", "op": "product", "dtype": "f32", "residual": False, "rows": 1, "cols": 960, "outs": 1600},
        # gate | up and down (with the residual) of 64 sequences
        {"name": "product-decode-gu", "op": "product", "dtype": "bf16", "residual": False, "rows": 64, "cols": 960, "outs": 5120},
        {"name": "product-decode-down", "op": "product", "dtype": "f32", "residual": True, "rows": 64, "cols": 2560, "outs": 960},
        # gate | up of a prefill: short reduction, the output's bytes weigh most
        {"name": "product-prefill", "op": "product", "dtype": "bf16", "residual": False, "rows": 32768, "cols": 960, "outs": 5120},
        # a wider model's square projection with a ragged number of tokens: long reduction
        {"name": "product-wide", "op": "product", "dtype": "f32", "residual": False, "rows": 4099, "cols": 4096, "outs": 4096},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rows", "norm", "swiglu", "product", "product"))
    c = {"op": op, "dtype": rng.choice(("f32", "bf16")), "rows": _spread(rng, 1, 32768)}
    if op == "product":
        c["cols"] = 16 * _spread(rng, 4, 512)
        c["outs"] = _spread(rng, 16, 8192)
        c["residual"] = rng.random() < 0.3
        most = min(32768 * 5120 * 960 // (c["cols"] * c["outs"]), 32768 * 2560 // c["outs"])
    else:
        c["cols"] = _spread(rng, 16, 16384)
        most = 32768 * 960 // c["cols"]
        if op == "norm":
            c["add"] = rng.choice(("none", "f32", "bf16"))
        if op != "swiglu":
            c["pad"] = rng.choice((0, 0, 1, 8, 64))   # elements between the end of a row and the next one's start
    c["rows"] = max(1, min(c["rows"], most))
    return c


def _rows_of(g, rows, cols, dtype, pad=0):
    """Activations: normal values, every 64th channel twenty times the others, as in a trained model's residual stream."""
    x = torch.randn(rows, cols + pad, generator=g, device="cuda")
    x[:, 5::64] *= 20.0
    return x.to(dtype)[:, :cols]


def _codes(g, rows, cols, std):
    x = torch.randn(rows, cols, generator=g, device="cuda") * std
    scale = x.abs().amax(1) / 127
    return torch.round(x / scale[:, None]).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n, c, op, dt = case["rows"], case["cols"], case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dt}
    if op == "product":
        s["q"], s["scale"] = _codes(g, n, c, 1.0)
        s["w"], s["wscale"] = _codes(g, case["outs"], c, 0.02)
        s["residual"] = torch.randn(n, case["outs"], generator=g, device="cuda").to(dt) if case["residual"] else None
        s["out"] = torch.empty(n, case["outs"], dtype=dt, device="cuda")
        return s
    if op == "swiglu":
        s["x"] = torch.randn(n, 2 * c, generator=g, device="cuda").mul_(1.5).to(dt)     # [gate | up]
    else:
        s["x"] = _rows_of(g, n, c, dt, case["pad"])
    if op == "norm":
        s["w"] = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
        s["add"] = None if case["add"] == "none" else (0.5 * torch.randn(n, c, generator=g, device="cuda")).to(DTYPES[case["add"]])
        s["sum"] = torch.empty(n, c, dtype=dt, device="cuda")
    s["codes"] = torch.empty(n, c, dtype=torch.int8, device="cuda")
    s["scales"] = torch.empty(n, dtype=torch.float32, device="cuda")
    s["values"] = torch.empty(n, c, dtype=torch.bfloat16, device="cuda")
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- plain form ----------------------------------------------------------------------------------------------------------
def _to_8_bits(v):
    scale = v.abs().amax(1, keepdim=True) / 127
    scale = torch.where(scale < TINY, torch.zeros_like(scale), scale)
    codes = torch.where(scale == 0, torch.zeros_like(v), torch.round(v * (1 / scale)))
    return {"values": (codes * scale).to(torch.bfloat16), "scale": scale[:, 0]}


def _run_plain(s):
    op, dt = s["op"], s["dtype"]
    if op == "product":
        out = (s["q"].float() @ s["w"].float().t()) * (s["scale"][:, None] * s["wscale"])
        return (out if s["residual"] is None else out + s["residual"].float()).to(dt)
    x = s["x"].float()
    if op == "rows":
        return _to_8_bits(x)
    if op == "swiglu":
        gate, up = x.chunk(2, 1)
        return _to_8_bits(gate / (1 + torch.exp(-gate)) * up)
    if s["add"] is not None:
        x = x + s["add"].float()
    out = _to_8_bits(x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["w"])
    if s["add"] is not None:
        out["sum"] = x.to(dt)
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------------------
_backend = None


def _lib():
    """The framework's context. Torch's own work goes to the context's stream from here on, so that both are ordered."""
    global _backend
    if _backend is None:
        import sys
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bare.metal_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import bmapi
        import bmcapi
        _backend = bmcapi.Backend(bmapi.load_product())
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.ExternalStream(_backend.lib.bmc_stream(_backend.ctx)))
    return _backend.lib, _backend.ctx


def _checked(rc):
    if rc:
        raise RuntimeError("the call was refused: %d" % rc)


def _run_own(s):
    lib, ctx = _lib()
    op, f32 = s["op"], torch.float32
    bf = 0 if s["dtype"] == f32 else 1
    if op == "product":
        (n, c), oc, r = s["q"].shape, s["w"].shape[0], s["residual"]
        _checked(lib.bmc_matmul_q8(ctx, bf, s["out"].data_ptr(), oc, s["q"].data_ptr(), c, s["scale"].data_ptr(), s["w"].data_ptr(),
                                   s["wscale"].data_ptr(), None if r is None else r.data_ptr(), oc, n, c, oc))
        return s["out"]
    x, codes, scales = s["x"], s["codes"], s["scales"]
    n, c = codes.shape
    if op == "rows":
        _checked(lib.bmc_quantize_rows_q8(ctx, bf, codes.data_ptr(), c, scales.data_ptr(), x.data_ptr(), x.stride(0), n, c))
    elif op == "swiglu":
        at = x.data_ptr()
        _checked(lib.bmc_swiglu_q8(ctx, bf, codes.data_ptr(), c, scales.data_ptr(), at, at + c * x.element_size(), 2 * c, n, c))
    else:
        a = s["add"]
        _checked(lib.bmc_rmsnorm_q8(ctx, bf, codes.data_ptr(), c, scales.data_ptr(), None if a is None else s["sum"].data_ptr(), c,
                                    x.data_ptr(), x.stride(0), 1 if a is not None and a.dtype != f32 else 0,
                                    None if a is None else a.data_ptr(), c, s["w"].data_ptr(), n, c, EPS))
    out = {"values": torch.mul(codes, scales[:, None], out=s["values"]), "scale": scales}
    if op == "norm" and s["add"] is not None:
        out["sum"] = s["sum"]
    return out


# ---- what one pass cannot do without, and the definition in 64 bits ---------------------------------------------------------
def work(case):
    n, c, e = case["rows"], case["cols"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "product":
        oc = case["outs"]
        return {"bytes": n * c + oc * c + 4 * (n + oc) + n * oc * e * (2 if case["residual"] else 1), "flops": 2 * n * c * oc}
    made = n * c + 4 * n
    if case["op"] == "rows":
        return {"bytes": n * c * e + made, "flops": 3 * n * c}
    if case["op"] == "swiglu":
        return {"bytes": 2 * n * c * e + made, "flops": 8 * n * c}
    a = {"none": 0, "f32": 4 + e, "bf16": 2 + e}[case["add"]]
    return {"bytes": n * c * (e + a) + 4 * c + made, "flops": 8 * n * c}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "product":
        total = torch.einsum("mk,nk->mn", s["q"].double(), s["w"].double())
        total.mul_(s["scale"].double()[:, None]).mul_(s["wscale"].double())
        return total if s["residual"] is None else total.add_(s["residual"].double())
    v, plus = s["x"].double(), None
    if s["op"] == "swiglu":
        half = v.shape[1] // 2
        v = v[:, :half] * torch.sigmoid(v[:, :half]) * v[:, half:]
    elif s["op"] == "norm":
        if s["add"] is not None:
            v = plus = v.add(s["add"].double())
        v = s["w"].double() * v / torch.sqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS)
    top = v.abs().max(1).values
    step = (top / 127)[:, None]
    out = {"values": (v / step).nan_to_num(0.0).round() * step, "scale": step[:, 0]}
    if plus is not None:
        out["sum"] = plus
    return out
