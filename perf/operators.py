"""Cases of the eight-bit operators: the int8 serving path and the 8-bit activation checkpoints of training.

``norm``    residual add + root-mean-square norm, its rows written in int8 with one scale each
``linear``  int8 matrix product with a scale per token and per output channel (bias, GELU), from int8 rows
            or from 16-bit activations that are quantised on the way
``gelu``    GELU that leaves an 8-bit checkpoint of its input (forward), and GELU's backward from it
``wgrad``   a Linear's weight gradient from the 8-bit checkpoint of its input

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, through
``double_attention_b200``.  An int8 or checkpointed tensor is returned as the values it stands for.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "none": 0}
BLOCK = 32  # columns of a checkpoint that share one exponent


def listed() -> list[dict]:
    return [
        # decoding one token: the residual of a 512-wide model, an attention branch in bf16
        {"name": "norm token", "op": "norm", "rows": 1, "dim": 512, "x": "fp32", "branch": "bf16"},
        # a whole language-model batch, 256 sequences of 1024 tokens, fp32 residual
        {"name": "norm lm batch", "op": "norm", "rows": 262144, "dim": 512, "x": "fp32", "branch": "bf16"},
        # a half-precision residual stream without a branch to add (a first norm), an uneven width and row count
        {"name": "norm uneven fp16", "op": "norm", "rows": 5003, "dim": 1000, "x": "fp16", "branch": "none"},
        # decoding one token through the feed-forward's first layer, fed by the norm's int8 rows
        {"name": "linear token", "op": "linear", "rows": 1, "inner": 512, "outer": 1536, "x": "int8", "bias": True,
         "gelu": True, "out": "bf16"},
        # decoding a batch of 24 sequences through a wide layer, its activations quantised on the way
        {"name": "linear decode batch", "op": "linear", "rows": 24, "inner": 4096, "outer": 4096, "x": "bf16",
         "bias": False, "gelu": False, "out": "bf16"},
        # prefill of 16 sequences of 2048 tokens through the feed-forward's first layer
        {"name": "linear prefill", "op": "linear", "rows": 32768, "inner": 512, "outer": 1536, "x": "int8",
         "bias": True, "gelu": True, "out": "bf16"},
        # a large square layer over a long batch, activations quantised on the way
        {"name": "linear large", "op": "linear", "rows": 8192, "inner": 4096, "outer": 4096, "x": "bf16",
         "bias": False, "gelu": False, "out": "bf16"},
        # training step of the language model: the feed-forward's hidden layer, forward
        {"name": "gelu forward", "op": "gelu", "rows": 262144, "dim": 1536, "dtype": "bf16", "backward": False},
        # the same layer's backward from the checkpoint
        {"name": "gelu backward", "op": "gelu", "rows": 262144, "dim": 1536, "dtype": "bf16", "backward": True},
        # a short fp16 batch whose width ends inside a block of the checkpoint
        {"name": "gelu backward uneven", "op": "gelu", "rows": 1025, "dim": 1000, "dtype": "fp16", "backward": True},
        # training step of the language model: weight gradient of the feed-forward's first layer, fp32 parameters
        {"name": "wgrad lm step", "op": "wgrad", "rows": 262144, "outer": 1536, "inner": 512, "dtype": "bf16",
         "out": "fp32"},
        # a small uneven layer and batch with 16-bit parameters
        {"name": "wgrad uneven", "op": "wgrad", "rows": 5001, "outer": 392, "inner": 1000, "dtype": "fp16",
         "out": "fp16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(max(n, lo), hi)
    return n - 1 if n == 3072 else n


def draw(rng) -> dict:
    op = rng.choice(["norm", "linear", "gelu", "wgrad"])
    if op == "norm":
        dim = _log(rng, 64, 8192)
        return {"op": op, "rows": min(_log(rng, 1, 262144), 134_000_000 // dim), "dim": dim,
                "x": rng.choice(["fp32", "bf16", "fp16"]), "branch": rng.choice(["bf16", "fp16", "fp32", "none"])}
    if op == "linear":
        inner, outer = _log(rng, 64, 4096), _log(rng, 64, 4096)
        return {"op": op, "rows": min(_log(rng, 1, 65536), 137_000_000_000 // (inner * outer)), "inner": inner,
                "outer": outer, "x": rng.choice(["int8", "bf16", "fp16"]), "bias": rng.random() < 0.5,
                "gelu": rng.random() < 0.5, "out": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "gelu":
        dim = _log(rng, 64, 8192)
        return {"op": op, "rows": min(_log(rng, 1, 262144), 402_000_000 // dim), "dim": dim,
                "dtype": rng.choice(["bf16", "fp16"]), "backward": rng.random() < 0.5}
    inner, outer = _log(rng, 64, 4096), _log(rng, 64, 4096)
    dtype = rng.choice(["bf16", "fp16"])
    return {"op": op, "rows": min(_log(rng, 64, 262144), 200_000_000_000 // (inner * outer)), "outer": outer,
            "inner": inner, "dtype": dtype, "out": rng.choice(["fp32", dtype])}


# ----------------------------------------------------------------------------- inputs
def _activations(g: torch.Generator, rows: int, dim: int, scale: float = 1.0) -> torch.Tensor:
    """Rows as a residual stream holds them: unit normal with a few channels several times larger."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    gain = 1.0 + 5.0 * (torch.rand(dim, generator=g, device="cuda") < 0.02)
    return x.mul_(gain).mul_(scale)


def _padded(values: torch.Tensor, to: int) -> torch.Tensor:
    """The same values with their row stride rounded up to ``to`` elements, as the quantisers lay rows out."""
    rows, dim = values.shape
    pad = -(-dim // to) * to
    out = torch.zeros(rows, pad, dtype=values.dtype, device=values.device)
    out[:, :dim] = values
    return out[:, :dim]


def _rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    amax = x.abs().amax(dim=1)
    q = torch.round(x * (torch.full_like(amax, 127.0) / amax)[:, None]).to(torch.int8)
    return _padded(q, 16), amax / 127.0


def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for whole numbers e in [-126, 127], from the number's exponent field."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x: torch.Tensor, lowest: int, highest: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Checkpoint of ``x`` [rows, dim]: int8 [rows, blocks * 32] and the blocks' exponents int8 [rows, blocks]."""
    rows, dim = x.shape
    blocks = -(-dim // BLOCK)
    if blocks * BLOCK != dim:
        x = torch.cat((x, x.new_zeros(rows, blocks * BLOCK - dim)), dim=1)
    x = x.float().view(rows, blocks, BLOCK)
    mantissa, exponent = torch.frexp(x.abs().amax(dim=2))  # in [0.5, 1) times 2^exponent
    e = exponent - 7 + (mantissa > 127.0 / 128.0).to(exponent.dtype)
    e = torch.where(mantissa == 0, torch.full_like(e, lowest), e).clamp_(lowest, highest)
    q = torch.round(x * _power(-e)[..., None]).clamp_(-127, 127)
    return q.view(rows, blocks * BLOCK).to(torch.int8), e.to(torch.int8)


def _range(dtype: str) -> tuple[int, int]:
    return (-24, 9) if dtype == "fp16" else (-126, 121)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    s: dict = {"case": case}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s["x"] = _activations(g, rows, dim, 2.0).to(DTYPES[case["x"]])
        s["branch"] = None
        if case["branch"] != "none":
            s["branch"] = torch.randn(rows, dim, generator=g, device="cuda").to(DTYPES[case["branch"]])
        s["norm"] = torch.nn.RMSNorm(dim, eps=1e-6, device="cuda")
        s["norm"].weight.data = 1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")
        s["norm"].requires_grad_(False)
    elif case["op"] == "linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        w = torch.randn(outer, inner, generator=g, device="cuda") * inner**-0.5
        s["w"] = _rows_int8(w)  # laid out once, when the model is loaded
        x = _activations(g, rows, inner)
        s["x"] = _rows_int8(x) if case["x"] == "int8" else x.to(DTYPES[case["x"]])
        s["bias"] = 0.1 * torch.randn(outer, generator=g, device="cuda") if case["bias"] else None
    elif case["op"] == "gelu":
        rows, dim = case["rows"], case["dim"]
        z = (1.5 * torch.randn(rows, dim, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
        if case["backward"]:
            s["dh"] = (1e-2 * torch.randn(rows, dim, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
            s["checkpoint"] = _blocks(z, *_range(case["dtype"]))
        else:
            s["z"] = z
    else:
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        x = _activations(g, rows, inner).to(DTYPES[case["dtype"]])
        s["checkpoint"] = _blocks(x, *_range(case["dtype"]))
        s["dy"] = (1e-2 * torch.randn(rows, outer, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    return s


# ----------------------------------------------------------------------------- plain form
def _gelu(z: torch.Tensor) -> torch.Tensor:
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _restored(checkpoint: tuple[torch.Tensor, torch.Tensor], dim: int) -> torch.Tensor:
    q, e = checkpoint
    x = q.float().view(q.shape[0], -1, BLOCK) * _power(e)[..., None]
    return x.reshape(q.shape[0], -1)[:, :dim]


def _plain(s: dict):
    case = s["case"]
    if case["op"] == "norm":
        x_out = s["x"]
        if s["branch"] is not None:
            x_out = (s["x"].float() + s["branch"].float()).to(s["x"].dtype)
        r = x_out.float()
        v = r * s["norm"].weight
        amax = v.abs().amax(dim=1)
        rstd = 1.0 / torch.sqrt((r * r).mean(dim=1) + s["norm"].eps)
        q = torch.round(v * (torch.full_like(amax, 127.0) / amax)[:, None])
        return {"x_out": x_out, "y": (q * (amax * rstd / 127.0)[:, None]).to(torch.bfloat16)}
    if case["op"] == "linear":
        xq, xs = s["x"] if case["x"] == "int8" else _rows_int8(s["x"].float())
        wq, ws = s["w"]
        y = (xq.float() @ wq.float().t()) * xs[:, None] * ws[None, :]
        if s["bias"] is not None:
            y = y + s["bias"]
        if case["gelu"]:
            y = _gelu(y)
        return {"y": y.to(DTYPES[case["out"]])}
    if case["op"] == "gelu" and not case["backward"]:
        h = _gelu(s["z"].float()).to(s["z"].dtype)
        kept = _blocks(s["z"], *_range(case["dtype"]))
        return {"h": h, "z": _restored(kept, case["dim"]).to(s["z"].dtype)}
    if case["op"] == "gelu":
        z = _restored(s["checkpoint"], case["dim"])
        slope = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        return {"dz": (s["dh"].float() * slope).to(s["dh"].dtype), "h": _gelu(z).to(s["dh"].dtype)}
    x = _restored(s["checkpoint"], case["inner"])
    return {"dw": (s["dy"].float().t() @ x).to(DTYPES[case["out"]])}


# ----------------------------------------------------------------------------- the framework's operators
def _framework(s: dict):
    import double_attention_b200 as da

    case = s["case"]
    if case["op"] == "norm":
        if s["branch"] is None:
            x_out, y = s["x"], da.rmsnorm_int8(s["x"], s["norm"])
        else:
            x_out, y = da.add_rmsnorm_int8(s["x"], s["branch"], s["norm"])
        return {"x_out": x_out, "y": y.dequantize(torch.bfloat16)}
    if case["op"] == "linear":
        x = da.Int8Rows(*s["x"]) if case["x"] == "int8" else da.quantize_int8(s["x"])
        return {"y": da.int8_linear(x, da.Int8Rows(*s["w"]), s["bias"], gelu=case["gelu"], dtype=DTYPES[case["out"]])}
    if case["op"] == "gelu" and not case["backward"]:
        h, kept = da.gelu_checkpoint8(s["z"])
        return {"h": h, "z": kept.restore()}
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "gelu":
        kept = da.Checkpoint8(*s["checkpoint"], shape=(case["rows"], case["dim"]), dtype=dtype)
        dz, h = da.gelu_checkpoint8_backward(s["dh"], kept)
        return {"dz": dz, "h": h}
    kept = da.Checkpoint8(*s["checkpoint"], shape=(case["rows"], case["inner"]), dtype=dtype)
    return {"dw": da.weight_grad_checkpoint8(s["dy"], kept, dtype=DTYPES[case["out"]])}


def run(state: dict):
    return _framework(state) if own else _plain(state)


# ----------------------------------------------------------------------------- work and definition
def work(case: dict) -> dict:
    rows = case["rows"]
    if case["op"] == "norm":
        size = BYTES[case["x"]]
        # without a branch the residual is not written again; the rows come back as bf16 values
        each = 2 * size + BYTES[case["branch"]] if case["branch"] != "none" else size
        n = rows * case["dim"]
        return {"bytes": n * (each + 2), "flops": 8 * n}
    if case["op"] == "linear":
        k, n = case["inner"], case["outer"]
        read = rows * k * (1 if case["x"] == "int8" else 2) + n * k + 4 * n + (4 * n if case["bias"] else 0)
        return {"bytes": read + rows * n * BYTES[case["out"]], "flops": 2 * rows * n * k}
    if case["op"] == "gelu":
        n = rows * case["dim"]
        kept = n + n // BLOCK
        if case["backward"]:
            return {"bytes": 2 * n + kept + 4 * n, "flops": 20 * n}
        return {"bytes": 2 * n + 2 * n + 2 * n, "flops": 14 * n}  # the checkpoint comes back as 16-bit values
    k, n = case["inner"], case["outer"]
    return {"bytes": rows * (2 * n + k + k // BLOCK) + n * k * BYTES[case["out"]], "flops": 2 * rows * n * k}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f64 = torch.float64
    half = torch.tensor(0.5, dtype=f64, device="cuda")

    def phi(t):  # standard normal distribution function
        return half * torch.special.erfc(-t * torch.sqrt(half))

    if case["op"] == "norm":
        if case["branch"] == "none":
            x_out = s["x"]
            r = x_out.to(f64)
        else:
            r = s["x"].to(f64) + s["branch"].to(f64)
            x_out = r
            if case["x"] != "fp32":  # the norm reads the residual as it is stored
                r = r.to(s["x"].dtype).to(f64)
        y = r * s["norm"].weight.to(f64) * torch.rsqrt(r.square().sum(1, keepdim=True) / case["dim"] + s["norm"].eps)
        step = y.abs().max(dim=1, keepdim=True).values / 127
        return {"x_out": x_out.to(f64), "y": (y / step).round() * step}
    if case["op"] == "linear":
        if case["x"] == "int8":
            x = s["x"][0].to(f64) * s["x"][1].to(f64).unsqueeze(1)
        else:
            x = s["x"].to(f64)
            step = x.abs().max(dim=1, keepdim=True).values / 127
            x = (x / step).round() * step
        y = torch.einsum("tk,nk->tn", x, s["w"][0].to(f64) * s["w"][1].to(f64).unsqueeze(1))
        if s["bias"] is not None:
            y = y + s["bias"].to(f64).unsqueeze(0)
        return {"y": y * phi(y) if case["gelu"] else y}

    def stored(values, exponents, columns):
        scale = torch.exp2(exponents.to(f64)).repeat_interleave(BLOCK, dim=1)
        return (values.to(f64) * scale)[:, :columns]

    if case["op"] == "gelu" and not case["backward"]:
        z = s["z"].to(f64)
        h = z * phi(z)
        rows, dim = z.shape
        z = torch.nn.functional.pad(z, (0, -dim % BLOCK)).unflatten(1, (-1, BLOCK))
        lowest, highest = _range(case["dtype"])
        # the smallest power of two whose 127-fold covers the block (16-bit values lie further apart than 1e-9)
        e = torch.ceil(torch.log2(z.abs().amax(dim=2, keepdim=True) / 127) - 1e-9).nan_to_num(neginf=lowest)
        unit = torch.exp2(e.clamp(lowest, highest))
        return {"h": h, "z": ((z / unit).round().clamp(-127, 127) * unit).flatten(1)[:, :dim]}
    if case["op"] == "gelu":
        z = stored(*s["checkpoint"], case["dim"])
        density = torch.exp(-half * z.square()) / math.sqrt(2 * math.pi)
        return {"dz": s["dh"].to(f64) * (phi(z) + z * density), "h": z * phi(z)}
    x = stored(*s["checkpoint"], case["inner"])
    return {"dw": torch.einsum("tn,tk->nk", s["dy"].to(f64), x)}
