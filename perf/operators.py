"""Operators on 4-bit weights and 8-bit activations, for timing and comparison.

Kinds (sizes in brackets are the ranges that `draw` covers; group scales over 32, 64 or 128 columns):

  norm     root-mean-square norm of [1..8192] rows of [64..8192] columns, with or without the residual's
           addition, to 8-bit codes with a scale per group
  matmul   [1..2048] rows of 8-bit codes times [64..152000] x [64..8192] weights in 4 bits, with bias, residual
           or SwiGLU
  linear   both in one call: float rows, normed or not, to 8 bits, times 4-bit weights: [1..512] rows
  pack     float weights, [64..16384] x [64..8192], to 4 bits and scales, and back to the values they stand for

Weights in 4 bits lie in tiles of 16 rows x 128 columns: byte i + 8 p of lane 16 j + r of a tile holds the codes of
row r at columns 64 p + 8 j + i (low half) and 64 p + 32 + 8 j + i (high half), i < 8, j < 4, p < 2; tiles along a row of
tiles first; scales bf16 [tile row][tile][16 rows][128 / group]; rows and columns behind the matrix are zero.
Codes of activations are int8 [rows][columns up to a multiple of 128], their scales float32.
"""
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # one token's hidden state, before a projection
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 1024, "dtype": "f32", "group": 128, "residual": True},
        # a ragged handful of rows of an odd width
        {"name": "norm_odd", "kind": "norm", "rows": 37, "cols": 1283, "dtype": "bf16", "group": 64, "residual": False},
        # the rows of many prompts
        {"name": "norm_prompts", "kind": "norm", "rows": 8192, "cols": 5120, "dtype": "bf16", "group": 128, "residual": True},
        # one token through an output projection, added to the residual stream
        {"name": "matvec_projection", "kind": "matmul", "rows": 1, "n": 1024, "k": 2048, "dtype": "f32", "group": 128, "bias": False,
         "residual": True, "swiglu": False},
        # one token's logits over the emotion decoder's vocabulary: the largest matrix of a step
        {"name": "matvec_head", "kind": "matmul", "rows": 1, "n": 151936, "k": 1024, "dtype": "f32", "group": 128, "bias": False,
         "residual": False, "swiglu": False},
        # eight sequences' logits over the mel vocabulary
        {"name": "matvec_batch", "kind": "matmul", "rows": 8, "n": 8194, "k": 1280, "dtype": "f32", "group": 64, "bias": True,
         "residual": False, "swiglu": False},
        # a few dozen rows, nothing a multiple of anything
        {"name": "matmul_ragged", "kind": "matmul", "rows": 45, "n": 3841, "k": 1283, "dtype": "bf16", "group": 32, "bias": False,
         "residual": False, "swiglu": False},
        # gate and up projections of a long prompt
        {"name": "matmul_prompt", "kind": "matmul", "rows": 2048, "n": 10240, "k": 5120, "dtype": "bf16", "group": 128, "bias": False,
         "residual": False, "swiglu": True},
        # one token: norm and the q, k, v projections
        {"name": "linear_token", "kind": "linear", "rows": 1, "n": 4096, "k": 1024, "dtype": "f32", "group": 128, "norm": True, "swiglu": False},
        # a prefix of the usual length: norm, gate and up projections
        {"name": "linear_prefix", "kind": "linear", "rows": 155, "n": 10240, "k": 1280, "dtype": "bf16", "group": 128, "norm": True, "swiglu": True},
        # a small odd matrix at load time
        {"name": "pack_small", "kind": "pack", "n": 2049, "k": 387, "dtype": "bf16", "group": 32},
        # a large one
        {"name": "pack_large", "kind": "pack", "n": 16384, "k": 5120, "dtype": "f32", "group": 128},
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["norm", "norm", "matmul", "matmul", "matmul", "linear", "linear", "pack"])
    dtype, group = rng.choice(["f32", "bf16", "f16"]), rng.choice([32, 64, 128])
    if kind == "norm":
        rows = log_int(1, 8192)
        return {"kind": kind, "rows": rows, "cols": log_int(64, min(8192, 8192 * 5120 // rows)), "dtype": rng.choice(["bf16", "f16"] if rows > 4096 else [dtype]),
                "group": group, "residual": rng.random() < 0.5}
    if kind == "pack":
        return {"kind": kind, "n": log_int(64, 16384), "k": log_int(64, 5120), "dtype": dtype, "group": group}
    swiglu = rng.random() < 0.3
    if kind == "linear":
        rows, k = log_int(1, 512), log_int(64, 8192)
        n = log_int(64, 16384)
        return {"kind": kind, "rows": rows, "n": n + (n & 1 if swiglu else 0), "k": k, "dtype": dtype, "group": group, "norm": rng.random() < 0.7, "swiglu": swiglu}
    rows, k = log_int(1, 2048), log_int(64, 8192)
    n = log_int(64, min(152000, 155_000_000 // k, 2048 * 10240 * 5120 // (rows * k)))
    return {"kind": kind, "rows": rows, "n": n + (n & 1 if swiglu else 0), "k": k, "dtype": dtype, "group": group, "bias": rng.random() < 0.4,
            "residual": rng.random() < 0.4, "swiglu": swiglu}


def up(v, m):
    return -(-v // m) * m


# ------------------------------------------------------------------ plain forms
def group_max(y, group, of):
    """`of` over each group of columns, the last one as far as the matrix goes: [rows][groups]."""
    y = torch.nn.functional.pad(y, (0, up(y.shape[1], group) - y.shape[1]))
    return of(y.view(y.shape[0], -1, group))


def spread(s, group, cols):
    return s.repeat_interleave(group, 1)[:, :cols]


def to_codes(y, s, group, lo, hi):
    """Nearest codes of y (64 bits: quotients lie next to borders) under scales s, zero where a scale is zero or not finite."""
    s64 = spread(s.double(), group, y.shape[1])
    q = (y.double() / s64).round().clamp(lo, hi)
    return torch.where((s64 > 0) & torch.isfinite(s64), q, torch.zeros((), dtype=torch.float64, device=y.device))


def activation_codes(y, group):
    s = (group_max(y.abs(), group, lambda v: v.amax(2)) / 127).float()
    s = torch.where(torch.isfinite(s), s, torch.full((), math.nan, device=s.device))
    return to_codes(y, s, group, -127, 127), s


def weight_codes(w, group):
    w = w.double()
    most = torch.maximum(group_max(w, group, lambda v: v.amax(2)) / 7, -group_max(w, group, lambda v: v.amin(2)) / 8)
    s = most.float().bfloat16()
    s = torch.where(torch.isfinite(s), s, torch.full((), math.nan, dtype=s.dtype, device=s.device))
    return to_codes(w, s, group, -8, 7), s


def rms(h, w, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()


def pack(q, s, group):
    """Codes [n][k] and their scales [n][groups] in the layout above."""
    n, k = q.shape
    np_, kp = up(n, 16), up(k, 128)
    q = torch.nn.functional.pad(q.to(torch.int8), (0, kp - k, 0, np_ - n))
    q = q.view(np_ // 16, 16, kp // 128, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)  # tile row, tile, j, row, 32-column block, i
    q = q.reshape(np_ // 16, kp // 128, 64, 2, 2, 8)
    b = (q[..., 0, :] & 15) | (q[..., 1, :] << 4)
    s = torch.nn.functional.pad(s, (0, kp // group - s.shape[1], 0, np_ - n))
    s = s.view(np_ // 16, 16, kp // 128, 128 // group).permute(0, 2, 1, 3)
    return b.reshape(np_ // 16, kp // 128, 1024).view(torch.uint8).contiguous(), s.contiguous()


def unpack(packed, scales, n, k, group):
    """The values (32 bits) that packed weights stand for: [n][k]."""
    nt, kb = packed.shape[:2]
    b = packed.view(torch.int8).view(nt, kb, 4, 16, 2, 1, 8)
    q = torch.cat([(b << 4) >> 4, b >> 4], 5)  # tile row, tile, j, row, p, half, i
    q = q.permute(0, 3, 1, 4, 5, 2, 6).reshape(nt * 16, kb * 128)[:n, :k]
    s = scales.permute(0, 2, 1, 3).reshape(nt * 16, kb * (128 // group))[:n].float()
    return q.float() * spread(s, group, k)


def epilogue(v, s):
    if s.get("bias") is not None:
        v = v + s["bias"]
    if s["case"]["swiglu"]:
        g, u = v[:, 0::2], v[:, 1::2]
        v = g / (1 + torch.exp(-g)) * u
    if s.get("residual") is not None:
        v = v + s["residual"].float()
    return v.to(TYPES[s["case"]["dtype"]])


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def hidden(rows, cols):
        # a few channels are far larger than the others, as in residual streams
        return normal(rows, cols) * (1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.01))

    kind, t, group, s = case["kind"], TYPES[case["dtype"]], case["group"], {"case": dict(case)}
    if kind == "norm":
        s["x"] = hidden(case["rows"], case["cols"]).to(t)
        s["weight"] = (1 + 0.1 * normal(case["cols"])).to(t)
        s["residual"] = hidden(case["rows"], case["cols"]).to(t) if case["residual"] else None
        return s
    if kind == "pack":
        s["w"] = (0.02 * normal(case["n"], case["k"])).to(t)
        return s
    rows, n, k = case["rows"], case["n"], case["k"]
    q, sw = weight_codes(0.02 * normal(n, k), group)
    s["packed"], s["scales"] = pack(q, sw, group)
    x = hidden(rows, k)
    if kind == "linear":
        s["x"] = x.to(t)
        s["weight"] = (1 + 0.1 * normal(k)).to(t) if case["norm"] else None
        return s
    q, sx = activation_codes(x, group)
    s["q"] = torch.nn.functional.pad(q.to(torch.int8), (0, up(k, 128) - k))
    s["sx"] = torch.nn.functional.pad(sx, (0, up(k, 128) // group - sx.shape[1]))
    s["bias"] = 0.1 * normal(n) if case["bias"] else None
    s["residual"] = normal(rows, n // 2 if case["swiglu"] else n).to(t) if case["residual"] else None
    return s


# ------------------------------------------------------------------ one pass
def operators():
    """The framework's operators."""
    at = str(Path.cwd() / "index-tts-25-metal_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import itts_ops

    return itts_ops


def run(s):
    c = s["case"]
    kind, group = c["kind"], c["group"]
    if own:
        ops = operators()
        if kind == "norm":
            r = ops.rmsnorm_q8(s["x"], s["weight"], EPS, residual=s["residual"], group=group, values=True)
            return {"h": r.h, "values": r.values, "scales": r.scales}
        if kind == "pack":
            return ops.q4_unpack(ops.q4_pack(s["w"], group), TYPES[c["dtype"]])
        w = ops.Q4Weight(s["packed"], s["scales"], c["n"], c["k"], group)
        if kind == "linear":
            return ops.q4_linear(s["x"], w, norm_weight=s["weight"], eps=EPS, swiglu=c["swiglu"], out_dtype=TYPES[c["dtype"]])
        return ops.q4_matmul(s["q"], s["sx"], w, bias=s["bias"], residual=s["residual"], swiglu=c["swiglu"], out_dtype=TYPES[c["dtype"]])
    if kind == "norm":
        x = s["x"]
        h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
        q, sx = activation_codes(rms(h, s["weight"], EPS), group)
        values = (q.float() * spread(sx, group, c["cols"])).to(x.dtype)
        return {"h": h, "values": values, "scales": torch.nn.functional.pad(sx, (0, up(c["cols"], 128) // group - sx.shape[1]))}
    if kind == "pack":
        q, sw = weight_codes(s["w"], group)
        return (q.float() * spread(sw.float(), group, c["k"])).to(s["w"].dtype)
    if kind == "linear":
        y = s["x"].double() if s["weight"] is None else rms(s["x"], s["weight"], EPS)
        q, sx = activation_codes(y, group)
        x = q.float() * spread(sx, group, c["k"])
    else:
        x = s["q"][:, : c["k"]].float() * spread(s["sx"], group, c["k"])
    return epilogue(x @ unpack(s["packed"], s["scales"], c["n"], c["k"], group).t(), s)


# ------------------------------------------------------------------ work
def work(case):
    kind, size, group = case["kind"], BYTES[case["dtype"]], case["group"]
    if kind == "norm":
        cells = case["rows"] * case["cols"]
        return {"bytes": cells * (size * (4 if case["residual"] else 2) + 1) + 4 * cells / group + size * case["cols"], "flops": 6 * cells}
    if kind == "pack":
        cells = case["n"] * case["k"]
        return {"bytes": cells * (2 * size + 1 + 4 / group), "flops": 4 * cells}
    rows, n, k = case["rows"], case["n"], case["k"]
    out = rows * (n // 2 if case["swiglu"] else n) * size
    moved = n * k * (0.5 + 2 / group) + out
    if kind == "linear":
        return {"bytes": moved + rows * k * size + (k * size if case["norm"] else 0), "flops": 2 * rows * n * k}
    return {"bytes": moved + rows * k * (1 + 4 / group) + (out if case["residual"] else 0) + (4 * n if case["bias"] else 0), "flops": 2 * rows * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind, group = case["kind"], case["group"]

    def codes(y, scale, lo, hi):
        """y and its group scales to the values that the nearest codes stand for."""
        at = torch.arange(y.shape[1], device=y.device) // group
        each = scale[:, at].double()
        return torch.clamp(torch.round(y / torch.where(each == 0, torch.ones_like(each), each)), lo, hi) * each

    def eight(y):
        ends = [y[:, i : i + group].abs().max(1).values for i in range(0, y.shape[1], group)]
        scale = (torch.stack(ends, 1) / 127).float()
        return codes(y, scale, -127, 127), scale

    def normed(h, weight):
        h = h.double()
        return h * torch.rsqrt((h * h).sum(1) / h.shape[1] + EPS)[:, None] * weight.double()

    if kind == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        values, scale = eight(normed(h.to(s["x"].dtype), s["weight"]))
        more = up(case["cols"], 128) // group - scale.shape[1]
        return {"h": h, "values": values, "scales": torch.cat([scale.double(), scale.new_zeros(scale.shape[0], more).double()], 1)}
    if kind == "pack":
        w = s["w"].double()
        parts = [w[:, i : i + group] for i in range(0, w.shape[1], group)]
        zero = w.new_zeros(1)
        tops = [torch.maximum(torch.maximum(p.max(1).values, zero) / 7, torch.maximum(-p.min(1).values, zero) / 8) for p in parts]
        return codes(w, torch.stack(tops, 1).float().bfloat16(), -8, 7)

    n, k = case["n"], case["k"]
    # each column's code by its place in the tile
    c = torch.arange(k, device="cuda")
    tile, p, half, j, i = c // 128, c % 128 // 64, c % 64 // 32, c % 32 // 8, c % 8
    flat = s["packed"].reshape(s["packed"].shape[0], -1).int()
    total = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
    if kind == "linear":
        x = eight(s["x"].double() if s["weight"] is None else normed(s["x"], s["weight"]))[0]
    else:
        x = s["q"][:, :k].double() * s["sx"].double()[:, c // group]
    for r in range(16):  # the rows r, r + 16, ... lie at the same place of their tiles
        byte = flat[: -(-(n - r) // 16), tile * 1024 + (16 * j + r) * 16 + 8 * p + i]
        code = torch.where(half == 1, byte // 16, byte % 16)
        code = torch.where(code > 7, code - 16, code)
        scale = s["scales"][: code.shape[0], tile, r, c % 128 // group].double()
        total[:, r::16] = x @ (code.double() * scale).t()
    if s.get("bias") is not None:
        total += s["bias"].double()
    if case["swiglu"]:
        total = total[:, 0::2] * torch.sigmoid(total[:, 0::2]) * total[:, 1::2]
    return total if s.get("residual") is None else total + s["residual"].double()
