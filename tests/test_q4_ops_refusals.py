"""What the operators on 4-bit weights and 8-bit activations refuse: checked before anything is enqueued, so
without a GPU, through itts_ops and through the C ABI."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops(itts):
    import itts_ops

    return itts_ops


def weight(ops, n=20, k=130, group=64):
    nt, kb = -(-n // 16), -(-k // 128)
    return ops.Q4Weight(torch.zeros(nt, kb, 1024, dtype=torch.uint8), torch.zeros(nt, kb, 16, 128 // group, dtype=BF16), n, k, group)


def refused(itts, match, fn, *args, **kw):
    with pytest.raises(itts.InvalidArgument, match=match):
        fn(*args, **kw)


def test_rows_to_codes(itts, ops):
    x, w = torch.zeros(3, 40), torch.ones(40)
    refused(itts, "on the GPU", ops.rmsnorm_q8, x, w)
    refused(itts, "on the GPU", ops.q8_quantize, x)
    refused(itts, "float32, bfloat16 or float16", ops.q8_quantize, x.double())
    refused(itts, "a matrix is wanted", ops.q8_quantize, x[0])
    refused(itts, "next to each other", ops.q8_quantize, x.t())
    refused(itts, "32, 64 or 128", ops.q8_quantize, x, 16)
    refused(itts, "32, 64 or 128", ops.rmsnorm_q8, x, w, group=256)
    refused(itts, "weight: 40", ops.rmsnorm_q8, x, w[:39])
    refused(itts, "weight: 40", ops.rmsnorm_q8, x, torch.ones(80)[::2])
    refused(itts, "weight: torch.float32 or float32", ops.rmsnorm_q8, x, w.bfloat16())
    refused(itts, "residual", ops.rmsnorm_q8, x, w, residual=x[:2])
    refused(itts, "residual", ops.rmsnorm_q8, x, w, residual=x.bfloat16())
    refused(itts, "h:", ops.rmsnorm_q8, x, w, h=torch.zeros(3, 41))
    refused(itts, "values:", ops.q8_quantize, x, values=torch.zeros(3, 41))
    refused(itts, "q:", ops.q8_quantize, x, q=torch.zeros(3, 40, dtype=torch.int8))
    refused(itts, "scales:", ops.q8_quantize, x, scales=torch.zeros(3, 2))


def test_weights(itts, ops):
    refused(itts, "on the GPU", ops.q4_pack, torch.zeros(3, 4))
    refused(itts, "without rows or columns", ops.q4_pack, torch.zeros(0, 4))
    refused(itts, "without rows or columns", ops.q4_pack, torch.zeros(4, 0))
    refused(itts, "32, 64 or 128", ops.q4_pack, torch.zeros(3, 4), 33)
    refused(itts, "Q4Weight", ops.q4_unpack, torch.zeros(3, 4))
    w = weight(ops)
    refused(itts, "on the GPU", ops.q4_unpack, w)
    refused(itts, "dtype", ops.q4_unpack, w, torch.int8)
    refused(itts, "out", ops.q4_unpack, w, out=torch.zeros(20, 131))
    refused(itts, "packed codes", ops.q4_unpack, w._replace(n=33))
    refused(itts, "packed codes", ops.q4_unpack, w._replace(packed=w.packed[:1]))
    refused(itts, "packed codes", ops.q4_unpack, w._replace(packed=w.packed.to(torch.int8)))
    refused(itts, "the scales", ops.q4_unpack, w._replace(group=32))
    refused(itts, "32, 64 or 128", ops.q4_unpack, w._replace(group=48))


def test_products(itts, ops):
    w = weight(ops)
    q, s = torch.zeros(3, 256, dtype=torch.int8), torch.zeros(3, 4)
    refused(itts, "on the GPU", ops.q4_matmul, q, s, w)
    refused(itts, "q: ", ops.q4_matmul, q[:, :128], s, w)
    refused(itts, "q: ", ops.q4_matmul, q.float(), s, w)
    refused(itts, "q: ", ops.q4_matmul, q[:, ::2], s, weight(ops, 20, 100))
    refused(itts, "scales: ", ops.q4_matmul, q, s[:2], w)
    refused(itts, "scales: ", ops.q4_matmul, q, torch.zeros(3, 2), w)
    refused(itts, "bias", ops.q4_matmul, q, s, w, bias=torch.zeros(19))
    refused(itts, "bias", ops.q4_matmul, q, s, w, bias=torch.zeros(20, dtype=BF16))
    refused(itts, "residual", ops.q4_matmul, q, s, w, residual=torch.zeros(3, 19))
    refused(itts, "residual", ops.q4_matmul, q, s, w, residual=torch.zeros(3, 20), out_dtype=BF16)
    refused(itts, "out_dtype", ops.q4_matmul, q, s, w, out_dtype=torch.float64)
    refused(itts, "out: ", ops.q4_matmul, q, s, w, out=torch.zeros(3, 21))
    refused(itts, "pairs of columns", ops.q4_matmul, torch.zeros(3, 128, dtype=torch.int8), torch.zeros(3, 2), weight(ops, 17, 100), swiglu=True)
    x = torch.zeros(3, 130)
    refused(itts, "on the GPU", ops.q4_linear, x, w)
    refused(itts, "rows of 130", ops.q4_linear, x[:, :129], w)
    refused(itts, "norm_weight", ops.q4_linear, x, w, norm_weight=torch.zeros(129))
    refused(itts, "norm_weight", ops.q4_linear, x, w, norm_weight=torch.zeros(130, dtype=BF16))


def library(itts):
    """The C ABI with the argument types of include/itts_ops.h."""
    lib = C.CDLL(str(itts.LIB_PATH))
    p, i64, i32, u32, f32, z = C.c_void_p, C.c_int64, C.c_int32, C.c_uint32, C.c_float, C.c_size_t
    for name, res, args in (
        ("itts_ops_last_error", C.c_char_p, []),
        ("itts_rmsnorm_q8", i32, [p, i64, p, i64, p, i32, i32, i64, i64, f32, i32, p, i64, p, i64, p, p, p]),
        ("itts_q4_packed_bytes", z, [i64, i64]),
        ("itts_q4_scale_count", z, [i64, i64, i32]),
        ("itts_q4_pack", i32, [p, i64, i32, i64, i64, i32, p, p, p]),
        ("itts_q4_unpack", i32, [p, p, i64, i64, i32, i32, p, i64, p]),
        ("itts_q4_matmul", i32, [p, p, i64, p, p, i64, i64, i32, p, p, i64, u32, i32, p, i64, p]),
        ("itts_q4_linear_workspace", z, [i64, i64, i64, i32]),
        ("itts_q4_linear", i32, [p, i64, i32, i64, p, i32, f32, p, p, i64, i64, i32, p, p, i64, u32, i32, p, i64, p, z, p]),
    ):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def test_two_hip_runtimes_are_refused():
    """torch's streams belong to the HIP runtime that torch brings: with itts_gpt imported first, on the
    system's runtime, the operators' import says so; the other order works."""
    pkg = str(Path(__file__).resolve().parent.parent / "index-tts-25-metal_amd")
    for order, fine in (("import torch, itts_gpt, itts_ops", True), ("import itts_ops", True), ("import itts_gpt, itts_ops", False)):
        p = subprocess.run([sys.executable, "-c", order], cwd=pkg, capture_output=True, text=True)
        one = "two HIP runtimes" not in p.stderr
        # (where torch brings no runtime of its own, there is one in any order)
        assert (p.returncode == 0) == one and (one or not fine), (order, p.stderr[-500:])


def place(i, off=0):
    """The i-th of some addresses 2^24 bytes apart (no buffer below is larger), and off bytes behind it."""
    return C.c_void_p(((i + 1) << 24) + off)


def calls(itts):
    """The C ABI's calls with arguments that would be accepted, each in a place of its own."""
    lib = library(itts)

    def norm(x=place(0), xs=64, res=None, rs=64, w=place(1), wt=0, t=0, rows=2, cols=64, eps=1e-6, g=64, h=None, hs=64, v=None, vs=64, q=place(2), s=place(3)):
        return lib.itts_rmsnorm_q8(x, xs, res, rs, w, wt, t, rows, cols, eps, g, h, hs, v, vs, q, s, None)

    def matmul(q=place(0), qs=place(1), rows=2, p=place(2), s=place(3), n=32, k=128, g=128, bias=None, res=None, rs=32, flags=0, t=0, out=place(4), os=32):
        return lib.itts_q4_matmul(q, qs, rows, p, s, n, k, g, bias, res, rs, flags, t, out, os, None)

    def linear(x=place(0), xs=128, xt=0, rows=200, nw=None, wt=0, eps=0.0, p=place(1), s=place(2), n=32, k=128, g=128, bias=None, res=None, rs=32, flags=0, t=0,
               out=place(3), os=32, work=place(4), bytes_=1 << 20):
        return lib.itts_q4_linear(x, xs, xt, rows, nw, wt, eps, p, s, n, k, g, bias, res, rs, flags, t, out, os, work, bytes_, None)

    def pack(w=place(0), ws=128, t=0, n=32, k=128, g=128, p=place(1), s=place(2)):
        return lib.itts_q4_pack(w, ws, t, n, k, g, p, s, None)

    def unpack(p=place(0), s=place(1), n=32, k=128, g=128, t=0, out=place(2), os=128):
        return lib.itts_q4_unpack(p, s, n, k, g, t, out, os, None)

    return lib, norm, matmul, linear, pack, unpack


def test_the_c_abi_refuses(itts, ops):
    """Addresses that are never read: every call here ends in its checks, with a message."""
    lib, norm, matmul, linear, pack, unpack = calls(itts)

    def no(fn, *cases, message=b""):
        for kw in cases:
            assert fn(**kw) == -1 and lib.itts_ops_last_error() and message in lib.itts_ops_last_error(), kw
            assert b"overlaps" not in lib.itts_ops_last_error(), kw

    assert norm(rows=0) == 0
    no(norm, {"x": None}, {"w": None}, {"q": None}, {"s": None}, message=b"Missing")
    no(norm, {"xs": -1}, {"h": place(5), "hs": 63}, {"v": place(5), "vs": 63}, {"res": place(5), "rs": -1}, message=b"stride")
    no(norm, {"t": 3}, {"t": -1}, {"wt": 1}, {"t": 1, "wt": 2}, {"rows": -1}, {"rows": 1 << 40}, {"cols": 0}, {"cols": 1 << 40}, {"eps": -1.0},
       {"eps": float("nan")}, {"g": 0}, {"g": 16})
    no(norm, {"q": place(2, 8)}, {"x": place(0, 1)}, {"s": place(3, 2)}, {"w": place(1, 2)}, message=b"Misaligned")

    assert matmul(rows=0) == 0
    no(matmul, {"q": None}, {"qs": None}, {"p": None}, {"s": None}, {"out": None}, message=b"Missing")
    no(matmul, {"n": 0}, {"n": 1 << 40}, {"k": 0}, {"k": 1 << 40}, {"g": 1}, {"flags": 2}, {"t": 7}, {"n": 33, "flags": 1, "os": 40}, {"rows": -1}, {"rows": 1 << 40})
    no(matmul, {"os": 31}, {"res": place(5), "rs": -2}, message=b"stride")
    no(matmul, {"q": place(0, 4)}, {"p": place(2, 4)}, {"out": place(4, 2)}, {"bias": place(5, 1)}, message=b"Misaligned")
    no(matmul, {"rows": 1 << 19, "n": 1 << 20, "os": 1 << 20}, message=b"Too many")

    need = lib.itts_q4_linear_workspace(200, 32, 128, 128)
    assert need >= 200 * 132 and linear(rows=0) == 0
    no(linear, {"x": None}, {"out": None}, message=b"Missing")
    no(linear, {"xs": -1}, {"xt": 5}, {"nw": place(5), "wt": 1}, {"nw": place(5), "eps": -1.0})
    no(linear, {"work": None}, {"bytes_": need - 1}, {"work": place(4, 16)}, message=b"orkspace")
    no(linear, {"x": place(0, 2)}, message=b"Misaligned")

    no(pack, {"w": None}, {"ws": -1}, {"t": 9}, {"n": 0}, {"k": 0}, {"g": 2}, {"p": None}, {"s": None}, {"p": place(1, 1)})
    no(unpack, {"out": None}, {"os": 127}, {"t": 9}, {"n": 0}, {"k": 0}, {"g": 2}, {"p": None}, {"s": None})
    # a workgroup a tile: no more tiles than a launch can have
    no(pack, {"n": 1 << 26, "k": 257, "ws": 0}, message=b"too large")
    no(unpack, {"n": 1 << 26, "k": 257, "os": 257}, message=b"too large")
    assert lib.itts_q4_packed_bytes(17, 129) == 4 * 1024 and lib.itts_q4_packed_bytes(0, 5) == 0 and lib.itts_q4_packed_bytes(1 << 40, 5) == 0
    assert lib.itts_q4_scale_count(17, 129, 32) == 4 * 64 and lib.itts_q4_scale_count(17, 129, 31) == 0


def test_outputs_over_inputs_and_each_other(itts, ops):
    """Workgroups write an output while others still read the inputs: no byte may belong to both."""
    lib, norm, matmul, linear, pack, unpack = calls(itts)

    def overlaps(fn, *cases):
        for kw in cases:
            assert fn(**kw) == -1 and b"overlaps" in lib.itts_ops_last_error(), (kw, lib.itts_ops_last_error())

    x, w, q, s, other = place(0), place(1), place(2), place(3), place(5)
    overlaps(norm, {"v": x}, {"h": place(0, 4)}, {"h": x, "hs": 65}, {"res": place(0, 128), "h": x}, {"v": place(0, 256)},
             {"xs": 128, "h": place(0, 252), "hs": 128})
    overlaps(norm, {"h": w}, {"v": w}, {"v": other, "h": other}, {"h": q}, {"v": q}, {"h": s}, {"v": s}, {"h": place(3, -508)}, {"q": x}, {"q": place(0, 496)},
             {"q": w}, {"res": other, "q": other}, {"s": x}, {"s": w}, {"res": other, "s": other}, {"s": place(2, 124)}, {"rows": 1, "h": w})
    p, bias = place(2), {"bias": other}
    overlaps(matmul, {"out": place(0)}, {"out": place(0, 252)}, {"out": place(1)}, {"out": place(1, -252)}, {"out": p}, {"out": place(2, 2048 - 4)}, {"out": s},
             {"out": place(3, 64 - 4)}, {**bias, "out": other}, {**bias, "out": other, "rows": 1}, {"out": place(5, 124), **bias}, {"res": place(4, 4)})
    overlaps(linear, {"out": place(0, 100), "os": 128}, {"rows": 1, "out": place(0, 100), "os": 128}, {"nw": place(3)}, {"rows": 1, "nw": place(3)},
             {"out": place(1)}, {"out": place(2)}, {"out": other, **bias})
    overlaps(linear, {"work": place(0)}, {"work": place(1)}, {"work": place(2)}, {"work": place(3)}, {"work": other, **bias}, {"work": other, "res": other},
             {"work": other, "nw": other})
    overlaps(pack, {"p": place(0)}, {"s": place(0)}, {"s": place(1)}, {"s": place(1, 2032)}, {"p": place(0, 4096)})
    overlaps(unpack, {"out": place(0)}, {"out": place(1)}, {"out": place(0, 2044)}, {"out": place(1, -512), "n": 2})


def test_weight_bits(itts):
    for kw in ({"weight_bits": 8}, {"weight_bits": 4, "head_bits": 16}, {"head_bits": 0}):
        refused(itts, "4 or 32 bits", itts.QwenDecoder, {}, **kw)
