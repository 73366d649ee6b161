"""The kernels that the operators on 4-bit weights and 8-bit activations choose for large calls, against their definitions
in 64 bits (q4_reference.py): each block shape of the products, and rows enough that a workgroup goes through several.

Products of more than 16 rows take blocks by the size of their grid; SHAPES has one size for each choice, named by the
block.  Few columns keep the reference cheap."""
import numpy as np
import pytest
import torch

import q4_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
GROUPS = [32, 64, 128]

# rows, weight rows (a multiple of 16), columns
SHAPES = {
    "32 x 64, columns by 4": (260, 2064, 1100),
    "32 x 64, columns by 4, one turn": (260, 2064, 130),
    "64 x 64": (200, 7184, 300),
    "64 x 64, rows of a half block": (20, 28688, 130),
    "64 x 128": (130, 21904, 300),
    "32 x 128": (20, 65424, 130),
    "5 to 16 rows, four tile rows": (16, 16400, 300),
    "5 to 16 rows, four tile rows, five of them": (5, 16400, 1100),
    "1 to 4 rows, four tile rows, one turn": (3, 32784, 300),
    "1 to 4 rows, four tile rows, two turns": (3, 32784, 1100),
}
BLOCKS = [name for name in SHAPES if "5 to" not in name and "1 to" not in name]


@pytest.fixture(scope="module")
def ops(itts):
    import itts_ops

    return itts_ops


def tensor(a, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype).cuda()


PERIOD = 1008  # 63 tile rows


def made(ops, r, n, k, group):
    """A weight of n rows, a multiple of 16, whose rows repeat after PERIOD (no block's tile rows divide 63), with the codes
    and scales of its first ones: the reference computes those columns alone."""
    period = min(n, PERIOD)
    q = r.integers(-8, 8, (period, k))
    s = ref.bf16(0.02 * r.random((period, -(-k // group))) + 0.01)
    s = np.pad(s, ((0, 0), (0, ref.up(k, 128) // group - s.shape[1])))
    packed, scales = (t.repeat(-(-n // period), *[1] * (t.dim() - 1))[: n // 16].cuda() for t in ref.pack_codes(q, s, group))
    return ops.Q4Weight(packed, scales, n, k, group), q, s


def columns(a, n):
    """a's columns, repeated up to n of them."""
    return np.tile(a, -(-n // a.shape[-1]))[..., :n]


def first_rows(w, n):
    """The weight's first n rows, of the same last tile row: padding codes and scales are zero."""
    packed, scales = w.packed.clone(), w.scales.clone()
    assert -(-n // 16) == packed.shape[0]
    if n % 16:
        packed[-1].view(-1, 4, 16, 16)[:, :, n % 16 :] = 0
        scales[-1, :, n % 16 :] = 0
    return w._replace(packed=packed, scales=scales, n=n)


def rows_of(r, rows, k, group):
    kp = ref.up(k, 128)
    q = r.integers(-127, 128, (rows, kp)).astype(np.int8)
    q[:, k:] = 0
    s = (0.02 * r.random((rows, kp // group)) + 1e-3).astype(np.float32)
    s[:, -(-k // group) :] = 0
    return q, s


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("name", SHAPES)
def test_each_block_shape_matches_the_definition(ops, name, group):
    """Rows of outputs and residuals that are 16-byte aligned and that are not, a ragged last block of rows' columns,
    bias, SwiGLU and residual, every type."""
    rows, n, k = SHAPES[name]
    r = np.random.default_rng((rows, n, group))
    full, qw, sw = made(ops, r, n, k, group)
    q, sx = rows_of(r, rows, k, group)
    tq, ts = torch.from_numpy(q).cuda(), torch.from_numpy(sx).cuda()
    bias, res = r.standard_normal(len(qw)).astype(np.float32), r.standard_normal((rows, n)).astype(np.float32)
    tb = tensor(columns(bias, n))
    one, two = ref.product(q, sx, qw, sw, group), ref.product(q, sx, qw, sw, group, bias=bias.astype(np.float64))
    pairs = ref.product(q, sx, qw, sw, group, bias=bias.astype(np.float64), swiglu=True)

    def check(out, product, t, what):
        want, err = (columns(a, out.shape[1]) for a in product)
        if t is not None:
            want = want + ref.to64(t)
            err = err + 2.0 ** -24 * (np.abs(want) + err)  # (one rounding for the residual)
        ref.check_product(out, want, err, what)

    for cols in (n, n - 9, n - 10):  # aligned rows, odd ones, and an odd number of pairs
        w = first_rows(full, cols)
        for dtype in TYPES:
            check(ops.q4_matmul(tq, ts, w, out_dtype=dtype), one, None, (cols, dtype, "bare"))
            t = tensor(res[:, :cols], dtype)
            out = ops.q4_matmul(tq, ts, w, bias=tb[:cols], residual=t, out_dtype=dtype)
            check(out, two, t, (cols, dtype, "bias and residual"))
            assert torch.equal(ops.q4_matmul(tq, ts, w, bias=tb[:cols], residual=t, out_dtype=dtype, out=t), out) and torch.equal(t, out)
            if cols % 2 == 0:
                t = tensor(res[:, : cols // 2], dtype)
                out = ops.q4_matmul(tq, ts, w, bias=tb[:cols], residual=t, swiglu=True, out_dtype=dtype)
                check(out, pairs, t, (cols, dtype, "SwiGLU"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", BLOCKS)
def test_products_at_any_address(ops, name, dtype):
    """Output and residual rows that begin at each of eight places in 16 bytes, and at another one each: the bits of
    aligned ones, and not an element around them changed."""
    rows, n, _ = SHAPES[name]
    k, group = 130, 64
    r = np.random.default_rng((rows, n))
    full, _, _ = made(ops, r, n, k, group)
    w = first_rows(full, n - 10)
    q, s = (torch.from_numpy(a).cuda() for a in rows_of(r, rows, k, group))
    bias = tensor(r.standard_normal(n - 10))
    for swiglu in (False, True):
        cols = w.n // 2 if swiglu else w.n
        t = tensor(r.standard_normal((rows, cols)), dtype)
        want = ops.q4_matmul(q, s, w, bias=bias, residual=t, swiglu=swiglu, out_dtype=dtype)
        for at in range(8):
            for stride in (ref.up(cols, 8) + 16, ref.up(cols, 8) + 17):

                def place():
                    whole = torch.full((rows + 1, stride), 7.0, dtype=dtype, device="cuda")
                    return whole, torch.as_strided(whole, (rows, cols), (stride, 1), at)

                (_, res), (whole, out) = place(), place()
                res.copy_(t)
                ops.q4_matmul(q, s, w, bias=bias, residual=res, swiglu=swiglu, out_dtype=dtype, out=out)
                assert torch.equal(out, want), (swiglu, at, stride)
                out.fill_(7.0)
                assert bool((whole == 7).all()), (swiglu, at, stride)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("name", BLOCKS)
def test_extreme_codes_and_values_that_are_not_finite(ops, name, group):
    """Codes at their ends stay whole numbers; a row, or a weight row, that is not finite spoils itself alone."""
    rows, n, _ = SHAPES[name]
    k = 256
    codes = np.full((16, k), -8)
    codes[1::2] = 7
    packed, scales = (t.repeat(n // 16, *[1] * (t.dim() - 1)).cuda() for t in ref.pack_codes(codes, np.ones((16, k // group), np.float32), group))
    w = ops.Q4Weight(packed, scales, n, k, group)
    q = np.full((rows, k), -128, np.int8)
    q[::2] = 127
    tq, ts = torch.from_numpy(q).cuda(), tensor(np.ones((rows, k // group)))
    want = tensor(columns(q.astype(np.float64) @ codes.T, n))  # (whole numbers of 18 bits)
    assert torch.equal(ops.q4_matmul(tq, ts, w), want)
    s, m, at = ts.clone(), rows - 2, n - 3
    s[m, 1] = float("nan")
    bad = w.scales.clone()
    bad.view(n // 16, 2, 16, 128 // group)[at // 16, 0, at % 16, 0] = float("nan")
    want[m], want[:, at] = float("nan"), float("nan")
    got = ops.q4_matmul(tq, s, w._replace(scales=bad))
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


# ------------------------------------------------------------------ rows to 8 bits
# More rows than workgroups are resident for: each goes through several, the next row's loads under way.  One to four
# runs of columns a lane, one to sixteen waves a row, aligned and not; beyond 32768 columns the rows are read twice.
MANY = [(4200, 500), (4200, 512), (8200, 129), (4200, 1000), (2100, 1290), (2100, 2048), (1100, 5120), (1100, 5121), (1100, 8192), (1030, 9000), (600, 8192), (516, 12296)]


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,cols", MANY)
def test_many_rows_are_the_definition(ops, rows, cols, group):
    r = np.random.default_rng((rows, cols, group))
    dtype = {32: F32, 64: F16, 128: BF16}[group] if cols % 8 else {32: BF16, 64: F32, 128: BF16}[group]
    a = r.standard_normal((rows, cols), np.float32) * (1 + 10 * (r.random(cols) < 0.02).astype(np.float32))
    x, res = tensor(a, dtype), tensor(r.standard_normal((rows, cols), np.float32), dtype)
    w = tensor(1 + 0.1 * r.standard_normal(cols), dtype)
    eps = float(np.float32(1e-6))
    h = (x.float() + res.float()).to(dtype)
    # the reference on the first rows, some between, and the last ones, which are later rows of their workgroups
    some = np.unique(np.concatenate([np.arange(20), r.integers(0, rows, 40), np.arange(rows - 200, rows)]))

    def check(got, of, norm, what):
        y = ref.to64(of[some])
        ref.check_codes(got.q[some], got.scales[some], ref.rms(y, ref.to64(w), eps) if norm else y, group, what)

    out = ops.rmsnorm_q8(x, w, 1e-6, residual=res, group=group, values=True)
    assert torch.equal(out.h, h)
    check(out, h, True, "norm of a sum")
    each = out.scales.repeat_interleave(group, 1)[:, :cols]
    assert torch.equal(out.values, (out.q[:, :cols].float() * each).to(dtype))
    check(ops.rmsnorm_q8(x, w, 1e-6, group=group), x, True, "norm")
    check(ops.q8_quantize(x, group), x, False, "quantize")
    # in place, over x and over the residual: the row ahead is read before it is written
    over_x, over_res = x.clone(), res.clone()
    for got, target in ((ops.rmsnorm_q8(over_x, w, 1e-6, residual=res, group=group, h=over_x, values=True), over_x),
                        (ops.rmsnorm_q8(x, w, 1e-6, residual=over_res, group=group, h=over_res, values=True), over_res)):
        assert torch.equal(target, h) and torch.equal(got.q, out.q) and torch.equal(got.scales, out.scales) and torch.equal(got.values, out.values)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1100, 20000), (1100, 20001), (1040, 33000), (1040, 33001), (4100, 512), (4100, 511), (3000, 1536), (3000, 3083), (1200, 16384)])
def test_a_row_has_its_own_bits_whatever_the_number_of_rows(ops, rows, cols, dtype):
    """A workgroup's later rows against calls that give it one row alone, with the norm, the residual and neither."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, res = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(cols, generator=g, device="cuda").to(dtype)
    for call in (lambda i: ops.rmsnorm_q8(x[i], w, residual=res[i], values=True), lambda i: ops.rmsnorm_q8(x[i], w), lambda i: ops.q8_quantize(x[i], 32, values=True)):
        whole = call(slice(None))
        for at in range(0, rows, 250):
            i = slice(at, min(at + 250, rows))
            for a, b in zip(whole, call(i)):
                assert (a is None and b is None) or torch.equal(a[i], b), at
