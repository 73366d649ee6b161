"""Operators on 4-bit weights and 8-bit activations (itts_ops, include/itts_ops.h) on the MI355X against
their definitions in 64 bits (tests/q4_reference.py), at the sizes, types, strides and values where they can go wrong."""
import numpy as np
import pytest
import torch

import q4_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


@pytest.fixture(scope="module")
def ops(itts):
    import itts_ops

    return itts_ops


def rng(*key):
    return np.random.default_rng(key)


def tensor(a, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype).cuda()


def weight_of(ops, r, n, k, group, scale=0.02):
    w = (scale * r.standard_normal((n, k))).astype(np.float32)
    q, s = ref.codes4(w, group)
    packed, scales = ref.pack_codes(q, s, group)
    return ops.Q4Weight(packed.cuda(), scales.cuda(), n, k, group), q, s


def codes_of(r, rows, k, group):
    """Codes over the whole range and scales, padding zero."""
    kp = ref.up(k, 128)
    q = r.integers(-127, 128, (rows, kp)).astype(np.int8)
    q[:, k:] = 0
    s = np.abs(r.standard_normal((rows, kp // group))).astype(np.float32) * 0.01 + 1e-3
    s[:, -(-k // group):] = 0
    return q, s


# ------------------------------------------------------------------ rows to 8 bits
ROWS = [(1, 1024), (1, 1), (3, 7), (2, 31), (5, 64), (4, 100), (2, 127), (2, 129), (7, 1280), (3, 2056), (2, 5121), (2, 8192), (1, 16387), (1, 40000), (300, 96), (2051, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_norm_codes_are_those_of_the_definition(ops, rows, cols, group, dtype):
    r = rng(rows, cols, group)
    x, res = tensor(r.standard_normal((rows, cols)) * (1 + 10 * (r.random(cols) < 0.02)), dtype), tensor(r.standard_normal((rows, cols)), dtype)
    w = tensor(1 + 0.1 * r.standard_normal(cols), dtype if group != 64 else F32)
    out = ops.rmsnorm_q8(x, w, 1e-6, residual=res, group=group, values=True)
    h = (x.cpu().float() + res.cpu().float()).to(dtype)
    assert torch.equal(out.h.cpu(), h)
    ref.check_codes(out.q, out.scales, ref.rms(ref.to64(h), ref.to64(w), float(np.float32(1e-6))), group)
    each = out.scales.cpu().repeat_interleave(group, 1)[:, :cols]
    assert torch.equal(out.values.cpu(), (out.q.cpu()[:, :cols].float() * each).to(dtype))
    bare = ops.rmsnorm_q8(x, w, 1e-6, group=group)
    assert bare.h is x and bare.values is None
    ref.check_codes(bare.q, bare.scales, ref.rms(ref.to64(x), ref.to64(w), float(np.float32(1e-6))), group)
    plain = ops.q8_quantize(x, group, values=True)
    ref.check_codes(plain.q, plain.scales, ref.to64(x), group)
    each = plain.scales.cpu().repeat_interleave(group, 1)[:, :cols]
    assert torch.equal(plain.values.cpu(), (plain.q.cpu()[:, :cols].float() * each).to(dtype))


@pytest.mark.parametrize("cols", [200, 256])
def test_norm_of_strided_rows_writes_only_them(ops, cols):
    """Rows inside wider matrices, at offsets that are and are not 16-byte aligned; what lies between
    them stays as it was; h may be x or the residual."""
    for dtype in TYPES:
        for off in (0, 3, 8):
            r = rng(cols, off)
            wide = [tensor(r.standard_normal((5, cols + 24)), dtype) for _ in range(4)]
            keep = [t.clone() for t in wide]
            x, res, h, val = (t[:, off : off + cols] for t in wide)
            w = tensor(1 + 0.1 * r.standard_normal(cols), dtype)
            out = ops.rmsnorm_q8(x, w, 1e-5, residual=res, group=32, h=h, values=val)
            whole = ops.rmsnorm_q8(x.contiguous(), w, 1e-5, residual=res.contiguous(), group=32, values=True)
            assert torch.equal(out.q, whole.q) and torch.equal(out.scales, whole.scales)
            assert torch.equal(h, whole.h) and torch.equal(val, whole.values)
            for t, k in zip(wide, keep):
                t[:, off : off + cols] = k[:, off : off + cols]
                assert torch.equal(t, k)
            for target in (x, res):
                again = ops.rmsnorm_q8(x, w, 1e-5, residual=res, group=32, h=target)
                assert torch.equal(target, whole.h) and torch.equal(again.q, whole.q) and torch.equal(again.scales, whole.scales)
                for t, k in zip(wide, keep):
                    t.copy_(k)
    one = tensor(rng(9).standard_normal((1, cols))).expand(6, cols)  # the same row six times
    out = ops.q8_quantize(one, 64)
    assert torch.equal(out.q, ops.q8_quantize(one.contiguous(), 64).q)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_codes_of_zeros_infinities_and_nan(ops, group):
    inf, nan = float("inf"), float("nan")
    for dtype in TYPES:
        top = torch.finfo(dtype).max
        x = rng(group).standard_normal((9, 300))
        x[1, :] = 0
        x[2, group : 2 * group] = 0
        x[3, 5] = inf
        x[4, 260] = -inf
        x[5, 299] = nan
        x[6, 0], x[6, 1] = nan, inf
        x[7, :] = -0.0
        t = tensor(x, dtype)
        t[8, :] = top
        q = ops.q8_quantize(t, group, values=True)
        ref.check_codes(q.q, q.scales, ref.to64(t), group, "quantize")
        w = torch.ones(300, dtype=dtype, device="cuda")
        w[7] = 0
        n = ops.rmsnorm_q8(t, w, 0.0 if dtype == F32 else 1e-6, group=group)
        ref.check_codes(n.q, n.scales, ref.rms(ref.to64(t), ref.to64(w), 0.0 if dtype == F32 else float(np.float32(1e-6))), group, "norm")
        w[100] = nan
        n = ops.rmsnorm_q8(t, w, 1e-6, group=group)
        ref.check_codes(n.q, n.scales, ref.rms(ref.to64(t), ref.to64(w), float(np.float32(1e-6))), group, "norm, NaN weight")


def test_codes_on_halves_go_to_the_even_one(ops):
    """Scales of one and three exactly, quotients on halves."""
    for s in (1.0, 3.0, 0.375):
        x = np.zeros((1, 128))
        x[0, 0] = 127
        x[0, 1:101] = np.arange(-50, 50) + 0.5
        out = ops.q8_quantize(tensor(x * s), 128)
        assert float(out.scales[0, 0]) == s
        assert np.array_equal(out.q.cpu().numpy()[0], np.rint(x[0]))


def test_tiny_numbers(ops):
    """Scales in and under the range of denormal numbers."""
    x = np.zeros((3, 128))
    x[0] = 1e-40 * rng(1).standard_normal(128)
    x[1, 3] = 1.4e-45
    x[2, :] = 3e-38
    t = tensor(x)
    out = ops.q8_quantize(t, 128)
    ref.check_codes(out.q, out.scales, ref.to64(t), 128)


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (15, 127), (17, 129), (33, 300), (130, 1024), (8, 40), (5, 2056)])
def test_packing_is_the_definition(ops, n, k, group, dtype):
    r = rng(n, k, group)
    w = tensor(0.02 * r.standard_normal((n, k)), dtype)
    got = ops.q4_pack(w, group)
    q, s = ref.codes4(ref.to64(w), group)
    packed, scales = ref.pack_codes(q, s, group)
    assert torch.equal(got.packed.cpu(), packed) and torch.equal(got.scales.cpu().view(torch.int16), scales.view(torch.int16))
    values = q * np.repeat(s, group, 1)[:, :k]
    for out in TYPES:
        v = torch.from_numpy(values).to(F32)  # exact: 4 and 8 bits
        assert torch.equal(ops.q4_unpack(got, out).cpu(), v.to(out))


def test_packing_special_values_and_strides(ops):
    inf, nan = float("inf"), float("nan")
    for group in (32, 64, 128):
        x = rng(3, group).standard_normal((20, 290))
        x[1] = 0
        x[2] = np.abs(x[2])
        x[3] = -np.abs(x[3])
        x[4, 3], x[5, 289], x[6, 200] = inf, -inf, nan
        x[7] *= 1e-40
        x[8] *= 1e37
        x[9] = 3.4e38
        x[10, ::2] = -7
        x[10, 1::2] = 6.5  # scale 13/14 rounded to BF16
        x[11] = np.arange(290) % 16 / 2 - 3.5  # halves of a scale that is a power of two
        x[11, ::32] = 3.5
        t = tensor(x)
        q, s = ref.codes4(ref.to64(t), group)
        packed, scales = ref.pack_codes(q, s, group)
        got = ops.q4_pack(t, group)
        assert torch.equal(got.packed.cpu(), packed)
        a, b = got.scales.cpu().float().numpy(), scales.float().numpy()
        assert np.array_equal(a, b, equal_nan=True)
        wide = torch.full((20, 310), 7.0, device="cuda")
        wide[:, 5:295] = t
        again = ops.q4_pack(wide[:, 5:295], group)
        assert torch.equal(again.packed, got.packed)
        out = torch.full((20, 310), 5.0, dtype=BF16, device="cuda")
        ops.q4_unpack(got, BF16, out=out[:, 4:294])
        assert torch.equal(out[:, 4:294].nan_to_num(), ops.q4_unpack(got, BF16).nan_to_num())
        assert bool((out[:, :4] == 5).all()) and bool((out[:, 294:] == 5).all())


# ------------------------------------------------------------------ products
SIZES = [(1, 1, 1), (1, 16, 128), (1, 1024, 2048), (2, 17, 129), (3, 100, 260), (4, 64, 1280), (5, 33, 700), (8, 130, 384), (9, 48, 640), (16, 50, 1024),
         (17, 96, 300), (33, 70, 520), (64, 130, 256), (65, 40, 1100), (100, 257, 130), (129, 320, 700), (257, 66, 2050), (1, 2, 9000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_products_match_the_definition(ops, rows, n, k, group, dtype):
    r = rng(rows, n, k, group)
    w, qw, sw = weight_of(ops, r, n, k, group)
    q, sx = codes_of(r, rows, k, group)
    tq, ts = torch.from_numpy(q).cuda(), torch.from_numpy(sx).cuda()
    out = ops.q4_matmul(tq, ts, w, out_dtype=dtype)
    v, e = ref.product(q, sx, qw, sw, group)
    ref.check_product(out, v, e, "bare")
    bias, res = r.standard_normal(n).astype(np.float32), r.standard_normal((rows, n))
    tres = tensor(res, dtype)
    out = ops.q4_matmul(tq, ts, w, bias=tensor(bias), residual=tres, out_dtype=dtype)
    v, e = ref.product(q, sx, qw, sw, group, bias=bias.astype(np.float64), residual=ref.to64(tres))
    ref.check_product(out, v, e, "bias and residual")
    same = tres.clone()
    assert ops.q4_matmul(tq, ts, w, bias=tensor(bias), residual=same, out_dtype=dtype, out=same) is same and torch.equal(same, out)
    if n % 2 == 0:
        tres = tensor(res[:, : n // 2], dtype)
        out = ops.q4_matmul(tq, ts, w, bias=tensor(bias), residual=tres, swiglu=True, out_dtype=dtype)
        v, e = ref.product(q, sx, qw, sw, group, bias=bias.astype(np.float64), swiglu=True, residual=ref.to64(tres))
        ref.check_product(out, v, e, "SwiGLU")


@pytest.mark.parametrize("rows", [1, 4, 20, 80])
def test_products_of_extreme_codes_are_exact(ops, rows):
    """Every code at its end: group sums of up to 128 * 128 * 8 stay integers."""
    for group in (32, 64, 128):
        n, k = 40, 512
        qw = np.full((n, k), -8)
        qw[1::2] = 7
        packed, scales = ref.pack_codes(qw, np.ones((n, 512 // group), np.float32), group)
        w = ops.Q4Weight(packed.cuda(), scales.cuda(), n, k, group)
        q = np.full((rows, k), -128, np.int8)
        q[::2] = 127
        out = ops.q4_matmul(torch.from_numpy(q).cuda(), torch.ones(rows, k // group, device="cuda"), w)
        assert np.array_equal(ref.to64(out), q.astype(np.float64) @ qw.T)


@pytest.mark.parametrize("rows", [1, 3, 7, 18, 70, 130])
def test_products_write_only_their_rows_and_columns(ops, rows):
    r = rng(rows)
    n, k, group = 50, 300, 64
    w, qw, sw = weight_of(ops, r, n, k, group)
    q, sx = codes_of(r, rows, k, group)
    tq, ts = torch.from_numpy(q).cuda(), torch.from_numpy(sx).cuda()
    for dtype in TYPES:
        for swiglu in (False, True):
            cols = n // 2 if swiglu else n
            wide = torch.full((rows + 4, cols + 9), 3.0, dtype=dtype, device="cuda")
            res = tensor(r.standard_normal((rows, cols + 5)), dtype)[:, 5:]
            out = ops.q4_matmul(tq, ts, w, residual=res, swiglu=swiglu, out_dtype=dtype, out=wide[2 : 2 + rows, 3 : 3 + cols])
            assert torch.equal(out, ops.q4_matmul(tq, ts, w, residual=res.contiguous(), swiglu=swiglu, out_dtype=dtype))
            out.fill_(3.0)
            assert bool((wide == 3).all())


@pytest.mark.parametrize("rows", [1, 6, 40, 100])
def test_a_row_that_is_not_finite_spoils_no_other(ops, rows):
    r = rng(rows, 5)
    n, k, group = 64, 400, 128
    w, qw, sw = weight_of(ops, r, n, k, group)
    x = r.standard_normal((rows, k))
    clean = ops.q4_linear(tensor(x), w)
    x[rows // 2, 17] = np.inf
    out = ops.q4_linear(tensor(x), w)
    keep = [i for i in range(rows) if i != rows // 2]
    assert bool(out[rows // 2].isnan().all()) and torch.equal(out[keep], clean[keep])
    s = w.scales.clone()
    s[1, 0, 3] = float("nan")  # weight row 19
    out = ops.q4_linear(tensor(r.standard_normal((rows, k))), w._replace(scales=s))
    bad = torch.zeros(n, dtype=torch.bool)
    bad[19] = True
    assert torch.equal(out.isnan().cpu(), bad.expand(rows, n))


# ------------------------------------------------------------------ norm and product in one call
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(1, 64, 1024), (1, 130, 200), (2, 4096, 1024), (3, 66, 2050), (4, 34, 1280), (5, 18, 96), (8, 40, 512), (40, 100, 300), (1, 48, 9001), (130, 64, 256)])
def test_linear_is_norm_then_product(ops, rows, n, k, group, dtype):
    """Bit for bit the two calls' result; with any of the epilogues."""
    r = rng(rows, n, k, group)
    w, _, _ = weight_of(ops, r, n, k, group)
    x = tensor(r.standard_normal((rows, k)) * (1 + 10 * (r.random(k) < 0.02)), dtype)
    nw = tensor(1 + 0.1 * r.standard_normal(k), dtype if group != 32 else F32)
    bias = tensor(r.standard_normal(n))
    for norm in (nw, None):
        eight = ops.rmsnorm_q8(x, norm, 1e-5, group=group) if norm is not None else ops.q8_quantize(x, group)
        for out_dtype in (dtype, F32):
            res = tensor(r.standard_normal((rows, n)), out_dtype)
            a = ops.q4_linear(x, w, norm_weight=norm, eps=1e-5, bias=bias, residual=res, out_dtype=out_dtype)
            b = ops.q4_matmul(eight.q, eight.scales, w, bias=bias, residual=res, out_dtype=out_dtype)
            assert torch.equal(a, b)
        a = ops.q4_linear(x, w, norm_weight=norm, eps=1e-5, swiglu=True)
        assert torch.equal(a, ops.q4_matmul(eight.q, eight.scales, w, swiglu=True, out_dtype=dtype))


def test_linear_may_add_to_its_own_rows(ops):
    """A residual stream updated in place by an output projection that reads other rows."""
    for rows in (1, 3, 30):
        r = rng(rows, 77)
        w, _, _ = weight_of(ops, r, 256, 512, 128)
        x, h = tensor(r.standard_normal((rows, 512))), tensor(r.standard_normal((rows, 256)))
        want = ops.q4_linear(x, w, residual=h)
        assert torch.equal(ops.q4_linear(x, w, residual=h, out=h), want)


def test_outputs_over_inputs(itts, ops):
    """A product over its own rows is refused; columns of one wider matrix are apart."""
    r = rng(31)
    w, _, _ = weight_of(ops, r, 256, 256, 128)
    for rows in (1, 3, 40):
        x = tensor(r.standard_normal((rows, 256)))
        with pytest.raises(itts.InvalidArgument, match="overlaps"):
            ops.q4_linear(x, w, out=x)
        wide = torch.zeros(rows, 600, device="cuda")
        wide[:, 300:556] = x
        got = ops.q4_linear(wide[:, 300:556], w, out=wide[:, 20:276])
        assert torch.equal(got, ops.q4_linear(x, w)) and torch.equal(wide[:, 300:556], x)
        with pytest.raises(itts.InvalidArgument, match="overlaps"):
            ops.rmsnorm_q8(x, torch.ones(256, device="cuda"), residual=x.clone(), values=x)
    with pytest.raises(itts.InvalidArgument, match="negated"):
        ops.q8_quantize(torch._neg_view(torch.zeros(2, 64, device="cuda")))
    a, b = torch.ones(2, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda")
    with pytest.raises(itts.InvalidArgument, match="no gradients"):
        ops.rmsnorm_q8(a, b)
    with torch.no_grad():
        ops.rmsnorm_q8(a, b)


def test_outputs_over_weights_and_scales(itts, ops):
    """The same for the tensors beside the rows; a scale matrix as wide as the product is one of them."""
    w, _, _ = weight_of(ops, rng(32), 2, 256, 128)
    norm, bias = torch.ones(256, device="cuda"), torch.ones(2, device="cuda")
    eight = ops.q8_quantize(tensor(rng(33).standard_normal((1, 256))), 128)
    with pytest.raises(itts.InvalidArgument, match="overlaps"):
        ops.q4_matmul(eight.q, eight.scales, w, out=eight.scales)
    with pytest.raises(itts.InvalidArgument, match="overlaps"):
        ops.q4_matmul(eight.q, eight.scales, w, bias=bias, out=bias[None])
    with pytest.raises(itts.InvalidArgument, match="overlaps"):
        ops.q4_linear(torch.ones(1, 256, device="cuda"), w, norm_weight=norm, out=norm[None, :2])
    with pytest.raises(itts.InvalidArgument, match="overlaps"):
        ops.rmsnorm_q8(torch.ones(1, 256, device="cuda"), norm, h=norm[None])


def test_autograd_sees_given_outputs_change(itts, ops):
    """A tensor that a backward pass keeps may not be written unseen; one of inference mode only in it."""
    w, _, _ = weight_of(ops, rng(34), 256, 256, 128)
    x, norm = tensor(rng(35).standard_normal((3, 256))), torch.ones(256, device="cuda")
    eight = ops.rmsnorm_q8(x, norm, values=True)
    outs = {
        "q4_matmul": lambda o: ops.q4_matmul(eight.q, eight.scales, w, out=o),
        "q4_linear": lambda o: ops.q4_linear(x, w, out=o),
        "h": lambda o: ops.rmsnorm_q8(x, norm, h=o),
        "values": lambda o: ops.q8_quantize(x, values=o),
    }
    for name, call in outs.items():
        kept, leaf = torch.ones(3, 256, device="cuda"), torch.ones(3, 256, device="cuda", requires_grad=True)
        loss = (leaf * kept).sum()
        with torch.no_grad():
            call(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            mine = torch.ones(3, 256, device="cuda")
            call(mine)
        assert torch.equal(mine, kept), name
        with pytest.raises(itts.InvalidArgument, match="inference mode"):
            call(mine)
    for t in (eight.q, eight.scales, x):
        before = t._version
        ops.rmsnorm_q8(x, norm, h=x, q=eight.q, scales=eight.scales)
        assert t._version == before + 1
    full = ops.q4_unpack(w)
    before = full._version
    ops.q4_unpack(w, out=full)
    assert full._version == before + 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 8, 67, 136, 1283])
def test_rows_at_any_address(ops, cols, dtype):
    """Rows that begin at each of eight places in 16 bytes, and at another one each: the bits of aligned
    ones, and not an element around them changed."""
    r = rng(cols, 5)
    x, res = (tensor(r.standard_normal((21, cols)), dtype) for _ in range(2))
    w = tensor(1 + 0.1 * r.standard_normal(cols), dtype)
    pad = -(-cols // 8) * 8
    want = ops.rmsnorm_q8(x, w, residual=res, values=True)
    packed = ops.q4_pack(x, 32)
    eight = ops.q8_quantize(tensor(r.standard_normal((40, 64))), 64)
    columns = ops.q4_pack(tensor(r.standard_normal((cols, 64))), 64)
    bias = tensor(r.standard_normal((40, cols)), dtype)
    products = {rows: ops.q4_matmul(eight.q[:rows], eight.scales[:rows], columns, residual=bias[:rows], out_dtype=dtype) for rows in (3, 9, 40)}
    full = ops.q4_unpack(packed, dtype)
    for at in range(8):
        for stride in (pad + 16, pad + 17):

            def place(t=None, rows=21):
                whole = torch.full((rows + 1, stride), 7.0, dtype=dtype, device="cuda")
                part = torch.as_strided(whole, (rows, cols), (stride, 1), at)
                if t is not None:
                    part.copy_(t)
                return whole, part

            def only(whole, part, value):
                assert torch.equal(part, value), (at, stride)
                part.fill_(7.0)
                assert torch.equal(whole, torch.full_like(whole, 7.0)), (at, stride)

            px, pr, (wh, ph), (wv, pv) = place(x)[1], place(res)[1], place(), place()
            weight = torch.as_strided(place(w.expand(21, cols))[0], (cols,), (1,), at)
            got = ops.rmsnorm_q8(px, weight, residual=pr, h=ph, values=pv)
            assert torch.equal(got.q, want.q) and torch.equal(got.scales, want.scales)
            only(wh, ph, want.h)
            only(wv, pv, want.values)
            again = ops.q4_pack(px, 32)
            assert torch.equal(again.packed, packed.packed) and torch.equal(again.scales, packed.scales)
            wo, po = place()
            ops.q4_unpack(packed, dtype, out=po)
            only(wo, po, full)
            for rows, product in products.items():
                wo, po = place(rows=rows)
                ops.q4_matmul(eight.q[:rows], eight.scales[:rows], columns, residual=place(bias[:rows], rows)[1], out_dtype=dtype, out=po)
                only(wo, po, product)
            one = ops.q4_linear(px[:1], ops.Q4Weight(*ops.q4_pack(x, 128)), norm_weight=weight)
            assert torch.equal(one, ops.q4_linear(x[:1], ops.q4_pack(x, 128), norm_weight=w))


# ------------------------------------------------------------------ a layer's run of them
def layer(ops, x, r_in, ws, nws, dtype):
    a = ops.rmsnorm_q8(x, nws[0], 1e-6, residual=r_in)
    qkv = ops.q4_matmul(a.q, a.scales, ws[0], out_dtype=dtype)
    mix = ops.q4_linear(qkv[:, : ws[1].k], ws[1], residual=a.h)
    ff = ops.q4_linear(mix, ws[2], norm_weight=nws[1], swiglu=True)
    return ops.q4_linear(ff, ws[3], residual=mix)


def layer_parts(ops, r, dtype, group=128):
    d, f = 256, 384
    ws = [ops.q4_pack(tensor(0.05 * r.standard_normal(s)), group) for s in ((3 * d, d), (d, d), (2 * f, d), (d, f))]
    return ws, [tensor(1 + 0.1 * r.standard_normal(d), dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 50])
def test_a_layer_of_them_matches_the_definition(ops, rows, dtype):
    """Norm, projections, SwiGLU and residuals as a decoder layer runs them, each step's output against the
    definition on that step's inputs."""
    r = rng(rows, 4)
    ws, nws = layer_parts(ops, r, dtype)
    vals = [ref.codes4(ref.to64(ops.q4_unpack(w)), 128) for w in ws]
    for w, (q, s) in zip(ws, vals):
        assert np.array_equal(q * np.repeat(s, 128, 1)[:, : w.k], ref.to64(ops.q4_unpack(w)))
    x, res = tensor(r.standard_normal((rows, 256)), dtype), tensor(r.standard_normal((rows, 256)), dtype)

    def linear(t, i, norm=None, **kw):
        y = ref.to64(t) if norm is None else ref.rms(ref.to64(t), ref.to64(norm), float(np.float32(1e-6)))
        quot, s = ref.codes8(y, 128)
        return ref.product(np.clip(np.rint(quot), -127, 127), s, *vals[i], 128, **kw)

    a = ops.rmsnorm_q8(x, nws[0], 1e-6, residual=res)
    ref.check_codes(a.q, a.scales, ref.rms(ref.to64(a.h), ref.to64(nws[0]), float(np.float32(1e-6))), 128)
    qkv = ops.q4_matmul(a.q, a.scales, ws[0], out_dtype=dtype)
    ref.check_product(qkv, *ref.product(a.q.cpu().numpy(), a.scales.cpu().numpy(), *vals[0], 128), "qkv")
    part = qkv[:, :256]
    mix = ops.q4_linear(part, ws[1], residual=a.h)
    ref.check_product(mix, *linear(part, 1, residual=ref.to64(a.h)), "output projection")
    ff = ops.q4_linear(mix, ws[2], norm_weight=nws[1], swiglu=True)
    ref.check_product(ff, *linear(mix, 2, norm=nws[1], swiglu=True), "gate and up")
    out = ops.q4_linear(ff, ws[3], residual=mix)
    ref.check_product(out, *linear(ff, 3, residual=ref.to64(mix)), "down")
    assert torch.equal(out, layer(ops, x, res, ws, nws, dtype))


@pytest.mark.parametrize("rows", [1, 40])
def test_a_layer_captured_and_replayed(ops, rows):
    """Two graphs of the same layer on inputs of their own, replayed in turn with eager work between, equal the
    eager results each time."""
    r = rng(rows, 8)
    ws, nws = layer_parts(ops, r, BF16)
    xs = [tensor(r.standard_normal((rows, 256)), BF16) for _ in range(2)]
    rs = [tensor(r.standard_normal((rows, 256)), BF16) for _ in range(2)]
    graphs, outs = [], []
    for x, s in zip(xs, rs):
        layer(ops, x, s, ws, nws, BF16)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(ops, x, s, ws, nws, BF16))
        graphs.append(g)
    for i in range(4):
        for x in xs:
            x.copy_(tensor(r.standard_normal((rows, 256)), BF16))
        want = [layer(ops, x, s, ws, nws, BF16) for x, s in zip(xs, rs)]
        for k in ((0, 1) if i % 2 else (1, 0)):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k], want[k]), (i, k)


def test_streams_at_once_give_the_same_bits(ops):
    """The same calls on two streams at once, and on a stream other than the one that made the tensors."""
    r = rng(12)
    ws, nws = layer_parts(ops, r, F32)
    for rows in (1, 33):
        x, s = tensor(r.standard_normal((rows, 256))), tensor(r.standard_normal((rows, 256)))
        want = layer(ops, x, s, ws, nws, F32)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for _ in range(3):
            for st in streams:
                with torch.cuda.stream(st):
                    got.append(layer(ops, x, s, ws, nws, F32))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_few_rows_give_each_row_its_own_bits(ops):
    """Batches of up to 16 rows: a row's result does not depend on its batch."""
    r = rng(15)
    for n, k, group in ((4096, 1024, 128), (100, 2048, 32), (8194, 1280, 64)):
        w, _, _ = weight_of(ops, r, n, k, group)
        x = tensor(r.standard_normal((16, k)))
        nw = tensor(1 + 0.1 * r.standard_normal(k))
        one = torch.cat([ops.q4_linear(x[i : i + 1], w, norm_weight=nw) for i in range(16)])
        for m in (2, 4, 5, 8, 13, 16):
            assert torch.equal(ops.q4_linear(x[:m], w, norm_weight=nw), one[:m]), (n, m)


def test_no_rows_and_one_column(ops):
    w = ops.q4_pack(torch.ones(5, 3, device="cuda"), 64)
    empty = torch.empty(0, 3, device="cuda")
    q = ops.q8_quantize(empty, 64, values=True)
    assert q.q.shape == (0, 128) and q.scales.shape == (0, 2) and q.values.shape == (0, 3)
    assert ops.rmsnorm_q8(empty, torch.ones(3, device="cuda"), residual=empty).h.shape == (0, 3)
    assert ops.q4_matmul(q.q, q.scales, w).shape == (0, 5) and ops.q4_linear(empty, w).shape == (0, 5)
    # ones are 8 codes of 1 / 7 rounded to BF16 away from 7 steps
    one = ops.q4_linear(torch.ones(1, 3, device="cuda"), w)
    step = ref.bf16(np.array([1 / 7]))[0]
    assert torch.allclose(one.cpu(), torch.full((1, 5), float(3 * min(7, round(1 / step)) * step)), rtol=1e-6)
