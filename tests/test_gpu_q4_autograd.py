"""What the operators on 4-bit weights and 8-bit activations owe to autograd beyond reverse mode: forward mode is
refused where it would lose a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(itts):
    import itts_ops

    return itts_ops


@pytest.fixture(scope="module")
def calls(ops):
    """Each call by the float tensor that it reads, or writes, beside others of its own."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 256, generator=g, device="cuda")
    one, bias = torch.ones(256, device="cuda"), torch.zeros(256, device="cuda")
    w = ops.q4_pack(x.new_ones(256, 256))
    e = ops.q8_quantize(x)
    return {
        "norm x": (x, lambda t: ops.rmsnorm_q8(t, one).q),
        "norm weight": (one, lambda t: ops.rmsnorm_q8(x, t).q),
        "norm residual": (x, lambda t: ops.rmsnorm_q8(x, one, residual=t).q),
        "norm h": (x, lambda t: ops.rmsnorm_q8(x, one, h=t).q),
        "quantize x": (x, lambda t: ops.q8_quantize(t).q),
        "quantize values": (x, lambda t: ops.q8_quantize(x, values=t).q),
        "pack": (x, lambda t: ops.q4_pack(t).packed),
        "unpack scales": (w.scales, lambda t: ops.q4_unpack(w._replace(scales=t))),
        "unpack out": (x.new_ones(256, 256), lambda t: ops.q4_unpack(w, out=t)),
        "matmul scales": (e.scales, lambda t: ops.q4_matmul(e.q, t, w)),
        "matmul bias": (bias, lambda t: ops.q4_matmul(e.q, e.scales, w, bias=t)),
        "matmul residual": (x, lambda t: ops.q4_matmul(e.q, e.scales, w, residual=t)),
        "linear x": (x, lambda t: ops.q4_linear(t, w)),
        "linear norm": (one, lambda t: ops.q4_linear(x, w, norm_weight=t)),
        "linear out": (x, lambda t: ops.q4_linear(x, w, out=t)),
    }


NAMES = ["norm x", "norm weight", "norm residual", "norm h", "quantize x", "quantize values", "pack", "unpack scales", "unpack out",
         "matmul scales", "matmul bias", "matmul residual", "linear x", "linear norm", "linear out"]


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused_not_dropped(itts, calls, name):
    t, call = calls[name]
    t = t.clone()
    want = call(t.clone())
    with fwd.dual_level():
        dual = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(itts.InvalidArgument, match="no gradients"):
            call(dual)
        with torch.no_grad(), pytest.raises(itts.InvalidArgument, match="no gradients"):
            call(dual)  # (forward mode goes on under no_grad)
        if dual.dim() == 2:
            with pytest.raises(itts.InvalidArgument, match="no gradients"):
                call(dual[:])  # a view has its base's tangent
        # the value alone, and a call where forward mode is off
        assert torch.equal(call(fwd.unpack_dual(dual).primal), want)
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(call(dual), want)
    assert torch.equal(call(t), want)
