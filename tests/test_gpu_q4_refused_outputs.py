"""A call that is refused leaves its outputs as they were, for autograd too: their version, by which a backward pass
knows that what it keeps has changed, counts writes alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_refused_call_counts_no_write(itts):
    import itts_ops as ops

    w = ops.q4_pack(torch.ones(256, 256, device="cuda"))
    one = torch.ones(256, device="cuda")
    x, other, leaf = torch.ones(3, 256, device="cuda"), torch.ones(3, 256, device="cuda"), torch.ones(3, 256, device="cuda", requires_grad=True)
    e = ops.q8_quantize(x)
    wide = torch.ones(3, 300, device="cuda")  # a row stride under its columns, once expanded
    refusals = {
        "norm values over x": (x, "overlaps", lambda: ops.rmsnorm_q8(x, one, residual=other, values=x)),
        "norm h and values": (other, "overlaps", lambda: ops.rmsnorm_q8(x, one, h=other, values=other)),
        "norm eps": (other, "eps", lambda: ops.rmsnorm_q8(x, one, -1.0, h=other)),
        "quantize values over x": (x, "overlaps", lambda: ops.q8_quantize(x, values=x)),
        "quantize q": (e.q, "stride", lambda: ops.q8_quantize(x, q=e.q, values=wide[:1, :256].expand(3, 256))),
        "quantize scales": (e.scales, "stride", lambda: ops.q8_quantize(x, scales=e.scales, values=wide[:1, :256].expand(3, 256))),
        "unpack": (w.scales, "stride", lambda: ops.q4_unpack(w, torch.bfloat16, out=w.scales.view(-1)[: 256].expand(256, 256))),
        "matmul": (wide, "stride", lambda: ops.q4_matmul(e.q, e.scales, w, out=wide[:1, :256].expand(3, 256))),
        "linear": (x, "overlaps", lambda: ops.q4_linear(x, w, out=x)),
        "linear eps": (other, "eps", lambda: ops.q4_linear(x, w, norm_weight=one, eps=-1.0, out=other)),
    }
    for name, (kept, message, call) in refusals.items():
        loss = (leaf * kept).sum() if kept.shape == leaf.shape else None
        before = kept._version
        with torch.no_grad(), pytest.raises(itts.InvalidArgument, match=message):
            call()
        assert kept._version == before, name
        if loss is not None:
            loss.backward()  # (the kept values are those of the forward pass)
    # and one that writes counts one
    before = other._version
    ops.q4_linear(x, w, out=other)
    assert other._version == before + 1
