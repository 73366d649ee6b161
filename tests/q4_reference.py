"""The operators on 4-bit weights and 8-bit activations in 64 bits, element by element from their
definitions (include/itts_ops.h), on the CPU."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step
NP = torch.float32, torch.bfloat16, torch.float16


def up(v, m):
    return -(-v // m) * m


def to64(t):
    return t.detach().cpu().double().numpy()


def groups_of(y, group):
    """[rows][groups][group], zeros behind the row's end up to a multiple of 128 columns."""
    rows, cols = y.shape
    out = np.zeros((rows, up(cols, 128)))
    out[:, :cols] = y
    return out.reshape(rows, -1, group)


def codes8(y, group):
    """(quotients y / s, scales float32) of rows y; a scale that is not finite is NaN."""
    with np.errstate(all="ignore"):
        g = groups_of(y, group)
        top = np.abs(g).max(2)  # (NaN stays)
        s = (top / 127.0).astype(np.float32)
        s[~np.isfinite(s)] = np.nan
        t = g / s.astype(np.float64)[:, :, None]
        t[~(s > 0)] = 0.0
    return t.reshape(y.shape[0], -1), s


def rms(h, w, eps):
    with np.errstate(all="ignore"):
        return h * w / np.sqrt((h * h).mean(1, keepdims=True) + eps)


def check_codes(q, s, y, group, what=""):
    """Codes and scales are those of y: scales to one float32 step (the quotient by 127 may lie next
    to a border), codes the nearest to y / s for the scale that was given; within 1e-9 of a half (64-bit
    arithmetic of a few operations: 1e-13 of 127) either neighbour."""
    t, ref = codes8(y, group)
    q, s = q.cpu().numpy().astype(np.float64), s.cpu().numpy()
    assert q.shape == t.shape and s.shape == ref.shape, what
    assert np.array_equal(np.isnan(s), np.isnan(ref)), what
    ok = ~np.isnan(ref)
    assert np.all(np.abs(s[ok].astype(np.float64) - ref[ok]) <= np.spacing(ref[ok]).astype(np.float64)), what
    with np.errstate(all="ignore"):
        t = (groups_of(y, group) / s.astype(np.float64)[:, :, None]).reshape(t.shape)
    live = np.repeat(s > 0, group, 1)
    assert np.all(q[~live] == 0), what
    t = np.clip(np.where(live, t, 0.0), -127, 127)
    assert np.all(np.abs(q - t) <= 0.5 + 1e-9), (what, np.abs(q - t).max())
    tie = np.abs(np.abs(t - np.rint(t)) - 0.5) < 1e-9
    assert np.array_equal(q[~tie], np.rint(t)[~tie]), what


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).bfloat16().float().numpy()


def codes4(w, group):
    """(codes int [n][k], scales float32 values of bfloat16 [n][groups]) of a weight matrix."""
    n, k = w.shape
    g = groups_of(w, group)
    in_k = (np.arange(up(k, 128)) < k).reshape(-1, group)
    with np.errstate(all="ignore"):
        top = np.where(in_k, g, -np.inf).max(2)
        low = np.where(in_k, -g, -np.inf).max(2)
        part = ~in_k.all(1)  # columns behind the end count as zeros
        top[:, part] = np.maximum(top[:, part], 0.0)
        low[:, part] = np.maximum(low[:, part], 0.0)
        top[np.isnan(g).any(2)] = np.nan
        s = bf16(np.maximum(top / 7.0, low / 8.0).astype(np.float32))
        s[~np.isfinite(s) | ~np.isfinite(g).all(2)] = np.nan
        t = g / s.astype(np.float64)[:, :, None]
    t = np.where((s > 0)[:, :, None], t, 0.0)
    return np.clip(np.rint(t), -8, 7).reshape(n, -1)[:, :k].astype(np.int64), s


def pack_codes(q, s, group):
    """Codes [n][k] and scales [n][padded groups] as packed bytes and BF16 scales, one by one."""
    n, k = q.shape
    nt, kb = up(n, 16) // 16, up(k, 128) // 128
    out = np.zeros((nt, kb, 1024), np.uint8)
    row, col = np.meshgrid(np.arange(n), np.arange(k), indexing="ij")
    c = col % 128
    byte = 16 * (16 * (c % 32 // 8) + row % 16) + 8 * (c // 64) + c % 8
    np.bitwise_or.at(out, (row // 16, col // 128, byte), ((q & 15) << np.where(c % 64 >= 32, 4, 0)).astype(np.uint8))
    sc = np.zeros((nt * 16, kb * (128 // group)), np.float32)
    sc[:n] = s
    sc = sc.reshape(nt, 16, kb, 128 // group).transpose(0, 2, 1, 3)
    return torch.from_numpy(out), torch.from_numpy(np.ascontiguousarray(sc)).bfloat16()


def product(q, sx, qw, sw, group, bias=None, swiglu=False, residual=None):
    """(result, error bound before the last rounding) of q4_matmul in 64 bits.  The kernels' sums: each of
    the `ng` groups' integers is exact; its product with the two scales' rounded product and the addition
    to the sum are two roundings of 2^-24, the order of the groups any, so a sum is off by at most
    (ng + 2) 2^-24 of the sum of the terms' sizes; one rounding each for the bias and the residual."""
    e = 2.0 ** -24
    rows, n = q.shape[0], qw.shape[0]
    qg = q.reshape(rows, -1, group).astype(np.float64)
    wg = np.zeros((n, q.shape[1]))
    wg[:, : qw.shape[1]] = qw
    wg = wg.reshape(n, -1, group)
    ng = qg.shape[1]
    total, size = np.zeros((rows, n)), np.zeros((rows, n))
    with np.errstate(all="ignore"):
        for g in range(ng):
            term = (qg[:, g] @ wg[:, g].T) * sx[:, g : g + 1].astype(np.float64) * sw[:, g].astype(np.float64)
            total += term
            size += np.abs(term)
        err = (ng + 2) * e * size
        if bias is not None:
            total = total + bias
            err = err + e * (np.abs(total) + err)
        if swiglu:
            g, u, eg, eu = total[:, 0::2], total[:, 1::2], err[:, 0::2], err[:, 1::2]
            sg = g / (1.0 + np.exp(-g))
            total = sg * u
            # |silu'| <= 1.1; exp to 2 steps, sum, quotient and product half a step each: 8 e covers them
            err = 1.1 * eg * (np.abs(u) + eu) + np.abs(sg) * eu + 8 * e * np.abs(total)
        if residual is not None:
            total = total + residual
            err = err + e * (np.abs(total) + err)
    return total, err


def check_product(out, ref, err, what=""):
    """out is ref, to err and one rounding to out's type (for numbers under the type's normal range, its smallest step)."""
    half = HALF[out.dtype]
    tiny = torch.finfo(out.dtype).tiny
    got = to64(out)
    assert got.shape == ref.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    ok = ~np.isnan(ref)
    bound = err[ok] + half * (np.abs(ref[ok]) + err[ok]) + tiny * half
    off = np.abs(got[ok] - ref[ok])
    assert np.all(off <= bound), (what, float(np.max(off / bound)))
