"""The encoder operators from their definitions in 64 bits, and what rounding may cost them."""
import numpy as np
import torch

#: half a unit in the last place of each type relative to the value: 2^-p at p significant bits (24, 8 and 11)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = UNIT[torch.float32]
#: smallest normal of each type: below it, rounding errs by a unit of that
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14}


def random_words(counter, key):
    """Philox4x32-10 on Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def element_words(first, count, seed, offset):
    """The words of elements first .. first + count - 1, as numpy uint32."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    g = np.arange(first // 4, (first + count + 3) // 4, dtype=u)
    c = [g & low, g >> u(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    for r in range(10):
        k = [u(((seed & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k[0], b & low, (a >> u(32)) ^ c[3] ^ k[1], a & low]
    return np.stack(c, 1).reshape(-1)[first % 4:first % 4 + count].astype(np.uint32)


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    return torch.from_numpy(element_words(0, n, seed, offset).astype(np.int64) >= round(p * 2 ** 32)).reshape(shape)


def dropped(x, p, seed, offset, residual=None, scale=None):
    """Bit for bit what the operator returns: a product in fp32, a sum in fp32, one rounding."""
    scale = np.float32((1 / (1 - p) if p < 1 else 0) if scale is None else scale)
    y = torch.where(keep_mask(x.shape, p, seed, offset), x.float() * torch.tensor(scale), torch.zeros(()))
    return (y if residual is None else residual.float() + y).to(x.dtype)


def norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * (1 if weight is None else weight.double()) + (0 if bias is None else bias.double())
    return y, xh, rstd


def norm_backward(dy, xh, rstd, weight):
    dy = dy.double()
    g = dy * (1 if weight is None else weight.double())
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def _depth(c):
    return max(16, -(-c // 1024)) + 12      # additions that a term of a row's sum goes through


def norm_bound(x, xh, rstd, weight, bias, y, dtype):
    """Rounding of the result, and of the statistics: a row's sums err by their depth in units of the sum of absolute values."""
    w = torch.ones(()).double() if weight is None else weight.double().abs()
    b = torch.zeros(()).double() if bias is None else bias.double().abs()
    off = F32 * (_depth(x.shape[1]) * rstd * x.double().abs().mean(1, keepdim=True) + (_depth(x.shape[1]) + 8) * xh.abs())
    return UNIT[dtype] * y.abs() + w * off + 4 * F32 * (b + y.abs()) + TINY[dtype]


def norm_backward_bound(x, dy, xh, rstd, weight, dx, dw, db, dtype, weight_dtype):
    n, c = x.shape
    w = torch.ones(()).double() if weight is None else weight.double().abs()
    g = dy.double().abs() * w
    xh_off = F32 * (_depth(c) * rstd * x.double().abs().mean(1, keepdim=True) + (_depth(c) + 8) * xh.abs())
    mean_g, mean_gx = g.mean(1, keepdim=True), (g * xh.abs()).mean(1, keepdim=True)
    terms = g + mean_g + xh.abs() * mean_gx
    sums_off = F32 * (_depth(c) + 8) * (mean_g + xh.abs() * mean_gx) + xh_off * mean_gx + xh.abs() * (g * xh_off).mean(1, keepdim=True)
    bound_dx = UNIT[dtype] * dx.abs() + rstd * (sums_off + F32 * (_depth(c) + 16) * terms) + TINY[dtype]
    depth = -(-n // 16) + 64                # rows that a workgroup adds one after the other, then the join of the workgroups
    bound_dw = UNIT[weight_dtype] * dw.abs() + (dy.double().abs() * (xh_off + depth * F32 * xh.abs())).sum(0) + TINY[weight_dtype]
    bound_db = UNIT[weight_dtype] * db.abs() + depth * F32 * dy.double().abs().sum(0) + TINY[weight_dtype]
    return bound_dx, bound_dw, bound_db


def assert_within(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its bound at %s: got %r want %r" % (
        what, int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(nan=float("inf")).max()), bad.nonzero()[0].tolist(),
        got[tuple(bad.nonzero()[0])].item(), want[tuple(bad.nonzero()[0])].item())


# ---- differential attention ----
def seen_keys(batch, queries, keys, causal=False, lengths=None, starts=None, key_mask=None):
    """bool (batch, queries, keys)"""
    j, i = torch.arange(keys), torch.arange(queries)
    seen = torch.ones(batch, queries, keys, dtype=torch.bool)
    if lengths is not None:
        seen &= (j[None] < lengths.long().clamp(0, keys)[:, None])[:, None]
    if key_mask is not None:
        seen &= key_mask[:, None]
    if causal:
        first = torch.full((batch,), keys - queries) if starts is None else starts.long()
        seen &= j[None, None] <= i[None, :, None] + first[:, None, None]
    return seen


class Attention:
    """Outputs, gradients and what rounding may cost them, in 64 bits.

    Scores are sums of d products of the operands as they are, exponentials of them err by the scores' absolute error, and a row's
    normaliser by as much again.  In 16-bit types probabilities, score gradients and the results handed to the backward are rounded to the type."""

    def __init__(self, q, k, v, lam, seen, scale=None, dout=None):
        dtype, group = q.dtype, q.shape[2] // max(1, k.shape[2])
        unit = UNIT[dtype] if dtype != torch.float32 else 0.0
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0    # half the spacing of its subnormal numbers
        self.dtype = dtype
        d, keys = q.shape[-1], k.shape[1]
        scale = d ** -0.5 if scale is None else scale
        live = seen.any(1)                                      # (batch, keys): what no query sees may hold anything
        k = torch.where(live[:, :, None, None, None], k, torch.zeros((), dtype=dtype))
        v = torch.where(live[:, :, None, None], v, torch.zeros((), dtype=dtype))
        q, k, v = q.double().permute(3, 0, 2, 1, 4), k.double().permute(3, 0, 2, 1, 4), v.double().permute(0, 2, 1, 3)
        k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 1)
        seen = seen[:, None]
        w = lam.double()[None, :, None, None]
        s = (q @ k.transpose(-1, -2)) * scale                   # (map, batch, head, query, key)
        masked = torch.where(seen, s, torch.tensor(-float("inf"), dtype=torch.float64))
        p = torch.nan_to_num(torch.softmax(masked, -1), nan=0.0) if keys else masked
        o = p @ v
        out = o[0] - w * o[1]
        self.out = out.transpose(1, 2)
        # errors
        off = F32 * ((d + 8) * scale * (q.abs() @ k.abs().transpose(-1, -2)) + 8 * s.abs())
        off = torch.where(seen, off, torch.zeros((), dtype=torch.float64))
        worst = off.amax(-1, keepdim=True) if keys else off.sum(-1, keepdim=True)
        share = off + worst + (keys / 16 + 64) * F32 + unit     # relative, of a probability
        p_off = p * share + tiny * seen
        o_off = p_off @ v.abs()
        out_off = o_off[0] + w.abs() * o_off[1] + 8 * F32 * (o[0].abs() + (w * o[1]).abs())
        self.out_bound = (UNIT[dtype] * out.abs() + out_off + TINY[dtype]).transpose(1, 2)
        if dout is None:
            return
        g = dout.double().transpose(1, 2)
        da = g @ v.transpose(-1, -2)
        delta = (g[None] * o).sum(-1, keepdim=True)
        dp = torch.stack((da, -w * da))
        ds = torch.stack((p[0] * (da - delta[0]), -w * p[1] * (da - delta[1])))
        dq, dk = ds @ k * scale, ds.transpose(-1, -2) @ q * scale
        a = p[0] - w * p[1]
        dv = a.transpose(-1, -2) @ g
        del dp
        dv_size = v.shape[-1]
        da_off = F32 * (dv_size + 8) * (g.abs() @ v.abs().transpose(-1, -2))
        # d1 and d2 from the results as they are kept: rounded to the type
        kept = torch.stack((UNIT[dtype] * (out.abs() + 2 * (w * o[1]).abs()) + out_off + w.abs() * o_off[1], UNIT[dtype] * o[1].abs() + o_off[1]))
        delta_off = (g.abs()[None] * (kept + F32 * (dv_size + 8) * (o.abs() + out.abs()[None]))).sum(-1, keepdim=True)
        size = torch.stack((torch.ones_like(p[0]), w.abs() * torch.ones_like(p[0])))
        diff = torch.stack((da - delta[0], da - delta[1]))
        ds_off = size * (p_off * (diff.abs() + da_off + delta_off) + p * (da_off + delta_off)) + (unit + 16 * F32) * ds.abs() + tiny * seen
        a_off = p_off[0] + w.abs() * p_off[1] + (unit + 4 * F32) * a.abs() + tiny * seen
        rows = (q.shape[-2] * group / 16 + 64) * F32
        dq_off = scale * ((ds_off + (keys / 16 + 64) * F32 * ds.abs()) @ k.abs())
        dk_off = scale * ((ds_off + rows * ds.abs()).transpose(-1, -2) @ q.abs())
        dv_off = (a_off + rows * a.abs()).transpose(-1, -2) @ g.abs()
        heads = lambda t: t.unflatten(-3, (-1, group)).sum(-3) if t.shape[-3] else t        # noqa: E731  (shared heads' gradients)
        final = lambda t, t_off: (t, UNIT[dtype] * t.abs() + t_off + TINY[dtype])           # noqa: E731
        self.dq, self.dq_bound = (t.permute(1, 3, 2, 0, 4) for t in final(dq, dq_off))
        self.dk, self.dk_bound = (t.permute(1, 3, 2, 0, 4) for t in final(heads(dk), heads(dk_off)))
        self.dv, self.dv_bound = (t.transpose(1, 2) for t in final(heads(dv), heads(dv_off)))
        self.dlam = -delta[1].sum((0, 2, 3))
        count = q.shape[1] * q.shape[-2]
        lam_off = delta_off[1].sum((0, 2, 3)) + (count / 1024 + 32) * F32 * delta[1].abs().sum((0, 2, 3))
        self.dlam_bound = UNIT[lam.dtype] * self.dlam.abs() + lam_off + TINY[lam.dtype]
