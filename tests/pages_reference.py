"""Norms with rotation, pages of a cache and attention over them from their definitions, in 64 bits and on the host, and what rounding may cost them."""
import torch

from encoder_reference import F32, TINY, UNIT, Attention

PI2 = 6.283185307179586


# ---- norms with rotation ----
def turned(x, positions, frequencies, interleaved, back=False):
    """Rows (batch, tokens, heads, maps, d) in 64 bits, by pairs."""
    half = 0 if frequencies is None else frequencies.numel()
    y = x.clone()
    if not half:
        return y
    angle = (positions.double()[..., None] * frequencies.double())[:, :, None, None]
    cos, sin = angle.cos(), angle.sin() * (-1 if back else 1)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y[..., a] = x[..., a] * cos[..., i] - x[..., b] * sin[..., i]
        y[..., b] = x[..., a] * sin[..., i] + x[..., b] * cos[..., i]
    return y


def pair_sizes(t, half, interleaved):
    """|a| + |b| of each element's pair, |x| of an element that has none."""
    out = t.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[..., a] = out[..., b] = t[..., a] + t[..., b]
    return out


class Rotation:
    """Results, gradients and bounds of one operand.

    Rounding in fp32: a row's mean square errs by its depth (adds over a lane's terms and the lanes) relative to itself, its root by half of that; the products with the root and the weight,
    and of the rotation, by a few units.  An angle is exact to 2^-24 of half a turn, its sine and cosine to as much and two units: each element of a pair errs by that share of both."""

    def __init__(self, x, weight, positions, frequencies, eps=1e-6, norm=True, interleaved=False, dy=None):
        dtype, d = x.dtype, x.shape[-1]
        half = 0 if frequencies is None else frequencies.numel()
        x = x.double()
        w = torch.ones(d, dtype=torch.float64) if weight is None else weight.double()
        depth = d / 16 + 16
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
        xh = x * r
        off = (depth / 2 + 8) * F32                         # relative, of a normed element
        turn = (PI2 / 2 + 4) * F32
        y = xh * w
        self.y = turned(y, positions, frequencies, interleaved)
        both = pair_sizes(y.abs(), half, interleaved)
        self.y_bound = UNIT[dtype] * self.y.abs() + (off + turn + 4 * F32) * both + TINY[dtype]
        if dy is None:
            return
        g = turned(dy.double(), positions, frequencies, interleaved, back=True)
        g_size = pair_sizes(dy.double().abs(), half, interleaved)
        g_off = (turn + 4 * F32) * g_size
        if not norm:
            self.dx, self.dx_bound = g, UNIT[dtype] * g.abs() + g_off + TINY[dtype]
            return
        gw = g * w
        mean = (gw * xh).mean(-1, keepdim=True)
        self.dx = r * (gw - xh * mean)
        gw_off = g_off * w.abs() + 2 * F32 * gw.abs()
        mean_off = ((gw_off + (depth + off / F32) * F32 * gw.abs()) * xh.abs()).mean(-1, keepdim=True)
        dx_off = r * (gw_off + xh.abs() * (mean_off + 2 * off * mean.abs()) + (off + 4 * F32) * (gw.abs() + xh.abs() * mean.abs()))
        self.dx_bound = UNIT[dtype] * self.dx.abs() + dx_off + TINY[dtype]
        dims = (0, 1, 2, 3)
        rows = x[..., 0].numel()
        weight_type = dtype if weight is None else weight.dtype
        # a lane adds up to rows / 8 of them one after the other (where one workgroup has them all), then the lanes, the waves, the workgroups
        adds = (rows / 8 + 80) * F32
        self.dw = (g * xh).sum(dims)
        self.dw_bound = UNIT[weight_type] * self.dw.abs() + ((g_off + (adds + off) * g.abs()) * xh.abs()).sum(dims) + TINY[weight_type]


# ---- pages ----
class Book:
    """The bookkeeping, request by request on lists."""

    def __init__(self, table, lengths, pages, page):
        self.page, self.pages, self.slots = page, pages, len(table[0]) if table else 0
        self.rows = [[p for p in row if p >= 0] for row in table]
        self.lengths = list(lengths)

    def used(self, n):
        return -(-n // self.page)

    def refs(self):
        held = [0] * self.pages
        for row in self.rows:
            for p in row:
                held[p] += 1
        return held

    def table(self):
        return [row + [-1] * (self.slots - len(row)) for row in self.rows]

    def trim(self, ends):
        for b, n in enumerate(ends):
            n = max(0, min(n, len(self.rows[b]) * self.page))
            self.lengths[b], self.rows[b] = n, self.rows[b][:self.used(n)]

    def fork(self, sources):
        rows, lengths = self.rows, self.lengths
        valid = [0 <= s < len(rows) for s in sources]
        self.rows = [rows[s][:self.used(lengths[s])] if ok else [] for s, ok in zip(sources, valid)]
        self.lengths = [lengths[s] if ok else 0 for s, ok in zip(sources, valid)]

    def extend(self, counts):
        refs = self.refs()
        free, granted, copies = [p for p, n in enumerate(refs) if n == 0], [], []
        for b, count in enumerate(counts):
            row, n = self.rows[b], self.lengths[b]
            granted.append(0)
            copies.append([-1, -1])
            if count <= 0 or n + count > self.slots * self.page:
                continue
            copy = n % self.page > 0 and refs[row[n // self.page]] > 1
            take = max(0, self.used(n + count) - len(row)) + copy
            if take > len(free):
                free = []
                continue
            granted[b] = count
            taken, free = free[:take], free[take:]
            if copy:
                at = n // self.page
                copies[b] = [row[at], taken[0]]
                refs[row[at]] -= 1
                row[at] = taken.pop(0)
            row.extend(taken)
        return granted, copies


def tree(parents):
    """(tokens, tokens): what each drafted token sees."""
    n = len(parents)
    seen = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            seen[i] |= seen[p]
    return seen


def bits(seen):
    """bool (..., n, n) as int64 masks."""
    n = seen.shape[-1]
    return (seen.long() << torch.arange(n)).sum(-1)


# ---- attention over pages ----
def dense(pool, table, tokens):
    """(batch, tokens, key heads, ...) of a pool's pages; tokens without a page are zeros."""
    page, slots = pool.shape[2], table.shape[1]
    out = torch.zeros(table.shape[0], slots * page, pool.shape[1], *pool.shape[3:], dtype=pool.dtype)
    for b in range(table.shape[0]):
        for s in range(slots):
            p = int(table[b, s])
            if 0 <= p < pool.shape[0]:
                out[b, s * page:(s + 1) * page] = pool[p].transpose(0, 1)
    return out[:, :tokens]


class PagesAttention:
    """diff_attention over the pages gathered, with a mask of its own for each query."""

    def __init__(self, q, k_pages, v_pages, table, lengths, lam, scale=None, counts=None, masks=None):
        b, n = q.shape[:2]
        page, slots = k_pages.shape[2], table.shape[1]
        room = slots * page
        lengths = lengths.long().clamp(0, room)
        counts = torch.full((b,), n) if counts is None else counts.long().clamp(0, n)
        keys = min(room, int((lengths + counts).max())) if b else 0
        j, i = torch.arange(keys), torch.arange(n)
        drafted = j[None, None] - lengths[:, None, None]
        if masks is None:
            new = drafted <= i[None, :, None]
        else:
            new = (masks[:, :, None] >> drafted.clamp(0, 63)) & 1 > 0
        there = (table[:, :, None].expand(-1, -1, page).reshape(b, room)[:, :keys])
        there = (there >= 0) & (there < k_pages.shape[0])
        seen = (drafted < 0) | (new & (drafted < counts[:, None, None]))
        seen = seen & there[:, None] & (i[None, :, None] < counts[:, None, None])
        self.seen = seen
        a = Attention(q, dense(k_pages, table, keys), dense(v_pages, table, keys), lam, seen, scale)
        self.out, self.out_bound = a.out, a.out_bound
