"""The operators of an encoder layer around the MAM layers, as a training loop and an inference server call them: layer
norm, dropout from a counter-based generator (alone, and joined with the residual and the next norm) and differential
attention; each with its plain form in elementary torch operations.

``own`` selects which of the two ``run`` takes: False the plain forms, in 32 bits and rounded once to the outputs' type,
True the framework's operators.  Sizes are those of the repository's own configurations (ViT-B/16: 64 images x 197 tokens x 768,
MLP of 3072; 256 x 4096 activations, 4096 x 4096 weights) or generic, odd ones among them, and, in ``draw``, anything in between.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5

#: bytes of the largest listed norm or dropout and of the largest token's cache, multiply-adds of the largest attention
MOST_BYTES = 6.8e8
MOST_CACHE = 5.4e8
MOST_PRODUCTS = 1.7e11


def _norm(name, kind, rows, cols, dtype, weights, **more):
    return dict({"name": name, "kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "weights": weights}, **more)


def _attention(name, *sizes):
    return dict({"name": name}, **_attention_sizes(*sizes))


def _attention_sizes(kind, batch, queries, keys, heads, kv_heads, d, dv, dtype, causal, ragged):
    return {"kind": kind, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "d": d, "dv": dv, "dtype": dtype, "causal": causal, "ragged": ragged}


def listed():
    return [
        # one image through one norm of a ViT-B/16: the smallest call, where latency counts
        _norm("norm_one_image", "norm", 197, 768, "f32", "f32"),
        # the norm in front of a half of the layer, 64 images: training step
        _norm("norm_train_vit", "norm_train", 12608, 768, "f32", "f32"),
        # a width that is no multiple of anything, last batch of an epoch, mixed precision with 32-bit weights
        _norm("norm_train_ragged", "norm_train", 4099, 1001, "bf16", "f32"),
        # the widest layers, half precision throughout
        _norm("norm_train_wide", "norm_train", 16384, 4096, "f16", "f16"),
        # dropout on the 256 x 4096 activations of a layer: a small training step
        {"name": "dropout_train", "kind": "dropout_train", "rows": 256, "cols": 4096, "dtype": "f32", "p": 0.1},
        # dropout on the hidden activations of the MLP of 64 images
        {"name": "dropout_train_mlp", "kind": "dropout_train", "rows": 12608, "cols": 3072, "dtype": "bf16", "p": 0.1},
        # the layer's join between its halves, 64 images: dropout of the first half's output, residual, norm of the second
        _norm("join_train_vit", "join_train", 12608, 768, "f32", "f32", p=0.1),
        # the same with a ragged width and half precision
        _norm("join_train_ragged", "join_train", 8191, 1030, "f16", "f16", p=0.25),
        # one token for each of 16 requests over caches of up to 16384 tokens, four query heads to a key head: serving
        _attention("attention_token", "attention", 16, 1, 16384, 16, 4, 64, 128, "bf16", False, True),
        # a prompt of odd length behind what its cache holds, ragged requests
        _attention("attention_prompt", "attention", 3, 1021, 2047, 8, 2, 128, 256, "f16", True, True),
        # attention of a ViT-B/16-shaped layer on 64 images: training step in the framework's own type
        _attention("attention_train_vit", "attention_train", 64, 197, 197, 6, 6, 64, 128, "f32", False, False),
        # long causal sequences in mixed precision: the largest training step
        _attention("attention_train_long", "attention_train", 2, 4096, 4096, 8, 8, 64, 128, "bf16", True, False),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over the logarithm; half of them round, half as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if v >= 512 else 16 if v >= 64 else 4
        v = max(step, v // step * step)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_train", "dropout_train", "dropout_train", "join_train", "join_train",
                       "attention_token", "attention_token", "attention_prompt", "attention_train", "attention_train"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    p = rng.choice([0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    if not kind.startswith("attention"):
        while True:
            case = {"kind": kind, "rows": _size(rng, 1 if kind == "norm" else 64, 32768), "cols": _size(rng, 64, 8192), "dtype": dtype}
            if kind != "dropout_train":
                case["weights"] = rng.choice(["f32", dtype])
            if kind in ("dropout_train", "join_train"):
                case["p"] = p
            if case["cols"] != 3072 and work(case)["bytes"] <= MOST_BYTES:
                return case
    d, kv_heads, group = rng.choice([32, 64, 64, 80, 128]), rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 1, 2, 4])
    dv = rng.choice([d, 2 * d, 2 * d])
    heads = kv_heads * group
    while True:
        if kind == "attention_token":
            batch, keys, queries = _size(rng, 1, 64), _size(rng, 64, 32768), rng.choice([1, 1, 1, 2, 4])
            case = _attention_sizes("attention", batch, queries, keys, heads, kv_heads, d, dv, dtype, queries > 1, rng.random() < 0.5)
            if work(case)["bytes"] <= MOST_CACHE:
                return case
            continue
        batch, keys = _size(rng, 1, 64), _size(rng, 32, 4096)
        queries = keys if rng.random() < 0.7 else _size(rng, 16, keys)
        case = _attention_sizes("attention_train" if kind == "attention_train" else "attention", batch, queries, keys, heads, kv_heads, d, dv,
                                dtype, rng.random() < 0.5, rng.random() < 0.4)
        # in 32 bits the matrix cores take 16 times as long for a product
        if _products(case) <= MOST_PRODUCTS / (16 if dtype == "f32" else 1) and batch * heads * queries * keys <= 2 ** 28:
            return case


# ---- sizes, the same for every seed ----
def _lengths(case):
    """Keys that each request has: all of them, or from all down to half."""
    n, b = case["keys"], case["batch"]
    return [n - (i * n) // (2 * b) if case["ragged"] else n for i in range(b)]


def _pairs(case):
    """(query, key) pairs that are not masked, of one head and all requests."""
    total = 0
    for length in _lengths(case):
        if not case["causal"]:
            total += case["queries"] * length
        else:                                       # query i is the token at length - queries + i
            first = length - case["queries"] + 1    # keys that the first query sees
            total += sum(max(0, first + i) for i in range(case["queries"]))
    return total


def _products(case):
    d, dv = case["d"], case["dv"]
    return _pairs(case) * case["heads"] * (2 * d + 2 * dv + (6 * d + 2 * dv if case["kind"] == "attention_train" else 0))


def work(case):
    kind, e = case["kind"], SIZES[case["dtype"]]
    if kind in ("norm", "norm_train", "join_train", "dropout_train"):
        n, c = case["rows"] * case["cols"], case["cols"]
        moved = {"norm": 2, "norm_train": 5, "join_train": 9, "dropout_train": 4}[kind] * e * n
        ops = {"norm": 8, "norm_train": 22, "join_train": 26, "dropout_train": 2}[kind] * n
        if kind != "dropout_train":
            moved += (2 if kind == "norm" else 5) * SIZES[case["weights"]] * c
        return {"bytes": moved, "flops": ops}
    b, q, h, d, dv = case["batch"], case["queries"], case["heads"], case["d"], case["dv"]
    rows, keys = b * q * h, sum(_lengths(case)) * case["kv_heads"]
    moved = e * (rows * (2 * d + dv) + keys * (2 * d + dv))
    if kind == "attention_train":                   # reads q, k, v, the output's gradient, writes those of q, k, v
        moved += e * (rows * (4 * d + dv) + 2 * keys * (2 * d + dv))
    return {"bytes": moved, "flops": 2 * _products(case)}


# ---- inputs ----
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    state = {"case": case}
    if kind in ("norm", "norm_train", "join_train", "dropout_train"):
        n, c = case["rows"], case["cols"]
        # a residual stream: channels of different means and sizes
        stream = lambda: (normal(n, c) * (0.5 + torch.rand(c, generator=gen, device=DEV)) + 0.3 * normal(c)).to(t)  # noqa: E731
        state["x"] = stream()
        if kind != "dropout_train":
            w = TYPES[case["weights"]]
            state["weight"], state["bias"] = (1 + 0.1 * normal(c)).to(w), (0.1 * normal(c)).to(w)
        if kind != "norm":
            state["dy"] = normal(n, c).to(t)
        if kind == "join_train":
            state["residual"], state["ds"] = stream(), normal(n, c).to(t)
        if "p" in case:
            state["seed"], state["offset"] = seed * 0x9E3779B1 + 12345, seed % 1000
        if kind != "norm":
            for name in ("x", "weight", "bias", "residual"):
                if name in state:
                    state[name].requires_grad_(True)
        return state
    b, q, s, h, hk, d, dv = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "d", "dv"))
    state["q"] = normal(b, q, h, 2, d).to(t)
    state["k"] = normal(b, s, hk, 2, d).to(t)
    state["v"] = normal(b, s, hk, dv).to(t)
    state["lam"] = (0.2 + 0.6 * torch.rand(h, generator=gen, device=DEV)).to(t)
    lengths = _lengths(case)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV) if case["ragged"] else None
    # the queries are the last tokens of their request
    state["starts"] = torch.tensor([n - q for n in lengths], dtype=torch.int32, device=DEV) if case["causal"] else None
    if kind == "attention_train":
        state["dout"] = normal(b, q, h, dv).to(t)
        for name in ("q", "k", "v", "lam"):
            state[name].requires_grad_(True)
    return state


# ---- plain forms ----
def _plain_norm(x, weight, bias):
    x = x.float()
    centred = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xh = centred * r
    return xh * weight.float() + bias.float(), xh, r


def _plain_norm_backward(dy, xh, r, weight):
    dy = dy.float()
    g = dy * weight.float()
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def _plain_keep(n, p, seed, offset):
    """Whether element i is kept: word i % 4 of Philox4x32-10 (J. K. Salmon et al., Parallel random numbers: as easy as
    1, 2, 3, 2011) with counter (i / 4, offset) and key seed is at least p * 2^32.  Every 32-bit word in 64 bits."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, device=DEV)
    c0, c1 = i & low, i >> 32
    c2, c3 = torch.full_like(i, offset & low), torch.full_like(i, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]
    return words >= round(p * 2 ** 32)


def _plain_dropout(x, p, seed, offset):
    keep = _plain_keep(x.numel(), p, seed, offset).view(x.shape)
    return torch.where(keep, x.float() * (1 / (1 - p)), 0.0), keep


def _plain_rows(t, kv_heads):
    """(batch, rows, heads, n) -> (batch, key heads, query heads of each x rows, n)."""
    b, q, h, n = t.shape
    return t.float().reshape(b, q, kv_heads, h // kv_heads, n).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, n)


def _plain_unrows(t, queries):
    b, hk, r, n = t.shape
    return t.view(b, hk, r // queries, queries, n).permute(0, 3, 1, 2, 4).reshape(b, queries, -1, n)


def _plain_attention(state):
    case = state["case"]
    queries, hk = case["queries"], case["kv_heads"]
    q, k, v, lam = (state[n].detach() for n in ("q", "k", "v", "lam"))
    b, s, scale = k.shape[0], k.shape[1], case["d"] ** -0.5
    j = torch.arange(s, device=DEV)
    seen = torch.ones(b, 1, s, dtype=torch.bool, device=DEV)
    if state["lengths"] is not None:
        seen = j[None, None] < state["lengths"][:, None, None]
        k = torch.where(seen[:, 0, :, None, None, None], k, 0)      # what a cache holds past its length may be anything
        v = torch.where(seen[:, 0, :, None, None], v, 0)
    if case["causal"]:
        i = torch.arange(queries, device=DEV)
        seen = seen & (j[None, None] <= i[None, :, None] + state["starts"][:, None, None])
    seen = seen.expand(b, queries if case["causal"] else 1, s)[:, None]
    if case["causal"]:
        seen = seen.repeat(1, 1, case["heads"] // hk, 1)
    qs = torch.stack([_plain_rows(q[..., m, :], hk) for m in (0, 1)])
    ks = torch.stack([k[..., m, :].float().transpose(1, 2).contiguous() for m in (0, 1)])
    vs = v.float().transpose(1, 2).contiguous()
    score = torch.matmul(qs, ks.transpose(-1, -2)) * scale
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)                                                # rows without keys: all 0
    o = torch.matmul(p, vs)
    weight = lam.float().view(1, hk, -1, 1).repeat_interleave(queries, 2)
    out = o[0] - weight * o[1]
    y = _plain_unrows(out, queries).to(q.dtype)
    if case["kind"] != "attention_train":
        return y
    do = _plain_rows(state["dout"], hk)
    da = torch.matmul(do, vs.transpose(-1, -2))
    dv = torch.matmul((p[0] - weight * p[1]).transpose(-1, -2), do)
    delta = (do * o).sum(-1, keepdim=True)
    ds = torch.stack((p[0] * (da - delta[0]), -weight * p[1] * (da - delta[1])))
    dq, dk = torch.matmul(ds, ks) * scale, torch.matmul(ds.transpose(-1, -2), qs) * scale
    dlam = -delta[1].view(b, hk, -1, queries).sum((0, 3)).reshape(-1)
    dq = torch.stack([_plain_unrows(t, queries) for t in dq], 3)
    dk, dv = torch.stack([t.transpose(1, 2) for t in dk], 3), dv.transpose(1, 2)
    return [y] + [t.to(q.dtype).contiguous() for t in (dq, dk, dv, dlam)]


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind.startswith("attention"):
        return _plain_attention(state)
    x = state["x"].detach()
    if kind == "dropout_train":
        y, keep = _plain_dropout(x, case["p"], state["seed"], state["offset"])
        dx = torch.where(keep, state["dy"].float() * (1 / (1 - case["p"])), 0.0)
        return [y.to(x.dtype), dx.to(x.dtype)]
    weight, bias = state["weight"].detach(), state["bias"].detach()
    if kind == "norm":
        return _plain_norm(x, weight, bias)[0].to(x.dtype)
    if kind == "norm_train":
        y, xh, r = _plain_norm(x, weight, bias)
        dx, dw, db = _plain_norm_backward(state["dy"], xh, r, weight)
        return [y.to(x.dtype), dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype)]
    dropped, keep = _plain_dropout(x, case["p"], state["seed"], state["offset"])
    s = (state["residual"].detach().float() + dropped).to(x.dtype)      # the norm is that of the sum as it is handed on
    y, xh, r = _plain_norm(s, weight, bias)
    dx, dw, db = _plain_norm_backward(state["dy"], xh, r, weight)
    dx = dx + state["ds"].float()
    dropped = torch.where(keep, dx * (1 / (1 - case["p"])), 0.0)
    return [y.to(x.dtype), s, dropped.to(x.dtype), dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype)]


# ---- one pass ----
def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    from mamtorch_amd.kernel import encoder

    case, kind = state["case"], state["case"]["kind"]
    grads = torch.autograd.grad
    if kind.startswith("attention"):
        train = kind == "attention_train"
        with torch.set_grad_enabled(train):
            out = encoder.diff_attention(state["q"], state["k"], state["v"], state["lam"], causal=case["causal"], lengths=state["lengths"],
                                         starts=state["starts"])
        return [out.detach(), *grads(out, [state[n] for n in ("q", "k", "v", "lam")], state["dout"])] if train else out
    if kind == "norm":
        with torch.no_grad():
            return encoder.layer_norm(state["x"], state["weight"], state["bias"], EPS)
    if kind == "norm_train":
        y = encoder.layer_norm(state["x"], state["weight"], state["bias"], EPS)
        return [y.detach(), *grads(y, [state[n] for n in ("x", "weight", "bias")], state["dy"])]
    if kind == "dropout_train":
        y = encoder.dropout(state["x"], case["p"], state["seed"], state["offset"])
        return [y.detach(), *grads(y, [state["x"]], state["dy"])]
    y, s = encoder.add_dropout_layer_norm(state["x"], state["residual"], state["weight"], state["bias"], case["p"], state["seed"],
                                          state["offset"], EPS)
    return [y.detach(), s.detach(), *grads([y, s], [state[n] for n in ("x", "residual", "weight", "bias")], [state["dy"], state["ds"]])]


# ---- 64 bits ----
def _exact_keep(n, p, seed, offset):
    """The generator's words in numpy's unsigned 64-bit arithmetic, a row of four for each counter."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    i = np.arange((n + 3) // 4, dtype=u)
    word = [i & low, i >> u(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32 & 0xFFFFFFFF)]
    for r in range(10):
        key = [u((seed + r * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        first, second = word[0] * u(0xD2511F53), word[2] * u(0xCD9E8D57)
        word = [second >> u(32) ^ word[1] ^ key[0], second & low, first >> u(32) ^ word[3] ^ key[1], first & low]
    words = np.stack(word, 1).reshape(-1)[:n]
    return torch.from_numpy(words.astype(np.float64) >= float(round(p * 2 ** 32))).to(DEV)


def _exact_norm(x, dy, weight, bias):
    """y and the gradients; the derivative of the mean and of the variance are followed apart."""
    c = x.shape[1]
    mean = x.sum(1, keepdim=True) / c
    var = ((x - mean) ** 2).sum(1, keepdim=True) / c
    sd = torch.sqrt(var + EPS)
    y = (x - mean) / sd * weight + bias
    if dy is None:
        return y
    g = dy * weight
    dvar = (g * (x - mean)).sum(1, keepdim=True) * -0.5 / sd ** 3
    dmean = -(g / sd).sum(1, keepdim=True)
    dx = g / sd + dvar * 2 * (x - mean) / c + dmean / c
    return y, dx, (dy * (x - mean) / sd).sum(0), dy.sum(0)


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in state.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    with torch.no_grad():
        return _exact(case, state, wide)


def _exact(case, state, wide):
    kind = case["kind"]
    if kind in ("dropout_train", "join_train"):
        keep = _exact_keep(wide["x"].numel(), case["p"], state["seed"], state["offset"]).view(wide["x"].shape).double() / (1 - case["p"])
    if kind == "dropout_train":
        return [wide["x"] * keep, wide["dy"] * keep]
    if kind == "norm":
        return _exact_norm(wide["x"], None, wide["weight"], wide["bias"])
    if kind == "norm_train":
        return list(_exact_norm(wide["x"], wide["dy"], wide["weight"], wide["bias"]))
    if kind == "join_train":
        s = wide["residual"] + wide["x"] * keep
        y, dx, dw, db = _exact_norm(s, wide["dy"], wide["weight"], wide["bias"])
        dx = dx + wide["ds"]
        return [y, s, dx * keep, dx, dw, db]
    return _exact_attention(case, state, wide)


def _exact_attention(case, state, wide):
    """Request by request and head by head, with a softmax over the keys that a query sees."""
    q, k, v, lam = (wide[n] for n in ("q", "k", "v", "lam"))
    train, group, scale = case["kind"] == "attention_train", case["heads"] // case["kv_heads"], 1 / math.sqrt(case["d"])
    out = torch.zeros(q.shape[:3] + v.shape[-1:], dtype=torch.float64, device=DEV)
    dq, dk, dv, dlam = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    lengths = _lengths(case)
    for b in range(case["batch"]):
        n = lengths[b]
        hidden = None
        if case["causal"]:
            at = torch.arange(case["queries"], device=DEV)[:, None] + (n - case["queries"])
            hidden = torch.arange(n, device=DEV)[None] > at
        for hk in range(case["kv_heads"]):
            h = slice(hk * group, (hk + 1) * group)
            qb, kb, vb = q[b, :, h].permute(2, 1, 0, 3), k[b, :n, hk].permute(1, 0, 2), v[b, :n, hk]
            s = torch.matmul(qb, kb[:, None].transpose(-1, -2)) * scale             # (map, head, query, key)
            if hidden is not None:
                s.masked_fill_(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            w = lam[h].view(-1, 1, 1)
            a = p[0] - w * p[1]
            out[b, :, h] = torch.matmul(a, vb).transpose(0, 1)
            if not train:
                continue
            g = wide["dout"][b, :, h].transpose(0, 1)
            dv[b, :n, hk] = torch.matmul(a.transpose(-1, -2), g).sum(0)
            da = torch.matmul(g, vb.T)
            dlam[h] -= (da * p[1]).sum((1, 2))
            dp = torch.stack((da, -w * da))
            ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
            dq[b, :, h] = torch.matmul(ds, kb[:, None]).permute(2, 1, 0, 3)
            dk[b, :n, hk] = torch.matmul(ds.transpose(-1, -2), qb).sum(1).permute(1, 0, 2)
    return [out, dq, dk, dv, dlam] if train else out
