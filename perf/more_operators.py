"""Operators that differential attention with positions needs in training and in serving: norms of queries and keys with the position
rotation in the same pass (its gradient; its serving form, which puts keys and values into a paged cache), the pages of that cache
(room, forks, copies, compaction, release), trees of drafted tokens, and attention over the pages; each with its plain form in
elementary torch operations.

``own`` selects which of the two ``run`` takes: False the plain forms, in 32 bits (angles in 64) and rounded once to the outputs' type,
True the framework's operators.  Sizes are those of the repository's own configurations (ViT-B/16: 64 images x 197 tokens, 6 heads of
two maps of 64) or generic, odd ones among them, and, in ``draw``, anything in between.

Layouts: q (batch, tokens, heads, 2, d), k (batch, tokens, key heads, 2, d), v (batch, tokens, key heads, dv); pages of keys (pages, key
heads, page size, 2, d) and of values (pages, key heads, page size, dv); table (batch, slots) the page that holds tokens slot * page size ..
of a request, -1 where there is none; lengths (batch) its tokens; refs (pages) how many requests hold a page, 0 where it is free.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 10000.0

#: bytes of the largest listed training step and of the largest cache, multiply-adds of the largest attention
MOST_BYTES = 6.8e8
MOST_CACHE = 5.4e8
MOST_PRODUCTS = 6e10


def _heads(heads, kv_heads, d, dv, dtype):
    return {"heads": heads, "kv_heads": kv_heads, "d": d, "dv": dv, "dtype": dtype}


def _rotate(batch, tokens, heads, kv_heads, d, rotary, dtype, weights, interleaved, first):
    """first: the place of the first token; -1: packed sequences, whose places begin anew."""
    return dict(_heads(heads, kv_heads, d, 2 * d, dtype), kind="rotate_train", batch=batch, tokens=tokens, rotary=rotary, weights=weights,
                interleaved=interleaved, first=first)


def _cache(kind, batch, tokens, keys, page, heads, kv_heads, d, dv, dtype, **more):
    """tokens: new ones of each request; keys: what the longest request has in the cache before them."""
    return dict(_heads(heads, kv_heads, d, dv, dtype), kind=kind, batch=batch, tokens=tokens, keys=keys, page=page, **more)


def listed():
    cases = {
        # queries and keys of a ViT-B/16-shaped layer on 64 images, in the framework's own type: training step
        "rotate_train_vit": _rotate(64, 197, 6, 6, 64, 64, "f32", "f32", False, 0),
        # packed documents in mixed precision with 32-bit weights, a head of which three quarters turn, neighbours paired
        "rotate_train_ragged": _rotate(3, 1021, 8, 2, 80, 60, "bf16", "f32", True, -1),
        # long sequences far behind the beginning of their document: the largest training step
        "rotate_train_long": _rotate(2, 8192, 16, 4, 128, 128, "f16", "f16", False, 500000),
        # one token for each of 16 requests, into pages: the smallest call, where latency counts
        "append_token": _cache("append", 16, 1, 1024, 64, 16, 4, 64, 128, "bf16", rotary=64, weights="bf16"),
        # a chunk of a long prompt of odd length
        "append_prompt": _cache("append", 3, 1021, 2047, 32, 8, 2, 128, 256, "f16", rotary=64, weights="f32"),
        # one token for each of 16 requests over caches of up to 16384 tokens, four query heads to a key head
        "attention_token": _cache("attention", 16, 1, 16384, 64, 16, 4, 64, 128, "bf16", tree=False),
        # trees of 32 drafted tokens for 8 requests
        "attention_tree": _cache("attention", 8, 32, 8192, 64, 16, 4, 64, 128, "bf16", tree=True),
        # a chunk of odd length behind a long cache in small pages, large heads
        "attention_chunk": _cache("attention", 2, 509, 4099, 16, 8, 2, 128, 256, "f16", tree=False),
        # a step of beam search for 2 prompts of 4 beams: short caches, 32 bits
        "beams_few": _cache("beams", 8, 1, 300, 16, 6, 6, 64, 128, "f32", group=4),
        # the same for 64 prompts
        "beams_many": _cache("beams", 256, 1, 1021, 64, 8, 2, 128, 256, "f16", group=4),
        # taking over the accepted path of 16 drafted tokens for each of 64 requests
        "accept": _cache("accept", 64, 16, 2000, 64, 16, 4, 64, 128, "bf16"),
        # drafting, appending, attention and taking over for 4 requests, in the framework's own type
        "step_draft": _cache("step", 4, 8, 777, 16, 6, 6, 64, 128, "f32", rotary=64, weights="f32"),
    }
    return [dict({"name": name}, **case) for name, case in cases.items()]


def _size(rng, lo, hi):
    """A size between lo and hi, even over the logarithm; half of them round, half as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 64 if v >= 512 else 16 if v >= 64 else 4
        v = max(step, v // step * step)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["rotate_train", "rotate_train", "append", "append", "attention", "attention", "attention", "beams", "accept", "step"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    d, kv_heads, group = rng.choice([32, 64, 64, 80, 128]), rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 2, 4])
    dv, heads = rng.choice([d, 2 * d, 2 * d]), kv_heads * group
    rotary, weights = rng.choice([d, d, d // 2, d - 4]), rng.choice(["f32", dtype])
    while True:
        if kind == "rotate_train":
            first = rng.choice([0, 0, -1, _size(rng, 1, 1000000)])
            case = _rotate(_size(rng, 1, 64), _size(rng, 32, 8192), heads, kv_heads, d, rotary, dtype, weights, rng.random() < 0.3, first)
            if work(case)["bytes"] <= MOST_BYTES:
                return case
            continue
        page = rng.choice([16, 32, 48, 64, 128])
        if kind == "append":
            case = _cache(kind, _size(rng, 1, 128), rng.choice([1, 1, _size(rng, 2, 2048)]), _size(rng, 16, 4096), page, heads, kv_heads, d, dv, dtype,
                          rotary=rotary, weights=weights)
        elif kind == "attention":
            tree = rng.random() < 0.5
            tokens = rng.randint(2, 64) if tree else rng.choice([1, 1, _size(rng, 2, 1024)])
            case = _cache(kind, _size(rng, 1, 64), tokens, _size(rng, 64, 32768), page, heads, kv_heads, d, dv, dtype, tree=tree)
            # in 32 bits the matrix cores take 16 times as long for a product
            if _products(case) > MOST_PRODUCTS / (16 if dtype == "f32" else 1) or case["batch"] * heads * tokens * case["keys"] > 2 ** 27:
                continue
        elif kind == "beams":
            beams = rng.choice([2, 3, 4, 8])
            case = _cache(kind, beams * _size(rng, 1, 64), 1, _size(rng, 16, 4096), page, heads, kv_heads, d, dv, dtype, group=beams)
        elif kind == "accept":
            case = _cache(kind, _size(rng, 1, 256), rng.randint(2, 64), _size(rng, 16, 4096), page, heads, kv_heads, d, dv, dtype)
        else:
            case = _cache(kind, _size(rng, 1, 32), rng.randint(2, 64), _size(rng, 16, 4096), page, heads, kv_heads, d, dv, dtype, rotary=rotary,
                          weights=weights)
            if _products(case) > MOST_PRODUCTS / 16:
                continue
        if _pages(case) * page * _token_bytes(case) <= MOST_CACHE:
            return case


# ---- sizes, the same for every seed ----
def _lengths(case):
    """Tokens that each request has in the cache: all of them, or from all down to half; beams of one prompt have as many."""
    n, b, g = case["keys"], case["batch"], case.get("group", 1)
    return [n - (i // g * g * n) // (2 * b) for i in range(b)]


def _slots(case):
    return -(-(case["keys"] + case["tokens"]) // case["page"])


def _pages(case):
    """Pages of the pool: what every request may need, and some.  Beams of one prompt have their whole pages in common."""
    p, g = case["page"], case.get("group", 1)
    if g > 1:
        return sum(n // p for n in _lengths(case)[::g]) + 3 * case["batch"] + 3
    return sum(-(-(n + case["tokens"]) // p) for n in _lengths(case)) + case["batch"] + 3


def _token_bytes(case):
    return SIZES[case["dtype"]] * case["kv_heads"] * (2 * case["d"] + case["dv"])


def _products(case):
    """Multiply-adds of both maps' scores and products with the values."""
    n, causal = case["tokens"], not case.get("tree", True)
    pairs = sum(n * length + (n * (n + 1) // 2 if causal else n * n // 4 + n) for length in _lengths(case))
    return pairs * case["heads"] * 2 * (case["d"] + case["dv"])


def work(case):
    kind, e, b, n = case["kind"], SIZES[case["dtype"]], case["batch"], case["tokens"]
    h, hk, d, dv = (case[k] for k in ("heads", "kv_heads", "d", "dv"))
    rows = b * n * 2 * d
    if kind == "rotate_train":                      # reads q, k and the outputs' gradients, writes the outputs and q's and k's gradients
        moved = 5 * e * rows * (h + hk) + 4 * SIZES[case["weights"]] * d + 8 * (case["rotary"] // 2)
        return {"bytes": moved, "flops": 30 * rows * (h + hk)}
    token, table = _token_bytes(case), 4 * b * _slots(case)
    new = b * n * (e * 2 * d * h * 2 + token)       # queries read and written, keys and values read
    if kind == "append":
        return {"bytes": new + b * n * token, "flops": 10 * rows * (h + hk)}
    if kind == "attention":
        return {"bytes": (sum(_lengths(case)) + b * n) * token + b * n * h * e * (2 * d + dv) + table, "flops": 2 * _products(case)}
    refs = 4 * _pages(case)
    if kind == "beams":                             # every beam but one of each prompt whose last page is begun gets a copy of it
        copies = sum(1 for i, length in enumerate(_lengths(case)) if length % case["page"] and (i + 1) % case["group"])
        return {"bytes": 2 * copies * case["page"] * token + 2 * table + 2 * refs, "flops": copies}
    if kind == "accept":
        moved = sum(_accepted(case, i) for i in range(b))
        return {"bytes": 2 * moved * token + 2 * table + refs, "flops": moved}
    attention = (sum(_lengths(case)) + b * n) * token + b * n * h * e * (2 * d + dv)
    return {"bytes": new + b * n * token + attention + 2 * sum(_accepted(case, i) for i in range(b)) * token + 2 * table + refs,
            "flops": 2 * _products(case) + 10 * rows * (h + hk)}


def _accepted(case, request):
    """How many of its drafted tokens a request takes over: one at least, and up to eight."""
    return 1 + (request * 5 + 2) % min(8, case["tokens"])


# ---- inputs ----
def _closure(hop):
    """Reflexive and transitive closure of a relation by squaring six times: paths of up to 64."""
    reach = ((hop + torch.eye(hop.shape[-1], device=DEV)) > 0).float()
    reach = (torch.matmul(reach, reach) > 0).float()
    reach = (torch.matmul(reach, reach) > 0).float()
    reach = (torch.matmul(reach, reach) > 0).float()
    reach = (torch.matmul(reach, reach) > 0).float()
    reach = (torch.matmul(reach, reach) > 0).float()
    return (torch.matmul(reach, reach) > 0).float()


def _plain_tree(parents, lengths):
    """What each drafted token sees of the others, itself and its ancestors, as bits; and its place: as far behind the cache as it is down."""
    b, n = parents.shape
    # node 0 stands above all roots
    node = torch.cat((torch.zeros(b, 1, dtype=torch.long, device=DEV), parents.long() + 1), 1)
    hop = (node[:, :, None] == torch.arange(n + 1, device=DEV)).float()
    seen = _closure(hop)[:, 1:, 1:] > 0
    masks = (seen.long() << torch.arange(n, device=DEV)).sum(-1)
    return masks, (lengths[:, None] + seen.sum(-1) - 1).int()


def _drafts(case, gen):
    """Trees of drafted tokens with a path down from the first one that is taken over: (parents, path, its length)."""
    b, n = case["batch"], case["tokens"]
    accepted = torch.tensor([_accepted(case, i) for i in range(b)], device=DEV)
    rank = torch.rand(b, n, generator=gen, device=DEV)
    rank[:, 0] = -1
    on_path = rank.argsort(1).argsort(1) < accepted[:, None]
    index = torch.arange(n, device=DEV).expand(b, n)
    path = torch.where(on_path, index, n).sort(1).values
    # a token of the path follows the one before it there, any other one some token before itself
    before = torch.cat((torch.full((b, 1), -1, device=DEV), torch.where(on_path, index, -1).cummax(1).values[:, :-1]), 1)
    other = (torch.rand(b, n, generator=gen, device=DEV) * index).long()
    parents = torch.where(on_path, before, other)
    return parents.int(), torch.where(path == n, 0, path).int(), accepted.int()


def _prepare_rotation(case, state, gen):
    w, d, r = TYPES[case["weights"]], case["d"], case["rotary"]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    state["q_weight"], state["k_weight"] = (1 + 0.2 * normal(d)).to(w), (1 + 0.2 * normal(d)).to(w)
    state["frequencies"] = BASE ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float64) / r)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, t = case["kind"], TYPES[case["dtype"]]
    b, n, h, hk, d, dv = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "d", "dv"))
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    # projections: elements of different means and sizes
    project = lambda heads: ((normal(b, n, heads, 2, d) + 0.5 * normal(d)) * (0.5 + torch.rand(heads, 2, 1, generator=gen, device=DEV))).to(t)  # noqa: E731
    state = {"case": case}
    if kind == "rotate_train":
        state["q"], state["k"] = project(h), project(hk)
        _prepare_rotation(case, state, gen)
        state["dq"], state["dk"] = normal(b, n, h, 2, d).to(t), normal(b, n, hk, 2, d).to(t)
        state["positions"] = None
        index = torch.arange(n, device=DEV)
        if case["first"] > 0:
            state["positions"] = (index + case["first"]).int().expand(b, n)
        elif case["first"] < 0:                     # packed sequences of 300 tokens or so
            begins = torch.rand(b, n, generator=gen, device=DEV) < 1 / 300
            state["positions"] = (index - torch.where(begins, index, 0).cummax(1).values).int()
        for name in ("q", "k", "q_weight", "k_weight"):
            state[name].requires_grad_(True)
        return state
    page, pages, slots, lengths = case["page"], _pages(case), _slots(case), torch.tensor(_lengths(case), device=DEV)
    state["k_pages"], state["v_pages"] = normal(pages, hk, page, 2, d).to(t), normal(pages, hk, page, dv).to(t)
    # the pages that are held, in any order; those of whole pages are a group's in common
    room = lengths + (n if kind in ("append", "attention") else 0)
    held, slot, group = -(-room // page), torch.arange(slots, device=DEV), case.get("group", 1)
    own_page = slot < held[:, None]
    if group > 1:
        first = torch.arange(b, device=DEV) % group == 0
        own_page &= first[:, None] | (slot >= (lengths // page)[:, None])
    count = own_page.flatten().cumsum(0).view(b, slots)
    order = torch.randperm(pages, generator=gen, device=DEV)
    table = torch.where(own_page, order[(count - 1).clamp(min=0)], -1)
    if group > 1:
        leader = table.view(b // group, group, slots)[:, :1].expand(-1, group, -1).reshape(b, slots)
        table = torch.where(slot < (lengths // page)[:, None], leader, table)
    state["table"], state["lengths"] = table.int(), lengths.int()
    state["refs"] = torch.bincount(torch.where(table < 0, pages, table).flatten(), minlength=pages + 1)[:pages].int()
    if kind in ("append", "step"):
        state["q"], state["k"], state["v"] = project(h), project(hk), normal(b, n, hk, dv).to(t)
        _prepare_rotation(case, state, gen)
    if kind in ("attention", "step"):
        if kind == "attention":
            state["q"] = normal(b, n, h, 2, d).to(t)
        state["lam"] = (0.2 + 0.6 * torch.rand(h, generator=gen, device=DEV)).to(t)
    if kind in ("accept", "step"):
        state["parents"], state["path"], state["accepted"] = _drafts(case, gen)
        state["start"] = state["lengths"].clone()
        state["drafted"] = torch.full((b,), n, dtype=torch.int32, device=DEV)
    if kind == "attention" and case["tree"]:
        state["masks"] = _plain_tree(_drafts(case, gen)[0], state["lengths"])[0]
    if kind == "beams":                             # the last beam of each prompt goes on in all of them
        index = torch.arange(b, device=DEV)
        state["sources"] = (index // group * group + group - 1).int()
        state["drafted"] = torch.ones(b, dtype=torch.int32, device=DEV)
    return state


# ---- plain forms: norms and rotation ----
def _plain_angles(positions, frequencies):
    """cos and sin (batch, tokens, 1, 1, pairs); angles in 64 bits."""
    angle = positions.double()[:, :, None] * frequencies
    return angle.cos().float()[:, :, None, None], angle.sin().float()[:, :, None, None]


def _plain_turn(x, cos, sin, interleaved):
    """x's first elements turned, as pairs (i, i + half) or (2 i, 2 i + 1)."""
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, c = (turned[..., ::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    a, c = a * cos - c * sin, a * sin + c * cos
    return torch.cat((torch.stack((a, c), -1).flatten(-2) if interleaved else torch.cat((a, c), -1), rest), -1)


def _plain_scale(x):
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_rotate(x, weight, cos, sin, interleaved=False):
    x = x.float()
    return _plain_turn(x * _plain_scale(x) * weight.float(), cos, sin, interleaved)


def _plain_rotate_backward(dy, x, weight, cos, sin, interleaved):
    x, w = x.float(), weight.float()
    r = _plain_scale(x)
    xh, g = x * r, _plain_turn(dy.float(), cos, -sin, interleaved)
    gw = g * w
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum((0, 1, 2, 3))


def _plain_rotate_train(state):
    case, b, n = state["case"], state["case"]["batch"], state["case"]["tokens"]
    q, k, wq, wk = (state[name].detach() for name in ("q", "k", "q_weight", "k_weight"))
    positions = torch.arange(n, device=DEV).expand(b, n) if state["positions"] is None else state["positions"]
    cos, sin = _plain_angles(positions, state["frequencies"])
    y, z = _plain_rotate(q, wq, cos, sin, case["interleaved"]), _plain_rotate(k, wk, cos, sin, case["interleaved"])
    dq, dwq = _plain_rotate_backward(state["dq"], q, wq, cos, sin, case["interleaved"])
    dk, dwk = _plain_rotate_backward(state["dk"], k, wk, cos, sin, case["interleaved"])
    return [t.to(q.dtype) for t in (y, z, dq, dk)] + [t.to(wq.dtype) for t in (dwq, dwk)]


# ---- plain forms: pages ----
def _plain_count(table, pages):
    """How many requests hold each page."""
    return torch.bincount(torch.where(table < 0, pages, table).flatten().long(), minlength=pages + 1)[:pages].int()


def _plain_trim(state, lengths):
    """Requests end at `lengths`; the pages behind are given back."""
    slot = torch.arange(state["table"].shape[1], device=DEV)
    state["table"].copy_(torch.where(slot < -(-lengths.long()[:, None] // state["case"]["page"]), state["table"], -1))
    state["lengths"].copy_(lengths)
    state["refs"].copy_(_plain_count(state["table"], state["refs"].shape[0]))


def _plain_fork(state, sources):
    """Request i goes on from request sources[i]: it holds the pages of that one's tokens too."""
    slot, source = torch.arange(state["table"].shape[1], device=DEV), sources.long()
    lengths = state["lengths"][source]
    table = torch.where(slot < -(-lengths.long()[:, None] // state["case"]["page"]), state["table"][source], -1)
    state["table"].copy_(table)
    state["lengths"].copy_(lengths)
    state["refs"].copy_(_plain_count(table, state["refs"].shape[0]))


def _plain_extend(state, counts):
    """Room for `counts` tokens behind each request, from the free pages of lowest number, in the requests' order.  A begun last page that
    others hold is given up for a new one, but by the last request that holds it.  (How many tokens each has room for; pages to copy: from, to)"""
    page, table, refs = state["case"]["page"], state["table"].long(), state["refs"]
    b, slots = table.shape
    lengths = state["lengths"].long()
    at, begun = lengths // page, lengths % page > 0
    last = torch.where(begun, table.gather(1, at.clamp(max=slots - 1)[:, None])[:, 0], -1)
    same = (last[:, None] == last[None]).tril(-1).sum(1)            # requests before it with that page
    shared = begun & (refs[last.clamp(min=0)] - same > 1)
    held = (table >= 0).sum(1)
    want = (-(-(lengths + counts) // page) - held).clamp(min=0)
    take = want + shared.long()
    until = take.cumsum(0)
    free = refs == 0
    served = (until <= free.sum()) | (take == 0)
    order = (~free).int().sort(stable=True).indices                 # free pages in order, then the others
    slot = torch.arange(slots, device=DEV)
    first = (until - take)[:, None]
    fresh = served[:, None] & (slot >= held[:, None]) & (slot < (held + want)[:, None])
    place = (first + shared[:, None].long() + slot - held[:, None]).clamp(0, order.shape[0] - 1)
    table = torch.where(fresh, order[place], table)
    moved = served & shared
    to = order[first[:, 0].clamp(max=order.shape[0] - 1)]
    copies = torch.stack((torch.where(moved, last, -1), torch.where(moved, to, -1)), 1)
    table = torch.where(moved[:, None] & (slot == at[:, None]), to[:, None], table)
    state["table"].copy_(table)
    state["refs"].copy_(_plain_count(table, refs.shape[0]))
    return torch.where(served, counts, 0), copies.int()


def _plain_copy(state, copies):
    """Pages of copies[:, 0] to copies[:, 1]; none where that is -1."""
    pair = copies[copies[:, 1] >= 0].long()
    state["k_pages"][pair[:, 1]] = state["k_pages"][pair[:, 0]]
    state["v_pages"][pair[:, 1]] = state["v_pages"][pair[:, 0]]


def _plain_places(state, tokens):
    """(page, token of the page) of the tokens that follow the cache's (batch, n)."""
    page, at = state["case"]["page"], state["lengths"].long()[:, None] + tokens
    return state["table"].long().gather(1, at // page), at % page


def _plain_compact(state, path, accepted):
    """The tokens path[:, i] behind the cache, i below `accepted`, stand behind it in this order."""
    n = path.shape[1]
    index = torch.arange(n, device=DEV)
    there = index < accepted[:, None]
    source, at = _plain_places(state, path.long())
    target, to = _plain_places(state, index.expand_as(path))
    state["k_pages"][target[there], :, to[there]] = state["k_pages"][source[there], :, at[there]]
    state["v_pages"][target[there], :, to[there]] = state["v_pages"][source[there], :, at[there]]


def _plain_append(state, positions):
    """Queries normed and turned; keys too, and with the values into the pages behind the cache."""
    case, t = state["case"], state["q"].dtype
    cos, sin = _plain_angles(positions, state["frequencies"])
    page, at = _plain_places(state, torch.arange(case["tokens"], device=DEV).expand(case["batch"], -1))
    state["k_pages"][page, :, at] = _plain_rotate(state["k"], state["k_weight"], cos, sin).to(t)
    state["v_pages"][page, :, at] = state["v"]
    return _plain_rotate(state["q"], state["q_weight"], cos, sin).to(t)


# ---- plain forms: attention ----
def _plain_rows(t, kv_heads):
    """(batch, rows, heads, n) -> (batch, key heads, query heads of each x rows, n)."""
    b, q, h, n = t.shape
    return t.float().reshape(b, q, kv_heads, h // kv_heads, n).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, n)


def _plain_attention(state, q, masks):
    case = state["case"]
    b, n, hk, page = case["batch"], case["tokens"], case["kv_heads"], case["page"]
    table, lengths = state["table"].long(), state["lengths"].long()[:, None, None]
    keys = table.shape[1] * page
    j, i = torch.arange(keys, device=DEV), torch.arange(n, device=DEV)
    seen = j < lengths
    drafted = j - lengths                                           # number of a new token
    if masks is None:
        seen = seen | (drafted <= i[:, None])
    else:
        bits = masks[:, :, None] >> drafted.clamp(0, 63)
        seen = seen | ((drafted >= 0) & (drafted < n) & (bits & 1 > 0))
    there = (j < lengths + n)[:, 0, None, :, None]                  # what a page holds behind its tokens may be anything
    take = table.clamp(min=0)
    k = state["k_pages"][take].transpose(1, 2).reshape(b, hk, keys, 2, -1)
    v = torch.where(there, state["v_pages"][take].transpose(1, 2).reshape(b, hk, keys, -1).float(), 0.0)
    seen = seen[:, None].repeat(1, 1, case["heads"] // hk, 1)
    qs = torch.stack([_plain_rows(q[..., m, :], hk) for m in (0, 1)])
    ks = torch.stack([torch.where(there, k[..., m, :].float(), 0.0) for m in (0, 1)])
    score = torch.where(seen, torch.matmul(qs, ks.transpose(-1, -2)) * case["d"] ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e / torch.where(total == 0, 1.0, total), v)                               # rows without keys: all 0
    out = o[0] - state["lam"].float().view(1, hk, -1, 1).repeat_interleave(n, 2) * o[1]
    return out.view(b, hk, -1, n, out.shape[-1]).permute(0, 3, 1, 2, 4).reshape(b, n, case["heads"], -1).to(q.dtype)


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "rotate_train":
        return _plain_rotate_train(state)
    if kind == "append":
        positions = state["lengths"][:, None] + torch.arange(case["tokens"], device=DEV)
        return [_plain_append(state, positions), state["k_pages"], state["v_pages"]]
    if kind == "attention":
        return _plain_attention(state, state["q"], state.get("masks"))
    if kind == "beams":
        _plain_fork(state, state["sources"])
        granted, copies = _plain_extend(state, state["drafted"])
        _plain_copy(state, copies)
        return [granted, copies, *_held(state)]
    # what an answer that is given up had taken over since is dropped
    _plain_trim(state, state["start"])
    granted, _ = _plain_extend(state, state["drafted"])
    masks, positions = _plain_tree(state["parents"], state["lengths"])
    outs = [granted, masks, positions]
    if kind == "step":
        outs.append(_plain_attention(state, _plain_append(state, positions), masks))
    _plain_compact(state, state["path"], state["accepted"])
    _plain_trim(state, state["lengths"] + state["accepted"])
    return [*outs, *_held(state)]


def _held(state):
    return [state[name] for name in ("table", "lengths", "refs", "k_pages", "v_pages")]


# ---- one pass ----
def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    from mamtorch_amd.kernel import encoder

    case, kind = state["case"], state["case"]["kind"]
    if kind == "rotate_train":
        leaves = [state[name] for name in ("q", "k", "q_weight", "k_weight")]
        outs = encoder.norm_rotate(*leaves, state["frequencies"], state["positions"], EPS, interleaved=case["interleaved"])
        grads = torch.autograd.grad(outs, leaves, [state["dq"], state["dk"]])
        return [outs[0].detach(), outs[1].detach(), *grads]
    with torch.no_grad():
        return _own_serving(encoder, state, case, kind)


def _own_serving(encoder, state, case, kind):
    table, lengths, refs, k_pages, v_pages = _held(state)
    page = case["page"]
    append = lambda positions: encoder.norm_rotate_append(  # noqa: E731
        state["q"], state["k"], state["v"], k_pages, v_pages, table, lengths, state["q_weight"], state["k_weight"], state["frequencies"],
        positions, EPS)
    if kind == "append":
        return [append(None), k_pages, v_pages]
    if kind == "attention":
        return encoder.diff_attention_pages(state["q"], k_pages, v_pages, table, lengths, state["lam"], masks=state.get("masks"))
    if kind == "beams":
        encoder.pages_fork(table, lengths, refs, state["sources"], page)
        granted, copies = encoder.pages_extend(table, lengths, refs, state["drafted"], page)
        encoder.pages_copy(k_pages, v_pages, copies)
        return [granted, copies, *_held(state)]
    encoder.pages_trim(table, lengths, refs, state["start"], page)
    granted, _ = encoder.pages_extend(table, lengths, refs, state["drafted"], page)
    masks, positions = encoder.draft_tree(state["parents"], lengths)
    outs = [granted, masks, positions]
    if kind == "step":
        outs.append(encoder.diff_attention_pages(append(positions), k_pages, v_pages, table, lengths, state["lam"], masks=masks))
    encoder.pages_compact(k_pages, v_pages, table, lengths, state["path"], state["accepted"])
    encoder.pages_trim(table, lengths, refs, lengths + state["accepted"], page)
    return [*outs, *_held(state)]


# ---- 64 bits ----
def _exact_rotate(x, weight, positions, frequencies, interleaved=False):
    """Pairs as complex numbers times exp(i angle)."""
    half = frequencies.shape[0]
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight
    pairs = torch.complex(y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved else torch.complex(y[..., :half], y[..., half:2 * half])
    pairs = pairs * torch.exp(1j * positions.double()[..., None, None, None] * frequencies)
    turned = torch.view_as_real(pairs).flatten(-2) if interleaved else torch.cat((pairs.real, pairs.imag), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _exact_rotate_train(case, state, wide):
    leaves = [wide[name].requires_grad_(True) for name in ("q", "k", "q_weight", "k_weight")]
    positions = state["positions"]
    if positions is None:
        positions = torch.arange(case["tokens"], device=DEV).expand(case["batch"], -1)
    with torch.enable_grad():
        outs = [_exact_rotate(x, w, positions, wide["frequencies"], case["interleaved"]) for x, w in zip(leaves[:2], leaves[2:])]
        grads = torch.autograd.grad(outs, leaves, [wide["dq"], wide["dk"]])
    return [t.detach() for t in outs] + list(grads)


class _ExactPages:
    """The pages' bookkeeping request by request on the host, tokens one after the other."""

    def __init__(self, case, state, wide):
        self.page, self.k, self.v = case["page"], wide["k_pages"], wide["v_pages"]
        self.table, self.lengths = state["table"].tolist(), state["lengths"].tolist()
        self.pages, self.slots = self.k.shape[0], state["table"].shape[1]
        self.table = [[p for p in row if p >= 0] for row in self.table]

    def refs(self):
        held = [0] * self.pages
        for row in self.table:
            for p in row:
                held[p] += 1
        return held

    def trim(self, lengths):
        self.lengths = list(lengths)
        self.table = [row[:-(-n // self.page)] for row, n in zip(self.table, lengths)]

    def fork(self, sources):
        self.table = [list(self.table[s][:-(-self.lengths[s] // self.page)]) for s in sources]
        self.lengths = [self.lengths[s] for s in sources]

    def extend(self, counts):
        refs, granted, copies = self.refs(), [], []
        free = [p for p in range(self.pages) if not refs[p]]
        for row, n, count in zip(self.table, self.lengths, counts):
            copy = n % self.page > 0 and refs[row[n // self.page]] > 1
            take = max(0, -(-(n + count) // self.page) - len(row)) + copy
            copies.append([-1, -1])
            granted.append(count if take <= len(free) else 0)
            if take > len(free):
                free = []
                continue
            taken, free = free[:take], free[take:]
            if copy:
                refs[row[n // self.page]] -= 1
                copies[-1] = [row[n // self.page], taken[0]]
                row[n // self.page] = taken.pop(0)
            row += taken
        return granted, copies

    def place(self, request, token):
        return self.table[request][token // self.page], token % self.page

    def compact(self, path, accepted):
        for b, (row, count) in enumerate(zip(path, accepted)):
            for i in range(count):
                (p, at), (t, to) = self.place(b, self.lengths[b] + row[i]), self.place(b, self.lengths[b] + i)
                self.k[t, :, to], self.v[t, :, to] = self.k[p, :, at], self.v[p, :, at]

    def held(self):
        table = [row + [-1] * (self.slots - len(row)) for row in self.table]
        whole = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in (table, self.lengths, self.refs())]
        return whole + [self.k, self.v]


def _exact_tree(parents, lengths):
    masks, positions = [], []
    for row, length in zip(parents, lengths):
        seen = []
        for i, parent in enumerate(row):
            seen.append(1 << i | (seen[parent] if parent >= 0 else 0))
        masks.append([m - 2 ** 64 if m >> 63 else m for m in seen])
        positions.append([length + bin(m).count("1") - 1 for m in seen])
    return torch.tensor(masks, device=DEV), torch.tensor(positions, dtype=torch.int32, device=DEV)


def _exact_append(case, pages, wide, positions):
    """Queries; keys and values go into the pages."""
    k = _exact_rotate(wide["k"], wide["k_weight"], positions, wide["frequencies"])
    for b in range(case["batch"]):
        at = torch.arange(case["tokens"], device=DEV) + pages.lengths[b]
        page = torch.tensor(pages.table[b], device=DEV)[at // pages.page]
        pages.k[page, :, at % pages.page], pages.v[page, :, at % pages.page] = k[b], wide["v"][b]
    return _exact_rotate(wide["q"], wide["q_weight"], positions, wide["frequencies"])


def _exact_attention(case, pages, q, lam, masks):
    """Request by request and key head by key head, with a softmax over the keys that a query sees."""
    n, hk, d, group = case["tokens"], case["kv_heads"], case["d"], case["heads"] // case["kv_heads"]
    out = torch.zeros(*q.shape[:3], case["dv"], dtype=torch.float64, device=DEV)
    index = torch.arange(n, device=DEV)
    for b in range(case["batch"]):
        length = pages.lengths[b]
        page = torch.tensor(pages.table[b], device=DEV)
        if masks is None:
            hidden = index[None] > index[:, None]
        else:
            hidden = masks[b][:, None] >> index[None] & 1 == 0
        hidden = torch.cat((torch.zeros(n, length, dtype=torch.bool, device=DEV), hidden), 1)
        for head in range(hk):
            h = slice(head * group, (head + 1) * group)
            kb = pages.k[page, head].reshape(-1, 2, d)[:length + n].permute(1, 0, 2)
            vb = pages.v[page, head].reshape(-1, case["dv"])[:length + n]
            s = torch.matmul(q[b, :, h].permute(2, 1, 0, 3), kb[:, None].transpose(-1, -2)) / math.sqrt(d)      # (map, head, query, key)
            p = torch.nan_to_num(torch.softmax(s.masked_fill_(hidden, -math.inf), -1), nan=0.0)
            out[b, :, h] = torch.matmul(p[0] - lam[h].view(-1, 1, 1) * p[1], vb).transpose(0, 1)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in state.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    with torch.no_grad():
        return _exact(case, state, wide)


def _exact(case, state, wide):
    kind = case["kind"]
    if kind == "rotate_train":
        return _exact_rotate_train(case, state, wide)
    pages = _ExactPages(case, state, wide)
    if kind == "append":
        positions = state["lengths"][:, None] + torch.arange(case["tokens"], device=DEV)
        return [_exact_append(case, pages, wide, positions), pages.k, pages.v]
    if kind == "attention":
        return _exact_attention(case, pages, wide["q"], wide["lam"], state.get("masks"))
    if kind == "beams":
        pages.fork(state["sources"].tolist())
        granted, copies = pages.extend(state["drafted"].tolist())
        for p, to in copies:
            if to >= 0:
                pages.k[to], pages.v[to] = pages.k[p], pages.v[p]
        return [torch.tensor(granted, dtype=torch.int32, device=DEV), torch.tensor(copies, dtype=torch.int32, device=DEV), *pages.held()]
    pages.trim(state["start"].tolist())
    granted, _ = pages.extend(state["drafted"].tolist())
    masks, positions = _exact_tree(state["parents"].tolist(), pages.lengths)
    outs = [torch.tensor(granted, dtype=torch.int32, device=DEV), masks, positions]
    if kind == "step":
        outs.append(_exact_attention(case, pages, _exact_append(case, pages, wide, positions), wide["lam"], masks))
    accepted = state["accepted"].tolist()
    pages.compact(state["path"].tolist(), accepted)
    pages.trim([n + more for n, more in zip(pages.lengths, accepted)])
    return [*outs, *pages.held()]
