"""GPU tests of the pages of a cache: bookkeeping against lists on the host, copies and compaction against indexing, trees, appended tokens; streams, graphs, refusals."""
import random

import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt
import pages_reference as pref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ints(values, shape=None):
    t = torch.tensor(values, dtype=torch.int32, device=DEV)
    return t if shape is None else t.reshape(shape)


def _make(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


class Both:
    """The bookkeeping on the GPU and on the host; every call is compared."""

    def __init__(self, batch, slots, pages, page):
        self.page = page
        self.table = torch.full((batch, slots), -1, dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        self.host = pref.Book([[-1] * slots for _ in range(batch)], [0] * batch, pages, page)

    def check(self, what):
        assert self.table.tolist() == self.host.table(), what
        assert self.lengths.tolist() == self.host.lengths, what
        assert self.refs.tolist() == self.host.refs(), what

    def extend(self, counts):
        granted, copies = enc.pages_extend(self.table, self.lengths, self.refs, _ints(counts), self.page)
        want = self.host.extend(counts)
        assert granted.tolist() == want[0] and copies.tolist() == want[1]
        self.check(("extend", counts))
        return want

    def trim(self, ends):
        enc.pages_trim(self.table, self.lengths, self.refs, _ints(ends), self.page)
        self.host.trim(ends)
        self.check(("trim", ends))

    def fork(self, sources):
        enc.pages_fork(self.table, self.lengths, self.refs, _ints(sources), self.page)
        self.host.fork(sources)
        self.check(("fork", sources))


def test_room_for_the_first_tokens_and_the_next():
    k = Both(3, 8, 20, 16)
    assert k.extend([1, 16, 33])[0] == [1, 16, 33]
    k.trim([1, 16, 33])
    k.extend([15, 1, 15])          # within the page, a new one, within
    k.trim([16, 17, 48])
    k.extend([0, -5, 0])           # none
    k.extend([1, 1, 1])
    k.extend([1, 1, 1])            # room that is there is not taken again
    k.trim([17, 0, 20])            # a request that ends, one that is cut back
    k.extend([100, 100, 100])


def test_a_request_that_does_not_fit_is_left_as_it_was():
    k = Both(4, 4, 6, 16)
    assert k.extend([40, 65, 40, 1])[0] == [40, 0, 40, 0]      # 65 tokens are more than its slots hold; the fourth finds no page
    k.trim([40, 0, 40, 0])
    assert k.extend([8, 1, 8, 0])[0] == [8, 0, 8, 0]           # room without a page; those behind a refused one are served where they need none
    assert k.extend([9, 0, 8, 1])[0] == [0, 0, 8, 0]
    k.trim([40, 0, 0, 0])
    assert k.extend([9, 33, 1, 0])[0] == [9, 0, 0, 0]          # three pages: one for the first, the second needs three, the third may not pass it
    k = Both(2, 4, 0, 16)
    assert k.extend([1, 0])[0] == [0, 0]
    k = Both(2, 0, 5, 16)
    assert k.extend([1, 0])[0] == [0, 0]
    k.fork([1, 0])
    k.trim([3, 0])


def test_begun_pages_in_common_are_copied_but_for_the_last_holder():
    k = Both(5, 6, 30, 16)
    k.extend([20, 32, 0, 0, 0])
    k.trim([20, 32, 0, 0, 0])
    k.fork([0, 1, 0, 0, 1])
    _, copies = k.extend([1, 1, 1, 1, 1])
    assert [c[0] >= 0 for c in copies] == [True, False, True, False, False]    # a whole last page is nobody's to write
    k.trim([21, 33, 21, 21, 33])
    k.fork([2, 2, 2, 2, 2])
    _, copies = k.extend([1, 0, 0, 1, 0])           # holders that do not write keep it
    assert [c[0] >= 0 for c in copies] == [True, False, False, True, False]
    k.fork([-1, 0, 99, 3, -7])
    k.fork([1, 3, 1, 3, 1])
    k.fork([0, 1, 2, 3, 4])


def test_a_copy_with_room_behind_it_and_pages_kept_from_before():
    k = Both(3, 8, 24, 16)
    k.extend([20, 0, 0])
    k.trim([20, 0, 0])
    k.fork([0, 0, 0])
    k.extend([40, 50, 12])
    k.extend([60, 50, 12])
    k.trim([30, 30, 30])
    k.fork([1, 1, 0])
    k.extend([3, 3, 40])


@pytest.mark.parametrize("seed", range(6))
def test_a_server_at_random(seed):
    rng = random.Random(seed)
    batch, page = rng.choice([1, 3, 17, 64]), rng.choice([16, 32, 48])
    slots = rng.choice([3, 9, 40])
    k = Both(batch, slots, rng.choice([batch * 2, batch * slots // 2 + 1, batch * slots + 5]), page)
    for _ in range(25):
        what = rng.random()
        if what < 0.5:
            granted, _ = k.extend([rng.choice([0, 1, 1, rng.randint(1, 2 * page)]) for _ in range(batch)])
            if rng.random() < 0.8:
                k.trim([n + rng.randint(0, g) for n, g in zip(k.host.lengths, granted)])
        elif what < 0.75:
            k.fork([rng.choice([b, rng.randint(-1, batch), rng.randrange(batch)]) for b in range(batch)])
        else:
            k.trim([rng.choice([n, rng.randint(0, n), 0, n + rng.randint(0, 2 * page)]) for n in k.host.lengths])


def test_many_requests_and_pages():
    # 4096 requests: the most; more pages than a turn of the search holds, the free ones far behind
    k = Both(4096, 3, 40000, 16)
    rng = random.Random(1)
    counts = [rng.randint(1, 40) for _ in range(4096)]
    k.extend(counts)
    k.trim([c - 1 for c in counts])
    k.fork([rng.randrange(4096) for _ in range(4096)])
    k.extend([1] * 4096)
    k = Both(2, 2, 40000, 16)
    k.refs.fill_(1)
    k.refs[39990:39994] = 0
    granted, _ = enc.pages_extend(k.table, k.lengths, k.refs, _ints([17, 20]), 16)
    assert granted.tolist() == [17, 20] and k.table.tolist() == [[39990, 39991], [39992, 39993]]


def test_one_request_over_a_long_table():
    k = Both(1, 5000, 6000, 16)
    k.extend([80000])
    k.trim([79999])
    k.trim([17])
    k.extend([60000])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page, hk, d, dv", [(16, 1, 64, 128), (48, 3, 33, 7), (128, 2, 128, 256), (16, 2, 1, 1)])
def test_copies_of_pages(page, hk, d, dv, dtype):
    k, v = _make((9, hk, page, 2, d), dtype, 1), _make((9, hk, page, dv), dtype, 2)
    kg, vg = k.to(DEV), v.to(DEV)
    enc.pages_copy(kg, vg, _ints([[3, 5], [-1, -1], [0, 8], [3, 1], [-1, 2], [4, -1], [7, 9], [9, 7], [6, 6]]))
    for a, b in ((3, 5), (0, 8), (3, 1)):
        k[b], v[b] = k[a], v[a]
    assert torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page, hk, d, dv", [(16, 1, 64, 128), (48, 3, 33, 7), (32, 4, 128, 256), (16, 2, 1, 1)])
@pytest.mark.parametrize("n", [1, 5, 31, 64])
def test_compaction(n, page, hk, d, dv, dtype):
    rng = random.Random(n)
    lengths = [0, 5, 16, 47, 30, 12, 9]
    b = len(lengths)
    book = pref.Book([[-1] * 12 for _ in range(b)], lengths, 90, page)
    order = list(range(90))
    rng.shuffle(order)
    for row, length in zip(book.rows, lengths):
        row.extend(order.pop() for _ in range(-(-(length + n) // page)))
    k, v = _make((90, hk, page, 2, d), dtype, 3), _make((90, hk, page, dv), dtype, 4)
    path = [sorted(rng.sample(range(n), n)) for _ in range(b)]
    counts = [min(n, c) for c in (1, 3, 20, 9, 0, n, n)]
    for row, count in zip(path, counts):
        row[:count] = sorted(rng.sample(range(n), count))
    path[5] = list(range(n))                # in place: nothing moves
    if n > 4:
        path[6][2] = path[6][1]             # does not ascend: its tokens stay from there on
    kg, vg = k.to(DEV), v.to(DEV)
    enc.pages_compact(kg, vg, _ints(book.table()), _ints(lengths), _ints(path), _ints(counts))
    for row, pages, length, count in zip(path, book.rows, lengths, counts):
        old = [(k[pages[(length + t) // page], :, (length + t) % page].clone(), v[pages[(length + t) // page], :, (length + t) % page].clone()) for t in range(n)]
        for i in range(count):
            if i and row[i] <= row[i - 1]:
                break
            k[pages[(length + i) // page], :, (length + i) % page], v[pages[(length + i) // page], :, (length + i) % page] = old[row[i]]
    assert torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)


def test_compaction_of_what_has_no_page_or_no_sense():
    k, v = _make((4, 1, 16, 2, 8), torch.float32, 5), _make((4, 1, 16, 8), torch.float32, 6)
    for table, lengths, path, counts in (([[0, -1]], [15], [[1, 2]], None), ([[-1, 3]], [0], [[1, 1]], [2]), ([[0, 9]], [14], [[3, 4]], [9]), ([[0, 1]], [-4], [[-1, 2]], [2]),
                                         ([[0, 1]], [900], [[1, 2]], [2]), ([[0, 1]], [3], [[7, 1]], [2]), ([[0, 1]], [3], [[2 ** 31 - 1, 1]], [2]), ([[0, 1]], [3], [[1, 2]], [-1])):
        kg, vg = k.to(DEV), v.to(DEV)
        enc.pages_compact(kg, vg, _ints(table), _ints(lengths), _ints(path), None if counts is None else _ints(counts))
        k_want, v_want = k.clone(), v.clone()
        if path == [[7, 1]]:            # up to where it does not ascend
            k_want[0, :, 3], v_want[0, :, 3] = k[0, :, 10], v[0, :, 10]
        assert torch.equal(kg.cpu(), k_want) and torch.equal(vg.cpu(), v_want), (table, lengths, path)


@pytest.mark.parametrize("n", [1, 2, 7, 33, 64])
def test_trees(n):
    rng = random.Random(n)
    rows = [[i - 1 for i in range(n)], [-1] * n, [0 if i else -1 for i in range(n)], [rng.randint(-1, i - 1) for i in range(n)], [rng.randint(-1, i - 1) for i in range(n)],
            [rng.choice([i, i + 1, 64, -1, -99, 2 ** 31 - 1, -2 ** 31]) for i in range(n)]]
    lengths = [0, 7, 100000, 3, 1, 2]
    seen = torch.stack([pref.tree(row) for row in rows])
    for given in (None, lengths):
        masks, positions = enc.draft_tree(_ints(rows), None if given is None else _ints(given))
        assert torch.equal(masks.cpu(), pref.bits(seen))
        assert torch.equal(positions.cpu(), (seen.sum(-1) - 1 + (0 if given is None else torch.tensor(given)[:, None])).int())
    masks, positions = enc.draft_tree(_ints([], (0, n)))
    assert masks.shape == (0, n) and positions.dtype == torch.int32


# ---- appended tokens ----
def _filled(lengths, n, page, pages, seed, spare=0):
    """Table with room for n tokens behind each request's."""
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    slots = max(-(-(length + n) // page) for length in lengths) + spare
    return [[order.pop() if s < -(-(length + n) // page) else -1 for s in range(slots)] for length in lengths]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, page, h, hk, d, dv, turned", [(1, 16, 4, 2, 64, 128, 64), (1, 48, 6, 6, 80, 33, 60), (37, 16, 8, 2, 128, 256, 128), (5, 32, 3, 1, 33, 7, 0), (130, 64, 2, 2, 32, 64, 20)])
def test_tokens_are_appended(n, page, h, hk, d, dv, turned, dtype):
    lengths = [0, 1, page - 1, page, 3 * page + 5]
    b = len(lengths)
    table = _filled(lengths, n, page, 60, 1, 1)
    q, k, v = _make((b, n, h, 2, d), dtype, 7), _make((b, n, hk, 2, d), dtype, 8), _make((b, n, hk, dv), dtype, 9)
    w, f = 1 + _make((d,), torch.float32, 10, 0.3), enc.rotary_frequencies(turned) if turned else None
    kp, vp = _make((60, hk, page, 2, d), dtype, 11), _make((60, hk, page, dv), dtype, 12)
    on = lambda t: None if t is None else t.to(DEV)                                     # noqa: E731
    places = torch.tensor(lengths, dtype=torch.int32)[:, None] + torch.arange(n, dtype=torch.int32)
    other = torch.randint(0, 9000, (b, n), generator=torch.Generator().manual_seed(13), dtype=torch.int32)
    counts = [n, 0, -3, (n + 1) // 2, n + 9]
    for given, some in ((None, None), (other, counts)):
        kg, vg = kp.to(DEV), vp.to(DEV)
        out = enc.norm_rotate_append(on(q), on(k), on(v), kg, vg, _ints(table), _ints(lengths), on(w), on(w), on(f), on(given), counts=None if some is None else _ints(some))
        at = places if given is None else given
        want = pref.Rotation(q, w, at, f)
        ref.assert_within(out, want.y, want.y_bound, "queries")
        want = pref.Rotation(k, w, at, f)
        k_want, k_bound, v_want = kp.double(), torch.zeros(kp.shape, dtype=torch.float64), vp.clone()
        for r in range(b):
            for i in range(n if some is None else max(0, min(n, some[r]))):
                p, o = table[r][(lengths[r] + i) // page], (lengths[r] + i) % page
                k_want[p, :, o], k_bound[p, :, o], v_want[p, :, o] = want.y[r, i], want.y_bound[r, i], v[r, i]
        ref.assert_within(kg, k_want, k_bound, "keys")                  # what was not appended is as it was
        assert torch.equal(vg.cpu(), v_want)


def test_tokens_without_a_page_are_not_written():
    q, k, v = (_make((3, 4, 2, 2, 16), torch.float32, 14).to(DEV), _make((3, 4, 1, 2, 16), torch.float32, 15).to(DEV), _make((3, 4, 1, 8), torch.float32, 16).to(DEV))
    kp, vp = _make((4, 1, 16, 2, 16), torch.float32, 17).to(DEV), _make((4, 1, 16, 8), torch.float32, 18).to(DEV)
    was = kp.clone(), vp.clone()
    out = enc.norm_rotate_append(q, k, v, kp, vp, _ints([[-1, -1], [4, 100], [0, 1]]), _ints([0, 14, 32]), norm=False)
    assert torch.equal(out, q) and torch.equal(kp, was[0]) and torch.equal(vp, was[1])
    enc.norm_rotate_append(q, k, v, kp, vp, _ints([[-1, -1], [3, 100], [0, 1]]), _ints([-5, 14, 30]), norm=False)
    assert torch.equal(kp[3, :, 14:].transpose(0, 1), k[1, :2]) and torch.equal(vp[1, :, 14:].transpose(0, 1), v[2, :2])
    kp[3, :, 14:], vp[3, :, 14:], kp[1, :, 14:], vp[1, :, 14:] = was[0][3, :, 14:], was[1][3, :, 14:], was[0][1, :, 14:], was[1][1, :, 14:]
    assert torch.equal(kp, was[0]) and torch.equal(vp, was[1])


def test_strided_keys_and_values_are_appended():
    b, n, h, hk, d, dv = 2, 6, 4, 2, 32, 24
    wide = _make((b, n, (h + hk) * 2 * d + hk * dv + 3), torch.float16, 19).to(DEV)
    q = wide[..., 1:1 + h * 2 * d].unflatten(-1, (h, 2, d))
    k = wide[..., 1 + h * 2 * d:1 + (h + hk) * 2 * d].unflatten(-1, (hk, 2, d))
    v = wide[..., 1 + (h + hk) * 2 * d:1 + (h + hk) * 2 * d + hk * dv].unflatten(-1, (hk, dv))
    outs = []
    for views in ((q, k, v), (q.contiguous(), k.contiguous(), v.contiguous()), (q, k.transpose(3, 4).contiguous().transpose(3, 4), v.transpose(1, 3).contiguous().transpose(1, 3))):
        kp, vp = torch.zeros(4, hk, 16, 2, d, dtype=torch.float16, device=DEV), torch.zeros(4, hk, 16, dv, dtype=torch.float16, device=DEV)
        y = enc.norm_rotate_append(*views, kp, vp, _ints([[2, 0], [1, 3]]), _ints([12, 0]), frequencies=enc.rotary_frequencies(d, device=DEV))
        outs.append((y, kp, vp))
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))


# ---- streams, graphs, versions, refusals ----
def test_a_step_on_another_stream_and_captured():
    b, n, hk, d, dv, page = 4, 3, 2, 32, 32, 16
    q, k, v = (_make((b, n, 4, 2, d), torch.float32, 20).to(DEV), _make((b, n, hk, 2, d), torch.float32, 21).to(DEV), _make((b, n, hk, dv), torch.float32, 22).to(DEV))
    lam, counts, path, accepted, sources = torch.full((4,), 0.4, device=DEV), _ints([3] * b), _ints([[0, 2, 2]] * b), _ints([2, 1, 0, 2]), _ints([1, 1, 3, 3])
    parents = _ints([[-1, 0, 0]] * b)
    f = enc.rotary_frequencies(d, device=DEV)

    class Run:
        def __init__(self):
            self.table = torch.full((b, 9), -1, dtype=torch.int32, device=DEV)
            self.lengths, self.refs = torch.zeros(b, dtype=torch.int32, device=DEV), torch.zeros(40, dtype=torch.int32, device=DEV)
            self.k, self.v = torch.zeros(40, hk, page, 2, d, device=DEV), torch.zeros(40, hk, page, dv, device=DEV)

        def step(self):
            enc.pages_fork(self.table, self.lengths, self.refs, sources, page)
            granted, copies = enc.pages_extend(self.table, self.lengths, self.refs, counts, page)
            enc.pages_copy(self.k, self.v, copies)
            masks, places = enc.draft_tree(parents, self.lengths)
            y = enc.norm_rotate_append(q, k, v, self.k, self.v, self.table, self.lengths, frequencies=f, positions=places, counts=granted)
            out = enc.diff_attention_pages(y, self.k, self.v, self.table, self.lengths, lam, counts=granted, masks=masks)
            enc.pages_compact(self.k, self.v, self.table, self.lengths, path, accepted)
            enc.pages_trim(self.table, self.lengths, self.refs, self.lengths + accepted, page)
            return out

        def state(self):
            return [t.clone() for t in (self.table, self.lengths, self.refs, self.k, self.v)]

    eager = Run()
    wants = []
    for _ in range(12):
        out = eager.step()
        wants.append([out.clone()] + eager.state())
    other = Run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for want in wants:
            assert all(torch.equal(x, y) for x, y in zip([other.step()] + other.state(), want))
    torch.cuda.current_stream().wait_stream(side)
    replayed, second = Run(), Run()
    graphs = []
    for run in (replayed, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, run.step(), run))
    for want in wants:
        for graph, out, run in graphs:          # two graphs in turn, eager work between them
            graph.replay()
            got = [out.clone()] + run.state()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_calls_that_change_a_tensor_are_seen_by_a_backward_pass():
    pages = torch.randn(2, 1, 16, 2, 8, device=DEV), torch.randn(2, 1, 16, 8, device=DEV)
    x = torch.ones((), device=DEV, requires_grad=True)
    y = (pages[0] * x).sum()
    enc.pages_copy(*pages, _ints([[0, 1]]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_serving_has_no_gradient():
    q, k, v = (torch.randn(1, 2, 2, 2, 8, device=DEV), torch.randn(1, 2, 1, 2, 8, device=DEV), torch.randn(1, 2, 1, 8, device=DEV))
    kp, vp, table, lengths, lam = torch.zeros(1, 1, 16, 2, 8, device=DEV), torch.zeros(1, 1, 16, 8, device=DEV), _ints([[0]]), _ints([0]), torch.zeros(2, device=DEV)
    for grad in (q, k, v):
        grad.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no_grad"):
            enc.norm_rotate_append(q, k, v, kp, vp, table, lengths)
        grad.requires_grad_(False)
    with pytest.raises(RuntimeError, match="no_grad"):
        enc.diff_attention_pages(q.requires_grad_(True), kp, vp, table, lengths, lam)
    with torch.no_grad():
        enc.norm_rotate_append(q, k, v, kp, vp, table, lengths)
        assert not enc.diff_attention_pages(q, kp, vp, table, lengths, lam).requires_grad


def test_refusals():
    make = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=DEV)     # noqa: E731
    i32 = torch.int32
    table, lengths, refs, counts = make(2, 4, t=i32), make(2, t=i32), make(8, t=i32), make(2, t=i32)
    for call in (enc.pages_extend, enc.pages_fork, enc.pages_trim):
        good = [table, lengths, refs, counts]
        for at, bad, text in ((0, table.long(), "int32"), (0, make(4, 4, t=i32)[::2], "contiguous"), (0, make(2, t=i32), "batch, slots"), (1, make(3, t=i32), "int32"), (1, lengths.cpu(), "different device"),
                              (2, make(2, 4, t=i32), "refs"), (2, refs.float(), "int32"), (3, make(3, t=i32), "int32"), (3, counts.long(), "int32"), (0, table.cpu(), None)):
            args = list(good)
            args[at] = bad
            with pytest.raises((RuntimeError, NotImplementedError), match=text):
                call(*args, 16)
        for page in (0, 8, 24, -16):
            with pytest.raises(RuntimeError, match="multiple of 16"):
                call(*good, page)
    q, k, v = make(2, 3, 4, 2, 16), make(2, 3, 2, 2, 16), make(2, 3, 2, 8)
    kp, vp, lam = make(8, 2, 16, 2, 16), make(8, 2, 16, 8), make(4)
    for bad, text in ((dict(q=q.half()), "type"), (dict(k=make(2, 3, 1, 2, 16)), "other keys|do not match"), (dict(v=make(2, 3, 2, 9)), "other keys"), (dict(v=v.half()), "type"), (dict(v=make(2, 2, 2, 8)), "do not match"),
                      (dict(k_pages=make(8, 2, 24, 2, 16), v_pages=make(8, 2, 24, 8)), "multiple of 16"), (dict(v_pages=make(7, 2, 16, 8)), "do not match"), (dict(k_pages=make(8, 16, 2, 2, 16).transpose(1, 2)), "contiguous"),
                      (dict(k_pages=kp.half(), v_pages=vp.half()), "type"), (dict(table=make(3, 4, t=i32), lengths=make(3, t=i32)), "requests"), (dict(lengths=make(3, t=i32)), "int32"),
                      (dict(counts=make(2, t=torch.long)), "int32"), (dict(q=make(2, 3, 4, 1, 16), k=make(2, 3, 2, 1, 16)), "heads, 2"), (dict(positions=make(2, 2, t=i32)), "int32"), (dict(k_pages=kp.cpu()), "device|GPU")):
        with pytest.raises((RuntimeError, NotImplementedError), match=text):
            enc.norm_rotate_append(**{**dict(q=q, k=k, v=v, k_pages=kp, v_pages=vp, table=table, lengths=lengths), **bad})
    odd = make(8 * 2 * 16 * 2 * 16 + 1)[1:].view(8, 2, 16, 2, 16)
    with pytest.raises(RuntimeError, match="16 bytes"):
        enc.norm_rotate_append(q, k, v, odd, vp, table, lengths)
    for bad, text in ((dict(q=q.half()), "type"), (dict(q=make(2, 3, 3, 2, 16), lam=make(3)), "divide"), (dict(q=make(1, 3, 4, 2, 16)), "requests"), (dict(q=make(2, 3, 4, 2, 8)), "do not match"),
                      (dict(lam=make(3)), "lam"), (dict(lam=lam.half()), "lam"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(masks=make(2, 3, t=i32)), "int64"),
                      (dict(masks=make(3, 3, t=torch.long)), "int64"), (dict(q=make(2, 65, 4, 2, 16), masks=make(2, 65, t=torch.long)), "64 tokens"), (dict(counts=make(3, t=i32)), "int32"), (dict(q=make(2, 3, 4, 16)), "must be")):
        with pytest.raises(RuntimeError, match=text):
            enc.diff_attention_pages(**{**dict(q=q, k_pages=kp, v_pages=vp, table=table, lengths=lengths, lam=lam), **bad})
    with pytest.raises(RuntimeError, match="copies"):
        enc.pages_copy(kp, vp, make(2, 3, t=i32))
    with pytest.raises(RuntimeError, match="int32"):
        enc.pages_copy(kp, vp, make(2, 2, t=torch.long))
    with pytest.raises(RuntimeError, match="path"):
        enc.pages_compact(kp, vp, table, lengths, make(3, 2, t=i32))
    with pytest.raises(RuntimeError, match="64 tokens"):
        enc.draft_tree(make(1, 65, t=i32))
    with pytest.raises(RuntimeError, match="int32"):
        enc.draft_tree(make(1, 5, t=torch.long))
