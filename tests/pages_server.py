"""A server over nn.PageTable that knows which tokens every request has, and the operators that it calls on the host."""
import torch

import mamtorch_amd as mt
import pages_reference as pref

PAGE = 16


class HostOperators:
    """The pages' operators on tensors of the host, from their definitions."""

    @staticmethod
    def _write(book, table, lengths, refs):
        table.copy_(torch.tensor(book.table(), dtype=torch.int32).view(table.shape))
        lengths.copy_(torch.tensor(book.lengths, dtype=torch.int32))
        refs.copy_(torch.tensor(book.refs(), dtype=torch.int32))

    def pages_extend(self, table, lengths, refs, counts, page):
        book = pref.Book(table.tolist(), lengths.tolist(), refs.numel(), page)
        granted, copies = book.extend(counts.tolist())
        self._write(book, table, lengths, refs)
        return torch.tensor(granted, dtype=torch.int32), torch.tensor(copies, dtype=torch.int32)

    def pages_fork(self, table, lengths, refs, sources, page):
        book = pref.Book(table.tolist(), lengths.tolist(), refs.numel(), page)
        book.fork(sources.tolist())
        self._write(book, table, lengths, refs)

    def pages_trim(self, table, lengths, refs, ends, page):
        book = pref.Book(table.tolist(), lengths.tolist(), refs.numel(), page)
        book.trim(ends.tolist())
        self._write(book, table, lengths, refs)

    def pages_copy(self, k, v, copies):
        for a, b in copies.tolist():
            if a >= 0 and b >= 0:
                k[b], v[b] = k[a], v[a]

    def pages_compact(self, k, v, table, lengths, path, counts=None):
        page = k.shape[2]
        for b, (row, length) in enumerate(zip(path.tolist(), lengths.tolist())):
            above = -1
            for i, step in enumerate(row[:None if counts is None else max(0, int(counts[b]))]):
                if step <= above:
                    break
                above = step
                if (length + step) // page >= table.shape[1]:
                    continue
                p, t = (int(table[b, (length + x) // page]) for x in (step, i))
                if p >= 0 and t >= 0:
                    for pool in (k, v):
                        pool[t, :, (length + i) % page] = pool[p, :, (length + step) % page]

    def draft_tree(self, parents, lengths=None):
        seen = torch.stack([pref.tree(row) for row in parents.tolist()])
        return pref.bits(seen), (seen.sum(-1) - 1 + (0 if lengths is None else lengths[:, None])).int()

    def norm_rotate_append(self, q, k, v, k_pages, v_pages, table, lengths, *rest, counts=None):
        for b, length in enumerate(lengths.tolist()):
            for i in range(k.shape[1] if counts is None else max(0, int(counts[b]))):
                p = int(table[b, (length + i) // PAGE])
                k_pages[p, :, (length + i) % PAGE], v_pages[p, :, (length + i) % PAGE] = k[b, i], v[b, i]
        return q


def place_on(device, monkeypatch):
    """The device that servers are on; the operators of the host are put in the place of those of the GPU."""
    if device == "cpu":
        host = HostOperators()
        for name in ("pages_extend", "pages_fork", "pages_trim", "pages_copy", "pages_compact", "draft_tree", "norm_rotate_append"):
            monkeypatch.setattr(mt.kernel.encoder, name, getattr(host, name))
    return device


class Server:
    """Requests whose tokens are numbers; after every call the pages hold them, for each request in its order."""

    def __init__(self, device, batch, pages, most=None):
        self.device, self.batch = device, batch
        self.table = mt.nn.PageTable(batch, pages, PAGE, most, device=device)
        self.caches = [mt.nn.DiffAttentionPages(self.table, 1, 8, 8, device=device) for _ in range(2)]
        for c in self.caches:               # what nobody has put there is no token
            c.k.fill_(-1.0)
            c.v.fill_(-1.0)
        self.tokens, self.next = [[] for _ in range(batch)], 0

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def new(self, n):
        """n tokens a request, as numbers and as keys and values."""
        ids = [[self.next + b * n + i for i in range(n)] for b in range(self.batch)]
        self.next += self.batch * n
        t = torch.tensor(ids, dtype=torch.float32, device=self.device).view(self.batch, n, 1, 1)
        return ids, t[..., None].expand(-1, -1, -1, 2, 8).contiguous(), t.expand(-1, -1, -1, 8).contiguous()

    def append(self, k, v):
        for c in self.caches:
            c.append(k, k, v, norm=False)

    def check(self, what):
        table, lengths = self.table.table.tolist(), self.table.lengths.tolist()
        assert lengths == [len(t) for t in self.tokens], what
        for c in self.caches:
            k, v = c.k[:, 0, :, :, 0].tolist(), c.v[:, 0, :, 0].tolist()
            for b, tokens in enumerate(self.tokens):
                got = [k[table[b][i // PAGE]][i % PAGE] for i in range(len(tokens))]
                assert got == [[t, t] for t in tokens], (what, "keys of request %d" % b)
                assert [v[table[b][i // PAGE]][i % PAGE] for i in range(len(tokens))] == tokens, (what, "values of request %d" % b)
        held = [0] * self.table.pages
        for row in table:
            for p in row:
                if p >= 0:
                    held[p] += 1
        assert self.table.refs.tolist() == held, what

    def step(self, counts, accepted=None):
        """Counts of new tokens, of which `accepted` (all by default) stay; returns what was granted."""
        granted = self.table.begin(self.ints(counts))
        got = granted.tolist()
        if max(got, default=0) > 0:
            ids, k, v = self.new(max(got))
            self.append(k, v)
        self.table.accept(None if accepted is None else None, None if accepted is None else self.ints(accepted))
        for b, n in enumerate(got):
            self.tokens[b] += ids[b][:n if accepted is None else max(0, min(n, accepted[b]))] if n else []
        self.check(("step", counts, got))
        return got

    def draft(self, parents, path, counts=None, drafted=None):
        """Trees of drafted tokens, of which the path's first `counts` stay."""
        granted = self.table.begin(None if drafted is None else self.ints(drafted), self.ints(parents)).tolist()
        ids, k, v = self.new(len(parents[0]))
        self.append(k, v)
        self.table.accept(self.ints(path), None if counts is None else self.ints(counts))
        for b, n in enumerate(granted):
            for i, step in enumerate(path[b][:n if counts is None else max(0, min(n, counts[b]))]):
                if not (path[b][i - 1] if i else -1) < step < n:
                    break
                self.tokens[b].append(ids[b][step])
        self.check(("draft", path, counts, granted))
        return granted

    def fork(self, sources):
        self.table.fork(self.ints(sources))
        self.tokens = [list(self.tokens[s]) if 0 <= s < self.batch else [] for s in sources]
        self.check(("fork", sources))

    def trim(self, ends):
        self.table.trim(self.ints(ends))
        self.tokens = [t[:max(0, n)] for t, n in zip(self.tokens, ends)]
        self.check(("trim", ends))
