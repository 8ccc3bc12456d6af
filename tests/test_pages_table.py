"""nn.PageTable as a server uses it: after every call each request's pages hold its own tokens, whoever shares them, on the host's operators and on the GPU's."""
import random

import pytest
import torch

from pages_server import PAGE, Server, place_on

GPU = pytest.param("cuda:0", marks=pytest.mark.gpu)


@pytest.fixture(params=["cpu", GPU])
def device(request, monkeypatch):
    return place_on(request.param, monkeypatch)


def test_pages_in_common_for_longer_than_one_step(device):
    s = Server(device, 3, 12)
    s.step([20, 0, 0])
    s.fork([0, 0, 0])
    s.step([1, 0, 0])               # the first one leaves the page; the others still share it
    s.step([0, 1, 0])
    s.step([1, 1, 1])


def test_a_step_of_no_tokens_after_a_fork(device):
    s = Server(device, 2, 12)
    s.step([20, 0])
    s.fork([0, 0])
    s.step([0, 0])
    s.step([1, 1])


def test_requests_cut_back_into_a_whole_page_in_common(device):
    s = Server(device, 2, 12)
    s.step([32, 0])
    s.fork([0, 0])
    s.step([1, 1])
    s.trim([26, 30])
    s.step([1, 1])


def test_a_refused_request_has_its_page_copied_when_there_is_room_again(device):
    s = Server(device, 3, 4)
    s.step([20, 0, 30])
    s.fork([0, 0, 2])
    assert s.step([1, 0, 0]) == [0, 0, 0]
    s.trim([20, 20, 0])
    assert s.step([1, 1, 0]) == [1, 1, 0]


@pytest.mark.gpu
def test_eager_steps_beside_captured_ones():
    s = Server("cuda:0", 3, 30)
    s.step([20, 0, 0])
    one, none = s.ints([1, 0, 0]), s.ints([0, 0, 0])

    def capture(what):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            what()
        return graph

    def step(counts):
        s.table.begin(counts)
        s.table.accept(counts=none)

    s.fork([0, 0, 0])
    capture(lambda: step(one))                      # nothing has run: the page is shared still
    s.check("captured begin")
    s.step([0, 1, 1])
    sources = s.ints([2, 2, 2])
    graph = capture(lambda: s.table.fork(sources))
    for turn in range(3):                           # forks that the host did not see
        s.step([1, 0, 1])
        s.step([1, 1, 1])
        graph.replay()
        s.tokens = [list(s.tokens[2]) for _ in range(3)]
        s.check(("replayed fork", turn))
        s.step([0, 1, 0])
        s.step([1, 1, 1])


def test_a_request_that_is_refused_keeps_the_page_that_it_would_have_left(device):
    s = Server(device, 2, 2)
    s.step([20, 0])
    s.fork([0, 0])
    s.trim([20, 18])
    assert s.step([1, 1]) == [0, 0]         # the first finds no page for its copy and holds on to the one in common: the second cannot write there
    s.trim([20, 0])
    assert s.step([1, 0]) == [1, 0]


@pytest.mark.parametrize("seed", range(12))
def test_a_server_with_few_pages_at_random(device, seed):
    rng = random.Random(seed)
    batch = rng.choice([2, 3, 5])
    s = Server(device, batch, rng.choice([batch, 2 * batch, 3 * batch]), 5 * PAGE)
    for _ in range(30):
        what = rng.random()
        if what < 0.5:
            s.step([rng.choice([0, 1, 1, rng.randint(1, 20)]) for _ in range(batch)], rng.choice([None, [rng.randint(-1, 20) for _ in range(batch)]]))
        elif what < 0.7:
            s.fork([rng.choice([b, rng.randint(-1, batch), rng.randrange(batch)]) for b in range(batch)])
        elif what < 0.85:
            s.trim([rng.choice([len(t), rng.randint(0, len(t)), 0]) for t in s.tokens])
        else:
            n = rng.choice([1, 4, 9])
            s.draft([[rng.randint(-1, i - 1) for i in range(n)] for _ in range(batch)], [sorted(rng.sample(range(n), n)) for _ in range(batch)], [rng.randint(0, n) for _ in range(batch)])


LINE = [[i - 1 for i in range(6)]] * 4


@pytest.mark.parametrize("counts", [None, [6, 6, 6, 6], [2, 3, 1, 0]])
def test_a_path_names_tokens_of_the_step_alone(device, counts):
    s = Server(device, 4, 24)
    s.step([20, 3, 16, 0])
    # padded trees of 4, 6, 2 and no tokens
    s.draft(LINE, [[0, 2, 5, 5, 5, 5], [1, 2, 4, 5, 0, 0], [0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5]], counts, drafted=[4, 6, 2, 0])
    # names that are none, and that do not ascend
    s.draft(LINE, [[-1, 0, 1, 2, 3, 4], [0, 0, 1, 2, 3, 4], [3, 2, 4, 5, 5, 5], [0, 1, 6, 7, 8, 9]], counts)
    s.draft(LINE, [[], [], [], []], counts)
    s.draft(LINE, [[0, 1, 2, 3, 4, 5, 6, 7]] * 4, counts)


def test_a_path_of_a_request_without_room(device):
    s = Server(device, 2, 3)
    s.step([16, 16])
    assert s.draft(LINE[:2], [[0, 1, 2, 3, 4, 5]] * 2) == [6, 0]


@pytest.mark.gpu
def test_a_captured_path_ends_where_the_eager_one_does():
    servers = [Server("cuda:0", 3, 40) for _ in range(2)]
    path, drafted = servers[0].ints([[0, 1, 2]] * 3), servers[0].ints([0] * 3)
    parents = servers[0].ints([[-1, 0, 1]] * 3)

    def step(s):
        s.table.begin(drafted, parents)
        s.table.accept(path)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(servers[0])
    for turn, rows in enumerate([[[0, 1, 2]] * 3, [[2, 1, 0], [1, 2, 0], [-1, 0, 1]], [[0, 2, 3], [3, 0, 1], [1, 2, 3]], [[0, 0, 0]] * 3]):
        path.copy_(servers[0].ints(rows))
        drafted.copy_(servers[0].ints([3, turn, 2]))
        graph.replay()
        step(servers[1])
        torch.cuda.synchronize()
        assert servers[0].table.lengths.tolist() == servers[1].table.lengths.tolist()
        assert torch.equal(servers[0].table.table, servers[1].table.table)


def test_a_tree_has_no_more_tokens_than_it_names(device):
    s = Server(device, 2, 12)
    s.step([20, 3])
    granted = s.table.begin(s.ints([9, 2]), s.ints([[-1, 0, 1]] * 2))
    assert granted.tolist() == [3, 2]
    ids, k, v = s.new(3)
    s.append(k, v)
    s.table.accept(s.ints([[0, 2, 5, 7]] * 2))
    s.tokens = [s.tokens[0] + [ids[0][0], ids[0][2]], s.tokens[1] + [ids[1][0]]]
    s.check("a path past the tree")
    s.table.begin(s.ints([40, 40]), s.ints([[-1]] * 2))
    ids, k, v = s.new(1)
    s.append(k, v)
    s.table.accept()
    s.tokens = [t + row for t, row in zip(s.tokens, ids)]
    s.check("trees of one token")
