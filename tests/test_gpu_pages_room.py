"""GPU tests of which requests find room where pages run out while others hold them too, against lists on the host."""
import random

import pytest
import torch

import mamtorch_amd as mt
from test_gpu_pages import Both

pytestmark = pytest.mark.gpu
enc = mt.kernel.encoder


def test_a_page_stays_with_a_holder_that_is_refused():
    k = Both(3, 4, 2, 16)
    k.extend([20, 0, 0])
    k.trim([20, 0, 0])
    k.fork([0, 0, -1])
    k.trim([20, 18, 0])
    assert k.extend([1, 1, 0])[0] == [0, 0, 0]
    assert k.extend([0, 1, 0])[0] == [0, 0, 0]
    k.trim([20, 0, 0])
    assert k.extend([1, 1, 0])[0] == [1, 0, 0]


def test_holders_in_front_of_the_refused_one_count():
    # four holders of a page, room for two copies: the third is refused, so the fourth may not write
    k = Both(5, 4, 4, 16)
    k.extend([20, 0, 0, 0, 0])
    k.trim([20, 0, 0, 0, 0])
    k.fork([0, 0, 0, 0, -1])
    k.trim([20, 19, 18, 17, 0])
    granted, copies = k.extend([1, 1, 1, 1, 0])
    assert granted == [1, 1, 0, 0, 0] and [c[0] >= 0 for c in copies] == [True, True, False, False, False]
    # and one that is refused for another reason does not keep a third page's last holder from writing
    k = Both(4, 6, 4, 16)
    k.extend([20, 40, 0, 0])
    k.trim([20, 0, 0, 0])
    k.extend([0, 8, 0, 0])
    k.trim([20, 8, 0, 0])
    k.fork([1, 0, 1, -1])           # requests 0 and 2 share a page
    assert k.extend([1, 60, 1, 0])[0] == [1, 0, 1, 0]


@pytest.mark.parametrize("seed", range(20))
def test_few_pages_at_random(seed):
    rng = random.Random(1000 + seed)
    batch = rng.choice([2, 3, 5, 9, 70])
    k = Both(batch, rng.choice([2, 3, 6]), rng.choice([2, batch, batch + 2, 2 * batch]), 16)
    for _ in range(40):
        what = rng.random()
        if what < 0.5:
            granted, _ = k.extend([rng.choice([0, 1, 1, 2, rng.randint(1, 20)]) for _ in range(batch)])
            k.trim([n + rng.randint(0, g) for n, g in zip(k.host.lengths, granted)])
        elif what < 0.8:
            k.fork([rng.choice([b, rng.randint(-1, batch), rng.randrange(min(batch, 3))]) for b in range(batch)])
        else:
            k.trim([rng.choice([n, rng.randint(0, n), max(0, n - 1)]) for n in k.host.lengths])


def test_many_requests_on_few_pages():
    # beyond 1024 requests a thread has several; pages in common among requests of different threads and turns
    rng = random.Random(3)
    k = Both(3000, 3, 40, 16)
    k.extend([20] + [0] * 2999)
    k.trim([20] + [0] * 2999)
    k.fork([0] * 3000)
    k.trim([rng.randint(17, 20) for _ in range(3000)])
    k.extend([rng.choice([0, 1]) for _ in range(3000)])
    k.trim([n - rng.choice([0, 1]) for n in k.host.lengths])
    for _ in range(3):
        k.extend([rng.choice([0, 1, 1]) if b > 2900 else 0 for b in range(3000)])
    k.trim([n if b > 2990 else 0 for b, n in enumerate(k.host.lengths)])
    k.extend([1] * 3000)


@torch.no_grad()
def test_a_cache_of_no_pages_takes_and_shows_nothing():
    make = lambda *s: torch.randn(*s, device="cuda:0")           # noqa: E731
    q, k, v, kp, vp = make(2, 3, 4, 2, 16), make(2, 3, 2, 2, 16), make(2, 3, 2, 8), make(0, 2, 16, 2, 16), make(0, 2, 16, 8)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda:0")       # noqa: E731
    table, lengths = ints([-1, 0], [5, -1]), ints(0, 20)
    assert torch.equal(enc.norm_rotate_append(q, k, v, kp, vp, table, lengths, norm=False), q)
    assert not enc.diff_attention_pages(q, kp, vp, table, lengths, make(4)).any()
    server = mt.nn.PageTable(2, 0, 16, most=64, device="cuda:0")
    module = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=12).to("cuda:0")
    cache = module.pages(server)
    assert server.begin(3).tolist() == [0, 0]
    assert torch.isfinite(module(make(2, 3, 96), cache=cache)).all()
    server.accept()
    server.fork(ints(1, 0))
    assert server.lengths.tolist() == [0, 0]
