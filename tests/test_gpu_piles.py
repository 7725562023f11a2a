"""Tokens sorted by expert and back, against torch's stable sort and sums in 64 bits."""
import itertools

import pytest
import torch

import coachwhip_amd as cw
from coachwhip_amd import ops, piles

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def say(*a):
    print(*a, flush=True)


def some_ids(t, k, e, seed, outside=True):
    """Picks of experts 0 .. e - 1, and of none where `outside`."""
    g = gen(seed)
    ids = torch.randint(-2 if outside else 0, e + (2 if outside else 0), (t, k), generator=g, device="cuda", dtype=torch.int32)
    if outside and ids.numel() > 4:
        ids.view(-1)[3] = -2 ** 31
        ids.view(-1)[1] = 2 ** 31 - 1
    return ids


def check_sort(ids, e):
    p = piles.sort_picks(ids, e)
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < e), flat, e)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=e + 1)
    assert torch.equal(p.order.long(), order)
    assert torch.equal(p.place.long()[order], torch.arange(flat.numel(), device="cuda"))
    assert torch.equal(p.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)[:e]]))
    # the tiles: every position once, none of two experts, 128 at most
    n = int(p.tiles[0])
    tiles = p.tiles[4:4 + 5 * n].view(n, 5).cpu().tolist()
    at, first = 0, {}
    for i, (x, pos0, m, f, of) in enumerate(tiles):
        assert pos0 == at and 0 < m <= 128
        first.setdefault(x, i)
        assert f == first[x] and of == (int(counts[x]) + 127) // 128 and (key[order[pos0:pos0 + m]] == x).all()
        at += m
    assert at == flat.numel()
    return p


@pytest.mark.parametrize("e", [1, 2, 8, 63, 64, 65, 256, 1000, 1023, 1024])
@pytest.mark.parametrize("t,k", [(0, 4), (1, 1), (1, 8), (7, 3), (64, 10), (1021, 8), (1024, 8), (2049, 8)])
def test_sort(t, k, e):
    say("sort", t, k, e)
    check_sort(some_ids(t, k, e, t * k + e), e)


@pytest.mark.parametrize("picks", [65536, 65537, 300001, 8192 * 256 + 5])
@pytest.mark.parametrize("e", [1, 200, 1024])
def test_sort_of_many(picks, e):
    say("sort", picks, e)
    check_sort(some_ids(picks, 1, e, picks), e)


@pytest.mark.parametrize("pick", [-1, 0, 5, 8])
def test_all_on_one(pick):
    check_sort(torch.full((3000, 4), pick, dtype=torch.int32, device="cuda"), 8)


def rows_of(g, n, h, dtype, ld=None, at=0):
    """n rows of h, ld apart, at any place of the type."""
    ld = ld or h
    flat = torch.randn(n * ld + at, generator=g, device="cuda").to(dtype)
    return flat[at:].view(n, ld)[:, :h]


SHAPES = [(1, 1, 1, 1), (1, 8, 256, 2048), (5, 3, 4, 7), (33, 10, 64, 513), (64, 1, 8, 128), (301, 4, 128, 2880), (9, 32, 40, 100), (2, 2, 2, 9001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,e,h", SHAPES)
def test_there_and_back(t, k, e, h, dtype):
    say("there and back", t, k, e, h, dtype)
    g = gen(h + t)
    ids = some_ids(t, k, e, h)
    p = piles.sort_picks(ids, e)
    key, place = ids.reshape(-1).long(), p.place.long()
    here = ((key >= 0) & (key < e))[:, None]
    for ld, at in ((h, 0), (h + 3, 1)):
        x = rows_of(g, t, h, dtype, ld, at)
        got = piles.to_piles(x, p)
        assert torch.equal(got[place], torch.where(here, x.repeat_interleave(k, 0), torch.zeros_like(x[:1])))
        # rows of no expert hold what nothing may show
        rows = rows_of(g, t * k, h, dtype, ld, at)
        rows[place[~here[:, 0]]] = float("nan")
        w = torch.randn(t, k, generator=g, device="cuda")
        for weights in (w, None):
            terms = torch.where(here, rows[place].double(), 0.0) * (1.0 if weights is None else weights.double().reshape(-1, 1))
            want, size = terms.view(t, k, h).sum(1), terms.abs().view(t, k, h).sum(1)
            got = piles.from_piles(rows, weights, p)
            assert got.dtype == dtype and got.shape == (t, h)
            # a rounding for each product joined to the sum, and that to the type
            assert ((got.double() - want).abs() <= k * U * size + half(dtype) * want.abs() + torch.finfo(dtype).tiny).all()
        assert torch.equal(piles.to_piles_grad(rows, p), piles.from_piles(rows, None, p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,e,h", SHAPES)
def test_gradients_match_the_formula(t, k, e, h, dtype):
    say("gradients", t, k, e, h, dtype)
    g = gen(h + t)
    ids = some_ids(t, k, e, h)
    p = piles.sort_picks(ids, e)
    key, place = ids.reshape(-1).long(), p.place.long()
    here = (key >= 0) & (key < e)
    for ld, at in ((h, 0), (h + 5, 1)):
        dout, rows, w = rows_of(g, t, h, dtype, ld, at), rows_of(g, t * k, h, dtype, ld + 1, at), torch.randn(t, k, generator=g, device="cuda")
        rows[place[~here]] = float("nan")
        drows, dw = piles.from_piles_grad(dout, rows, w, p)
        grow = dout.double().repeat_interleave(k, 0)
        want = torch.where(here[:, None], grow * w.double().reshape(-1, 1), 0.0)
        assert ((drows[place].double() - want).abs() <= (U + half(dtype)) * want.abs() + torch.finfo(dtype).tiny).all()
        terms = torch.where(here[:, None], grow * rows[place].double(), 0.0)
        assert ((dw.double().reshape(-1) - terms.sum(1)).abs() <= (h + 8) * U * terms.abs().sum(1)).all()


def test_gradients_match_differences():
    """The whole way, tokens to piles and back, is linear in the rows and in the weights, so that a difference of any width gives the derivative."""
    t, k, e, h = 13, 3, 5, 37
    g = gen(3)
    p = piles.sort_picks(some_ids(t, k, e, 3), e)
    x, w, c = (torch.randn(*s, generator=g, device="cuda") for s in ((t, h), (t, k), (t, h)))

    def value(x, w):
        return (piles.from_piles(piles.to_piles(x, p), w, p).double() * c.double()).sum()

    drows, dw = piles.from_piles_grad(c, piles.to_piles(x, p), w, p)
    dx = piles.to_piles_grad(drows, p)
    for leaf, grad, of in ((x, dx, lambda v: value(v, w)), (w, dw, lambda v: value(x, v))):
        step = torch.randn(leaf.shape, generator=g, device="cuda")
        slope = (of(leaf + step) - of(leaf - step)) / 2
        want = (grad.double() * step.double()).sum()
        # values of up to t h sums of k products, each term below 40 (normal numbers): U each, many times over
        assert abs(slope - want) <= 64 * U * t * h * k


def test_a_route_sorts():
    t, e, k = 77, 40, 6
    ids, _ = ops.route(torch.randn(t, e, generator=gen(1), device="cuda"), k, True)
    check_sort(ids, e)


def test_same_bits_each_time_and_in_a_graph():
    t, k, e, h = 2100, 8, 64, 256
    g = gen(5)
    ids, x, w = some_ids(t, k, e, 5), torch.randn(t, h, generator=g, device="cuda").bfloat16(), torch.randn(t, k, generator=g, device="cuda")

    def run():
        p = piles.sort_picks(ids, e)
        rows = piles.to_piles(x, p)
        out = piles.from_piles(rows, w, p)
        drows, dw = piles.from_piles_grad(out, rows, w, p)
        return p.order, p.place, p.offsets, rows, out, drows, dw, piles.to_piles_grad(drows, p)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in (6, 7, 8):
        ids.copy_(some_ids(t, k, e, seed))
        x.copy_(torch.randn(t, h, generator=gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    p = piles.sort_picks(ids, 3)
    x, rows, w = torch.randn(4, 8, device="cuda"), torch.randn(8, 8, device="cuda"), torch.randn(4, 2, device="cuda")
    bad = [lambda: piles.sort_picks(ids.long(), 3), lambda: piles.sort_picks(ids.cpu(), 3), lambda: piles.sort_picks(ids.t(), 3),
           lambda: piles.sort_picks(ids, 0), lambda: piles.sort_picks(ids, 1025), lambda: piles.sort_picks(ids[:, :0], 3),
           lambda: piles.to_piles(x[:3], p), lambda: piles.to_piles(x.double(), p), lambda: piles.to_piles(x.t(), p), lambda: piles.to_piles(x.cpu(), p),
           lambda: piles.from_piles(x, w, p), lambda: piles.from_piles(rows, w.double(), p), lambda: piles.from_piles(rows, w[:3], p), lambda: piles.from_piles(rows, w.view(2, 4), p),
           lambda: piles.from_piles_grad(x, rows, None, p), lambda: piles.from_piles_grad(x, rows.half(), w, p),
           lambda: piles.from_piles_grad(x, rows[:, :7], w, p), lambda: piles.from_piles_grad(rows, rows, w, p)]
    for call in bad:
        with pytest.raises(cw.CwError):
            call()
    assert piles.to_piles(x, p).shape == (8, 8)
