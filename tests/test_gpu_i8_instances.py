"""The layer of 8-bit experts in every kernel instance that its rules can take (tests/test_i8_dispatch.py asserts that these sizes
take them): against the same formulas in 64 bits."""
import pytest
import torch

from coachwhip_amd import i8

from .test_gpu_i8 import DTYPES, Experts, rand_rows, say

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------------------ a few tokens: E, K, H, I, T

# each routing width (experts), row length of x and number of rows a wave of gate and up
GATEUP = [(E, 4, H, I, T) for E in (40, 300, 600) for H in (900, 1900, 2500, 4000) for I, T in ((61, 1), (300, 4), (300, 28))
          if not (H > 2048 and T == 28)]
# each length of the K hidden rows end to end and number of rows a wave of down; rows that are read twice
DOWN = [(64, 8, 4090, I, T) for I in (100, 200, 500) for T in (1, 4, 9)] + [(64, 8, 4090, 1000, T) for T in (1, 4)] + [
    (64, 8, 1000, 1500, 1), (64, 8, 1000, 2000, 2), (8, 1, 300, 16000, 1), (8, 2, 300, 6000, 2), (8, 2, 300, 8100, 1), (12, 3, 4000, 2600, 4), (12, 5, 700, 1500, 1),
    (12, 5, 700, 2400, 2), (16, 4, 3300, 1000, 5), (40, 32, 500, 100, 3), (40, 32, 500, 500, 1), (40, 3, 3999, 300, 9)]


@pytest.mark.parametrize("E,K,H,I,T", sorted(set(GATEUP + DOWN)))
def test_layer_of_a_few_tokens(E, K, H, I, T):
    say("few tokens", E, K, H, I, T)
    clamped = (H + I + T) % 2 == 1
    ex = Experts(E, H, I, "clamped" if clamped else "silu", clamped, E + H + I + T)
    x, logits = ex.inputs(T)
    for dtype in DTYPES if T == 4 else [torch.float32]:
        out, ids, w = ex.layer(K).forward(i8.I8Rows(*x, H), logits, dtype)
        ex.check(x, logits, K, True, out, ids, w)


# ------------------------------------------------------------------------------ many tokens: E, K, H, I, T, picks of the experts

# tiles of every number of 16-pick groups, whole and ragged; experts without picks
COUNTS = (1, 15, 16, 17, 32, 33, 48, 49, 63, 64, 65, 80, 81, 96, 97, 127, 128, 129, 144, 161, 193, 200, 257, 300, 0, 2)
GROUPED = [
    (64, 6, 700, 1100, 600, COUNTS, "clamped", True),    # four weight groups: blocks of columns with a rest, an odd number of steps
    (300, 10, 2050, 130, 400, COUNTS, "silu", False),
    (40, 4, 260, 1920, 700, COUNTS, "silu", True),
    (24, 4, 500, 300, 600, COUNTS[:21], "clamped", True),  # two weight groups
    (30, 5, 1030, 257, 500, COUNTS, "silu", False),
    (70, 2, 4200, 90, 30, (1, 2, 30, 17, 0), "silu", True),  # routed by the plan, at every width
    (400, 10, 4200, 40, 9, (9, 1, 0, 5), "clamped", False),
    (1024, 32, 4200, 16, 32, (32, 31, 16, 0, 1), "silu", False),
    (24, 8, 300, 200, 1300, COUNTS[:12], "silu", False),   # ids read twice
    (24, 10, 300, 200, 1300, COUNTS[:12], "clamped", True),  # picks not staged
]


def picked_logits(E, K, T, counts, g):
    """Logits whose picks are `counts` of the first experts (each at most T), and of the others what is left over: the picks one after
    the other, expert by expert, dealt to the tokens in turn."""
    counts = [min(c, T) for c in counts][:E]
    left, rest = T * K - sum(counts), E - len(counts)
    assert 0 <= left <= rest * T
    counts += [left // rest + (e < left % rest) for e in range(rest)] if rest else []
    order = torch.randperm(E, generator=g, device="cuda").cpu()
    expert = torch.cat([torch.full((c,), int(order[e])) for e, c in enumerate(counts)])
    logits = torch.randn(T, E, generator=g, device="cuda")
    token = torch.arange(T * K) % T
    logits[token.cuda(), expert.cuda()] += 12
    return logits, counts


def all_counts(E, K, T, counts):
    """The experts' numbers of picks, as picked_logits deals them."""
    counts = [min(c, T) for c in counts][:E]
    left, rest = T * K - sum(counts), E - len(counts)
    return counts + [left // rest + (e < left % rest) for e in range(rest)]


@pytest.mark.parametrize("E,K,H,I,T,counts,act,bias", GROUPED)
def test_layer_of_many_tokens(E, K, H, I, T, counts, act, bias):
    say("many tokens", E, K, H, I, T, act, bias)
    ex = Experts(E, H, I, act, bias, E + H + I + T)
    x = rand_rows(ex.g, T, H)
    logits, _ = picked_logits(E, K, T, counts, ex.g)
    for dtype in DTYPES if T == 600 else [torch.float32]:
        out, ids, w = ex.layer(K).forward(i8.I8Rows(*x, H), logits, dtype)
        assert sorted(torch.bincount(ids.reshape(-1).long(), minlength=E).tolist()) == sorted(all_counts(E, K, T, counts))
        ex.check(x, logits, K, True, out, ids, w)


@pytest.mark.parametrize("T", [5, 1100])
def test_the_bound_separates(T):
    """What the check of these tests refuses: nothing, the negative, neighbouring columns or tokens in each other's place, a hundredth
    too much, one output of another token."""
    E, K, H, I = 32, 4, 500, 300
    ex = Experts(E, H, I, "clamped", True, 11)
    x, logits = ex.inputs(T)
    out, ids, w = ex.layer(K).forward(i8.I8Rows(*x, H), logits, torch.float32)
    one = out.clone()
    one[T - 1, H - 1] = out[0, H - 1]
    ex.check(x, logits, K, True, out, ids, w)
    for wrong in (out * 0, -out, out.roll(1, 1), out.roll(1, 0), out * 1.01, one):
        with pytest.raises(AssertionError):
            ex.check(x, logits, K, True, wrong, ids, w)
