"""Batched verification over the whole range of temperatures and of logits' magnitudes: p and q depend on differences of logits alone,
however small T is or however large the logits are beside those differences."""
import math

import pytest
import torch

import paged_reference as R
from test_verify_drafts_gpu import case, run

pytestmark = pytest.mark.gpu
TEMPS = [0.7, 1e-3, 1e-6, 1e-8, 1e-12, 1e-16, 1e-20, 1e-30, 1e-45]             # (the last one: the smallest fp32 number, 2^-149)
LARGE = [(1e8, 10.0), (1e8, 0.01), (1e12, 1.0), (1e12, 1e5), (1e16, 1.0), (1e16, 1e9), (1e30, 1.0), (-1e30, 1e23), (3e38, 1e-20)]


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import get_ops
    o = get_ops()
    assert o.name == "hip" and o.lib.sq_device_ready() == 1
    return o


def on_a_border(ops, dtype, p_top, q_top, temperature):
    """p = 1/4 at four tokens of three parts of a row, q = 1/2 at two of them, all of it exact: u q = p is a rejection and the largest
    u below is none; what is left of p lies on the other two, half and half."""
    vocab, none = 9000, -math.inf
    t, d = torch.full((2, vocab), none), torch.full((1, vocab), none)
    t[0, [5, 4100, 8200, 8999]], t[1, [17, 8998]], d[0, [5, 8999]] = p_top, q_top, q_top
    t, d = t.to(dtype), d.to(dtype)
    for u, un, want in ((0.5, 0.5, ([0], [8200])), (0.5, 0.5 - 2.0 ** -25, ([0], [4100])), (0.5 - 2.0 ** -25, 0.5, ([1], [8998])),
                        (0.5 - 2.0 ** -25, 0.5 - 2.0 ** -25, ([1], [17]))):
        for token in (5, 8999):
            assert run(ops, t, d, torch.tensor([token]), [0, 1], torch.tensor([u]), torch.tensor([un]), temperature) == want, (u, un, token)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", TEMPS)
def test_exact_borders_at_any_temperature(ops, temperature, dtype):
    for p_top, q_top in ((9.3671875, 8.7109375), (-23.1, 24.9), (0.0, 3.3)):
        on_a_border(ops, dtype, p_top, q_top, temperature)


@pytest.mark.parametrize("top,temperature", LARGE)
def test_exact_borders_of_large_logits(ops, top, temperature):
    on_a_border(ops, torch.float32, top, top * 0.77, temperature)


def definition(target, draft, tokens, cu, ua, un, temps):
    """R.verify of the rows less their maxima, in 64 bits: the same distributions, and no rounding of x / T that matters."""
    less = lambda rows: rows.double() - rows.double().amax(-1, keepdim=True)
    return R.verify(less(target), less(draft), tokens.tolist(), cu, ua.tolist(), un.tolist(), torch.tensor(temps, dtype=torch.float32).tolist())


def with_plateaus(counts, vocab, dtype, seed, offset=0.0):
    """Random rows; the target's have six tokens at or a step or two under their maximum, the draft's four of them and two others, and
    it drew from these."""
    t, d, tok, cu, ua, un = case(counts, vocab, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    t, d = (t.float() + offset).to(dtype), (d.float() + offset).to(dtype)
    owner = [b for b, c in enumerate(counts) for _ in range(c)]

    def plant(row, places):
        value = row.float().max()
        for i, at in enumerate(places):
            v = value.to(dtype)
            for _ in range(i % 3):
                v = torch.nextafter(v.float(), torch.tensor(-math.inf)).to(dtype) if dtype == torch.float32 else v
            row[at] = v

    for r in range(t.shape[0]):
        plant(t[r], torch.randperm(vocab, generator=g)[:6])
    for i, b in enumerate(owner):
        top = t[i + b].float().topk(6).indices
        places = torch.cat((top[:4], torch.randperm(vocab, generator=g)[:2]))
        d[i, top] = d[i].float().min().to(dtype)
        plant(d[i], places[torch.randperm(6, generator=g)])
        tok[i] = places[int(torch.randint(0, 6, (1,), generator=g))]
    return t, d, tok, cu, ua, un


def check(ops, inputs, temperature):
    t, d, tok, cu, ua, un = inputs
    each = [temperature] * (len(cu) - 1)
    want_a, want_n, margin = definition(t, d, tok, cu, ua, un, each)
    assert margin > 1e-12, "the inputs put a decision on a border"
    assert run(ops, t, d, tok, cu, ua, un, temperature) == run(ops, t, d, tok, cu, ua, un, each) == (want_a, want_n)
    return want_a


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", TEMPS)
def test_any_temperature_matches_the_definition(ops, temperature, dtype):
    counts = [3, 0, 2, 5, 1, 4, 4, 2]
    check(ops, with_plateaus(counts, 9000, dtype, 71), temperature)
    check(ops, with_plateaus(counts, 37, dtype, 72), temperature)


@pytest.mark.parametrize("offset,temperature", LARGE)
def test_large_logits_match_the_definition(ops, offset, temperature):
    check(ops, with_plateaus([3, 0, 2, 5, 1, 4, 4, 2], 9000, torch.float32, 73, offset), temperature)


@pytest.mark.parametrize("temperature", [1e31, 1e34, 3e38])
def test_large_logits_at_large_temperatures(ops, temperature):
    """Steps of fp32 near 3e38 are 2e31 wide: the same order as these temperatures, or far under them."""
    check(ops, with_plateaus([3, 0, 2, 5, 1, 4, 4, 2], 9000, torch.float32, 74, 3e38), temperature)
    inputs = case([3, 0, 2, 5], 5000, torch.float32, 75)
    check(ops, (3e37 * inputs[0], 3e37 * inputs[1], *inputs[2:]), temperature)


def test_an_infinite_temperature_is_flat(ops):
    """Every token above -inf has the same mass."""
    t, d, tok, cu, ua, un = case([0, 0], 4000, torch.float16, 76)
    t[:, ::3] = -math.inf
    left = [i for i in range(4000) if i % 3]
    want = [left[int(float(u) * len(left))] for u in un]
    assert run(ops, t, d, tok, cu, ua, un, [math.inf, 1.0e38]) == ([0, 0], want)
