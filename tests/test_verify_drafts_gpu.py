"""Batched verification of drafted tokens on the GPU against the definition in 64 bits."""
import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import get_ops
    o = get_ops()
    assert o.name == "hip" and o.lib.sq_device_ready() == 1
    return o


def case(counts, vocab, dtype, seed, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    n, b = sum(counts), len(counts)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    owner = [i for i, c in enumerate(counts) for _ in range(c)]
    target = 2.0 * torch.randn((n + b, vocab), generator=g)
    draft = target[[i + o for i, o in enumerate(owner)]] + torch.randn((n, vocab), generator=g)
    if masked:
        target[torch.rand(target.shape, generator=g) < masked] = -math.inf
        target[:, 0] = 0.0
    target, draft = target.to(dtype), draft.to(dtype)
    tokens = torch.multinomial(torch.softmax(draft.float(), -1), 1, generator=g)[:, 0] if n else torch.zeros(0, dtype=torch.int64)
    return target, draft, tokens, cu, torch.rand((n,), generator=g), torch.rand((b,), generator=g)


def run(ops, target, draft, tokens, cu, ua, un, temperature):
    b = len(cu) - 1
    acc, nxt = torch.full((b,), -7, dtype=torch.int32, device=DEV), torch.full((b,), -7, dtype=torch.int64, device=DEV)
    t = torch.tensor(temperature, dtype=torch.float32, device=DEV) if isinstance(temperature, list) else temperature
    ops.verify_drafts(target.to(DEV), draft.to(DEV), tokens.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), ua.to(DEV), un.to(DEV), t, acc, nxt)
    torch.cuda.synchronize()
    return acc.cpu().tolist(), nxt.cpu().tolist()


def check(ops, target, draft, tokens, cu, ua, un, temperature):
    temps = torch.tensor(temperature if isinstance(temperature, list) else [temperature] * (len(cu) - 1), dtype=torch.float32).tolist()
    want_a, want_n, margin = R.verify(target, draft, tokens.tolist(), cu, ua.tolist(), un.tolist(), temps)
    # both sides compute in 64 bits: sums of up to 1.3e5 terms, each off by a few units in the last place -- 1e-12 holds with room
    assert margin > 1e-12, "the inputs put a decision on a border"
    got = run(ops, target, draft, tokens, cu, ua, un, temperature)
    assert got == (want_a, want_n)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,vocab", [([5], 32000), ([0], 7), ([1, 0, 3, 8], 1000), ([4] * 9, 4096), ([2, 6], 4097), ([3, 3], 50001),
                                          ([i % 4 for i in range(70)], 515), ([30], 2048), ([1], 128261)])
def test_matches_the_definition(ops, counts, vocab, dtype):
    acc, _ = check(ops, *case(counts, vocab, dtype, vocab + len(counts), masked=0.1), 0.7)
    assert all(0 <= a <= c for a, c in zip(acc, counts))


def test_temperatures_of_the_batch_greedy_among_them(ops):
    counts = [4] * 12
    t, d, tok, cu, ua, un = case(counts, 3001, torch.float16, 4)
    temps = [0.0, 0.3, 1.0, 2.5] * 3
    for b in range(0, 12, 4):                                          # the greedy ones agree for a while
        for i in range(b // 4 + 2):
            tok[cu[b] + i] = int(t[cu[b] + b + i].float().argmax())
    acc, _ = check(ops, t, d, tok, cu, ua, un, temps)
    assert acc[0] >= 2 and acc[4] >= 3
    check(ops, t, d, tok, cu, ua, un, 0)


def test_greedy_ties_go_to_the_lowest_index(ops):
    vocab = 9000
    t = torch.zeros((2, vocab))
    t[:, [4100, 8200, 4099]] = 3.0
    d = torch.zeros((1, vocab))
    half = torch.tensor([0.5])
    assert run(ops, t.half(), d.half(), torch.tensor([4099]), [0, 1], half, half, 0.0) == ([1], [4099])
    assert run(ops, t.half(), d.half(), torch.tensor([4100]), [0, 1], half, half, 0.0) == ([0], [4099])


@pytest.mark.parametrize("u", [0.0, 0.25, 1.0 - 2.0 ** -24])
def test_the_ends_of_the_uniforms(ops, u):
    """Exact distributions (powers of two): the draw at u = 0 is the first token with mass, at the largest u below 1 the last one."""
    vocab = 4100
    t = torch.full((1, vocab), -math.inf)
    t[0, [5, 17, 4097, 4099]] = 0.0
    one = torch.tensor([u])
    want = {0.0: 5, 0.25: 17}.get(u, 4099)                             # the running mass must exceed u: at exactly 1/4 the second
    got = run(ops, t, torch.zeros((0, vocab)), torch.zeros(0, dtype=torch.int64), [0, 0], torch.zeros(0), one, 1.0)
    assert got == ([0], [want])


def test_acceptance_is_strict_and_the_residual_leaves_the_rejected_token_out(ops):
    """p = (1/2, 1/2), q = (1, 0) up to the format: u q = p exactly is a rejection, and only token 1 has mass left."""
    t = torch.tensor([[0.0, 0.0, -math.inf], [0.0, -math.inf, -math.inf]])
    d = torch.tensor([[0.0, -math.inf, -math.inf]])
    tok, un = torch.tensor([0]), torch.tensor([0.0])
    assert run(ops, t, d, tok, [0, 1], torch.tensor([0.5]), un, 1.0) == ([0], [1])
    assert run(ops, t, d, tok, [0, 1], torch.tensor([0.5 - 2.0 ** -25]), un, 1.0) == ([1], [0])


def test_equal_rows_and_tokens_without_mass(ops):
    """p = q: everything with mass is accepted; a drafted token that has none is refused, and p itself is drawn from."""
    t, d, tok, cu, ua, un = case([3, 3], 600, torch.float16, 5)
    d = torch.stack([t[0], t[1], t[2], t[4], t[5], t[6]])
    assert run(ops, t, d, tok, cu, ua, un, 0.9)[0] == [3, 3]
    t[4, 11] = d[3, 11] = -math.inf
    tok[3] = 11
    acc, nxt = check(ops, t, d, tok, cu, ua, un, 0.9)
    assert acc == [3, 0] and nxt[1] != 11


def test_rows_that_are_no_distribution_and_tokens_outside_the_vocabulary(ops):
    vocab = 5000
    t, d, tok, cu, ua, un = case([2, 2, 2, 2, 2, 1], vocab, torch.float32, 6)
    ua.zero_()                                                         # u = 0: accepted wherever p > 0
    t[0, 4500] = math.nan                                              # sequence 0, first row
    t[4, 3] = math.inf                                                 # sequence 1, second row
    t[8] = -math.inf                                                   # sequence 2, the row behind its tokens
    tok[6] = vocab                                                     # sequence 3
    tok[8] = -1                                                        # sequence 4
    d[10, 7] = math.nan                                                # sequence 5: q is no distribution
    for temp in (1.0, 0.0):
        acc, nxt = run(ops, t, d, tok, cu, ua, un, temp)
        if temp:
            assert acc == [0, 1, 2, 0, 0, 0] and nxt[:3] == [-1, -1, -1] and nxt[5] == -1
            assert all(0 <= n < vocab for n in nxt[3:5])
        else:
            assert acc[0] == 0 and nxt[0] == -1 and acc[3] == acc[4] == 0 and all(0 <= n < vocab for n in nxt[3:])


def test_strided_rows_and_a_padded_batch(ops):
    """Logits as columns of a wider matrix, more rows than the offsets use, drafts that no sequence owns."""
    t, d, tok, cu, ua, un = case([3, 0, 2], 777, torch.bfloat16, 8)
    want = run(ops, t, d, tok, cu, ua, un, 0.8)
    wide_t, wide_d = torch.full((t.shape[0] + 4, 800), 9.0, dtype=t.dtype), torch.full((d.shape[0] + 4, 781), 9.0, dtype=t.dtype)
    wide_t[:t.shape[0], :777], wide_d[:d.shape[0], 1:778] = t, d
    tok2, ua2 = torch.cat([tok, torch.tensor([1, 2])]), torch.cat([ua, torch.zeros(2)])
    acc, nxt = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    ops.verify_drafts(wide_t.to(DEV)[:, :777], wide_d.to(DEV)[:, 1:778], tok2.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), ua2.to(DEV),
                      un.to(DEV), 0.8, acc, nxt)
    assert (acc.tolist(), nxt.tolist()) == want


def test_draws_follow_the_target(ops):
    """Speculation changes nothing: over many uniforms the first token out of (accepted draft | residual draw) has the target's
    distribution, whatever the draft's."""
    vocab, n = 12, 40000
    g = torch.Generator().manual_seed(12)
    tr, dr = 1.5 * torch.randn(vocab, generator=g), 1.5 * torch.randn(vocab, generator=g)
    p, q = torch.softmax(tr.double() / 0.8, 0), torch.softmax(dr.double() / 0.8, 0)
    tok = torch.multinomial(q, n, replacement=True, generator=g)
    target, draft = tr.expand(2 * n, vocab).contiguous(), dr.expand(n, vocab).contiguous()
    acc, nxt = run(ops, target, draft, tok, list(range(n + 1)), torch.rand(n, generator=g), torch.rand(n, generator=g), 0.8)
    first = [int(t) if a else x for t, a, x in zip(tok, acc, nxt)]
    seen = torch.bincount(torch.tensor(first), minlength=vocab).double()
    chi2 = float(((seen - n * p) ** 2 / (n * p)).sum())
    assert chi2 < 40.0, chi2                                           # 11 degrees of freedom: 1 in 3e4 is above 40


def test_replays_in_a_graph(ops):
    t, d, tok, cu, ua, un = case([4, 2, 7], 6000, torch.float16, 15)
    td, dd, tk, c, a, u = t.to(DEV), d.to(DEV), tok.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), ua.to(DEV), un.to(DEV)
    temps = torch.tensor([0.6, 0.0, 1.2], device=DEV)
    acc, nxt = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    ops.verify_drafts(td, dd, tk, c, a, u, temps, acc, nxt)           # loads the code
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(td, dd, tk, c, a, u, temps, acc, nxt)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        a.copy_(torch.rand(a.shape, generator=g))
        u.copy_(torch.rand(u.shape, generator=g))
        acc.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        want = run(ops, t, d, tok, cu, a.cpu(), u.cpu(), temps.cpu().tolist())
        assert (acc.tolist(), nxt.tolist()) == want


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,vocab", [([2, 0], 270001), ([1, 2], 8), ([2], 9), ([3, 1], 15), ([1] * 130, 21), ([2, 1], 513), ([40], 9000)])
def test_odd_and_very_wide_vocabularies(ops, counts, vocab, dtype):
    """More than 64 parts of a row and 512 blocks of tokens; rows that end inside a lane's eight tokens; more sequences than a wave."""
    check(ops, *case(counts, vocab, dtype, 3 * vocab + len(counts), masked=0.05), 0.9)


@pytest.mark.parametrize("vocab", [3000, 32000, 140000])
def test_a_long_chain_is_judged_to_its_end(ops, vocab):
    """u = 0 accepts whatever has mass: all tokens of a chain that takes several steps, up to the one planted without any."""
    counts = [70, 9, 33]
    t, d, tok, cu, ua, un = case(counts, vocab, torch.bfloat16, 31)
    ua.zero_()
    assert check(ops, t, d, tok, cu, ua, un, 0.8)[0] == counts
    t[66, tok[66]] = t[cu[2] + 2 + 32, tok[cu[2] + 32]] = -math.inf      # sequence 0's token 66, sequence 2's last
    assert check(ops, t, d, tok, cu, ua, un, 0.8)[0] == [66, 9, 32]
    check(ops, t, d, tok, cu, ua, un, 0.0)


@pytest.mark.parametrize("vocab", [5000, 40000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_whose_maximum_comes_late(ops, vocab, dtype):
    """The running maximum moves with every chunk of a row, by little and by so much that nothing before it counts; chunks and parts
    that hold nothing."""
    counts = [2] * 4
    t, d, tok, cu, ua, un = case(counts, vocab, dtype, 41)
    ramp = torch.linspace(-1.0, 1.0, vocab)
    for b, height in enumerate((4.0, 900.0, -30000.0)):
        t[3 * b:3 * b + 3] = (t[3 * b:3 * b + 3].float() * 0.2 + height * ramp).to(dtype)
        d[2 * b:2 * b + 2] = (d[2 * b:2 * b + 2].float() * 0.2 + height * ramp).to(dtype)
        tok[2 * b:2 * b + 2] = d[2 * b:2 * b + 2].float().argmax(-1)
    t[9:, :vocab - 700] = -math.inf
    d[6:, 100:] = -math.inf
    tok[6:] = 50
    check(ops, t, d, tok, cu, ua, un, 1.1)
    check(ops, t, d, tok, cu, ua, un, 0.0)
