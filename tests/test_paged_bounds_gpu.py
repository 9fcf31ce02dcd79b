"""The paged operators at the ends of what their arguments may hold, in every kernel of the attention: one tile of 16 and of 32 rows,
whole and shared out; many rows, unsplit, split and shared out."""
import math

import pytest
import torch

import paged_reference as R
from test_paged_gpu import DEV, Pool, cu, i32, run_attention

pytestmark = pytest.mark.gpu
# heads, h_kv, d, page, past, new
KERNELS = [
    (4, 4, 64, 16, [20, 100], [3, 2]),
    (4, 4, 64, 16, [1400, 100], [3, 2]),
    (8, 1, 128, 64, [37, 30], [4, 3]),
    (8, 1, 128, 64, [37, 1500], [4, 3]),
    (4, 4, 64, 32, [20, 10], [150, 40]),
    (8, 2, 128, 64, [1800, 40], [40, 3]),
    (32, 4, 64, 16, [(37 * i) % 400 + 20 for i in range(34)], [5] * 34),
]


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import get_ops
    o = get_ops()
    assert o.name == "hip" and o.lib.sq_device_ready() == 1
    return o


def queries(heads, rows, d, dtype, seed=3):
    return torch.randn((heads, rows, d), generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("heads,h_kv,d,page,past,new", KERNELS)
def test_a_value_that_fp16_does_not_hold_reaches_who_sees_it(ops, heads, h_kv, d, page, past, new):
    """e4m3 rows stand for code * 2^(byte - 127), whoever wrote them: 448 * 2^13 is an infinity of fp16, wherever in a sequence it
    stands; 2^13 and smaller values beside it are not.  A result that an infinity is part of is not finite."""
    total = [p + n for p, n in zip(past, new)]
    for back in (1, 2):                                                  # the last stored row (everyone sees it), the chunk's second
        pool = Pool(total, h_kv, d, page, torch.float16, True, 91)
        codes, scales = torch.full(pool.pages[1].shape, 0x38, dtype=torch.uint8), torch.full(pool.scales[1].shape, 127, dtype=torch.uint8)
        for b, p in enumerate(past):
            at = p - 1 if back == 1 else p + 1
            codes[int(pool.table[b, at // page]), :, at % page, 5] = 0x7e
            codes[int(pool.table[b, at // page]), :, at % page, 9] = 0xfe
            scales[int(pool.table[b, at // page]), :, at % page] = 140
        pool.dev[1], pool.dev_scales[1] = codes.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)
        out = run_attention(ops, pool, queries(heads, sum(new), d, torch.float16).to(DEV), past, new, d ** -0.5, max_rows=max(new), max_len=max(total))
        out, t = out.view(-1, heads, d), 0
        for n in new:
            sees = torch.arange(n) >= (0 if back == 1 else 1)
            got = out[t:t + n]
            # (an infinity, or NaN where its weight is below what 16 bits hold beside the row's largest: 0 times an infinity)
            assert not bool(got[sees][:, :, [5, 9]].isfinite().any())
            assert not bool((got[sees][:, :, 5] == -math.inf).any() or (got[sees][:, :, 9] == math.inf).any())
            others = [i for i in range(d) if i not in (5, 9)]
            assert bool(got[~sees].isfinite().all()) and bool(got[:, :, others].isfinite().all())
            t += n


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30 + 5])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", KERNELS)
def test_a_length_of_any_size_sees_the_keys_that_count(ops, heads, h_kv, d, page, past, new, length):
    """Keys from max_len on are left out, however far the length goes beyond."""
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, torch.float16, False, 92)
    most = pool.width * page
    keys = [torch.arange(most)] + [torch.arange(t) for t in total[1:]]
    q = queries(heads, sum(new), d, torch.float16)
    out, t = run_attention(ops, pool, q.to(DEV), [length] + past[1:], new, d ** -0.5, max_rows=max(new), max_len=most), 0
    for b, n in enumerate(new):
        k, v = (R.stored(pool.pages[i], None, pool.table[b], keys[b]) for i in (0, 1))
        want, bound = R.attention(q[:, t:t + n].double(), k, v, past[b] if b else most, d ** -0.5, torch.float16)
        assert bool(((out[t:t + n].view(n, heads, d).double() - want).abs() <= bound).all()), b
        t += n


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", KERNELS)
def test_pages_outside_the_pool(ops, heads, h_kv, d, page, past, new, quantised):
    """Entries that name no page, in one sequence's table: its rows in front of them and the other sequences are right, nothing but the
    rows of the batch is written, the pages stay as they are."""
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, torch.bfloat16, quantised, 93)
    bad = -(-(past[0] + 1) // page)                                      # the first page behind the first new token's keys
    pool.table[0, bad:] = torch.tensor([-5, 1 << 30, -(2 ** 31), pool.n_pages] * (pool.width // 4 + 1), dtype=torch.int32)[:pool.width - bad]
    rows, cols = sum(new), heads * d
    q = queries(heads, rows, d, torch.bfloat16)
    guard = torch.full((rows + 4, cols + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    before = [t.view(torch.uint8).clone() for t in pool.dev]
    ops.paged_attention(q.to(DEV), out=guard[2:2 + rows, 4:4 + cols], seq_lens=i32(past), cu_rows=cu(new).to(DEV), scale=d ** -0.5, max_rows=max(new),
                        max_len=max(total), **pool.kw())
    torch.cuda.synchronize()
    for a, b in zip(pool.dev, before):
        assert torch.equal(a.view(torch.uint8), b)
    guard = guard.cpu()
    out = guard[2:2 + rows, 4:4 + cols].clone()
    guard[2:2 + rows, 4:4 + cols] = 3.0
    assert bool((guard == 3.0).all())
    t = 0
    for b, (p, n) in enumerate(zip(past, new)):
        seen = n if b else max(1, min(n, bad * page - p))                # rows whose keys all lie in front of the bad pages
        k, v = (R.stored(pool.pages[i], pool.scales[i], pool.table[b], torch.arange(p + seen)) for i in (0, 1))
        want, bound = R.attention(q[:, t:t + seen].double(), k, v, p, d ** -0.5, torch.bfloat16)
        assert bool(((out[t:t + seen].view(seen, heads, d).double() - want).abs() <= bound).all()), b
        t += n


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", KERNELS)
def test_a_call_repeats_itself_whatever_its_workspace_held(ops, heads, h_kv, d, page, past, new, quantised):
    """The same bits each time: the workspace comes from memory that held NaN, or zeros, or another call's sums."""
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, torch.float16, quantised, 94)
    q = queries(heads, sum(new), d, torch.float16).to(DEV)
    size = ops.lib.sq_paged_attention_workspace_bytes(len(new), sum(new), max(new), max(total), heads, h_kv, d)
    want = None
    for fill in (0, 0xff, None, 0x7f, None):
        if size and fill is not None:
            block = torch.full((size,), fill, dtype=torch.uint8, device=DEV)
            del block                                                    # the next allocation of this size
        got = run_attention(ops, pool, q, past, new, d ** -0.5, max_rows=max(new), max_len=max(total))
        want = got if want is None else want
        assert torch.equal(got, want)
