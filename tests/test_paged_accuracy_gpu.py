"""What the rounding of the attention's weights may cost, sharply: with one rounding of a weight, of numerator and denominator alike,
a result is off by what the weights' roundings move between values -- not by a part of the value that all keys have in common -- and
by nothing of weights that are small beside the row's largest."""
import math

import pytest
import torch

import paged_reference as R
from test_paged_gpu import DEV, Pool, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import get_ops
    o = get_ops()
    assert o.name == "hip" and o.lib.sq_device_ready() == 1
    return o


def attention(q, k, v, past, scale, dtype):
    """q [H, n, D], k / v [H_kv, past + n, D] float64 -> (o [n, H, D], bound).  Element by element, with u = half a step of the element
    type, e = 2^-24, w_j the softmax weights:
      the output's rounding: half a step of its own binade
      a weight's rounding in a_j, |a_j| <= u, and below fp16's normal range 2^-25 of what the weights are multiplied by, 2^7 at least:
      sum w_j (1 + a_j) v_j / sum w_j (1 + a_j) - o = sum w_j a_j (v_j - o) / sum w_j (1 + a_j)
      weights off by a factor each before that rounding (fp32 scores of D products, exponentials; numerator and denominator alike):
      d = 2 (D + 4) e scale sum |q_i k_ij| + 4 e |s| + 4 e, times sum w_j |v_j - o| as well
      fp32 sums over n keys, at worst (n + 8) e of sum w_j |v_j| and of the denominator"""
    h, n, d = q.shape
    group = h // k.shape[0]
    kk, vv = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    keys = kk.shape[1]
    hidden = torch.arange(keys)[None, :] > past + torch.arange(n)[:, None]
    s = (torch.matmul(q, kk.transpose(1, 2).contiguous()) * scale).masked_fill(hidden, -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    w = w / total
    o = torch.matmul(w, vv)
    apart, unseen = torch.zeros_like(o), torch.zeros_like(o)
    for i in range(n):                                                   # |v_j - o|, row by row
        far = (vv - o[:, i:i + 1]).abs()
        apart[:, i] = torch.matmul(w[:, i:i + 1], far)[:, 0]
        unseen[:, i] = torch.matmul((~hidden[i]).double(), far)
    e, u = 2.0 ** -24, R.EPS[dtype]
    mag = torch.matmul(q.abs(), kk.abs().transpose(1, 2).contiguous()).masked_fill(hidden, 0.0) * scale
    off = (2 * (d + 4) * e * mag + 4 * e * s.masked_fill(hidden, 0.0).abs()).amax(-1, keepdim=True) + 4 * e
    tiny = 2.0 ** -32 if dtype == torch.float16 else 0.0
    inner = (u + 2 * off) * apart + tiny * unseen / total + 2 * (keys + 8) * e * torch.matmul(w, vv.abs())
    inner = inner * (1 + 4 * u)
    step = torch.exp2(torch.floor(torch.log2(o.abs() + inner)).clamp(min=-14 if dtype == torch.float16 else -126)) * u
    return o.transpose(0, 1), (step + inner).transpose(0, 1)


def check(pool, q, out, past, new, scale):
    t, (h, _, d) = 0, q.shape
    for b, (p, n) in enumerate(zip(past, new)):
        k, v = (R.stored(pool.pages[i], pool.scales[i], pool.table[b], torch.arange(p + n)) for i in (0, 1))
        want, bound = attention(q[:, t:t + n].double(), k, v, p, scale, q.dtype)
        off = (out[t:t + n].view(n, h, d).double() - want).abs() / bound
        assert bool((off <= 1.0).all()), (b, p, n, float(off.max()), float((off > 1.0).double().mean()))
        t += n


SHAPES = [
    # heads, h_kv, d, page, past, new: few rows (16, 32), with and without shared parts; many rows, unsplit, split and shared
    (8, 8, 64, 16, [2, 30, 140], [1, 1, 2]),
    (8, 2, 128, 64, [3, 700, 1500], [4, 1, 3]),
    (16, 2, 64, 32, [5, 900], [4, 4]),
    (8, 1, 128, 16, [1, 60], [9, 16]),
    (8, 1, 64, 64, [1400], [12]),
    (4, 4, 128, 64, [0, 37], [150, 90]),
    (32, 4, 64, 16, [(7 * i) % 300 + 1 for i in range(34)], [5] * 34),
]


@pytest.mark.parametrize("dtype,quantised", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", SHAPES)
def test_what_all_values_have_in_common_comes_back_whole(ops, heads, h_kv, d, page, past, new, dtype, quantised):
    """Values of 8 and a little: the little is all that roundings of weights may touch."""
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, quantised, 81)
    g = torch.Generator().manual_seed(82)
    if quantised:                                                        # codes of 8 and 9, of 16 and 18 half as large
        pool.pages[1] = (0x50 + torch.randint(0, 2, pool.pages[1].shape, generator=g) + 8 * torch.randint(0, 2, pool.pages[1].shape[:3], generator=g)[..., None]).to(torch.uint8)
        pool.scales = (pool.scales[0], (127 - ((pool.pages[1][..., 0] & 8) >> 3)).to(torch.uint8))
        pool.dev[1] = pool.pages[1].to(DEV).view(torch.float8_e4m3fn)
        pool.pages[1] = pool.pages[1].view(torch.float8_e4m3fn)
        pool.dev_scales[1] = pool.scales[1].to(DEV)
    else:
        pool.pages[1] = (8.0 + 0.25 * torch.rand(pool.pages[1].shape, generator=g)).to(dtype)
        pool.dev[1] = pool.pages[1].to(DEV)
    q = torch.randn((heads, sum(new), d), generator=g).to(dtype)
    out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, max_rows=max(new), max_len=max(total))
    check(pool, q, out, past, new, d ** -0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("above", [8.0, 17.0, 20.0])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", [(8, 8, 64, 64, [6000], [1]), (4, 2, 128, 16, [150, 4000], [3, 2]), (8, 1, 64, 64, [5000], [9]),
                                                        (4, 4, 64, 64, [3000], [140]), (32, 4, 64, 64, [(41 * i) % 700 + 300 for i in range(34)], [5] * 34)])
def test_many_small_weights_beside_a_large_one(ops, heads, h_kv, d, page, past, new, above, dtype):
    """The first key of every sequence stands out by `above` (e^17 = 2^24.5) and has a value of 0: what comes back is the others' share, all
    of it."""
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, False, 83)
    pool.pages[0] = torch.zeros_like(pool.pages[0])
    pool.pages[1] = torch.ones_like(pool.pages[1])
    for b in range(len(past)):
        first = int(pool.table[b, 0])
        pool.pages[0][first, :, 0, 0] = above
        pool.pages[1][first, :, 0] = 0.0
    pool.dev = [t.to(DEV) for t in pool.pages]
    q = torch.zeros((heads, sum(new), d))
    q[:, :, 0] = 1.0
    q = q.to(dtype)
    out = run_attention(ops, pool, q.to(DEV), past, new, 1.0, max_rows=max(new), max_len=max(total))
    check(pool, q, out, past, new, 1.0)
