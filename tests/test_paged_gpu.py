"""The paged-cache operators on the GPU against plain 64-bit forms (tests/paged_reference.py states the bounds)."""
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


class Pool:
    """Pages of one layer with random contents, a table of distinct pages in random order, one page more than the table names."""

    def __init__(self, total, h_kv, d, page, dtype, quantised, seed, extra=1, width=None):
        g = torch.Generator().manual_seed(seed)
        n = len(total)
        self.width = width or max(1, max(-(-t // page) for t in total))
        self.n_pages = n * self.width + extra
        self.table = torch.randperm(self.n_pages, generator=g)[:n * self.width].to(torch.int32).view(n, self.width)
        shape = (self.n_pages, h_kv, page, d)
        self.scales = (None, None)
        if quantised:
            codes = [torch.randint(0, 256, shape, generator=g).to(torch.uint8) for _ in range(2)]
            self.pages = [torch.where(c & 127 == 127, c & 128, c).view(torch.float8_e4m3fn) for c in codes]
            self.scales = [torch.randint(115, 122, shape[:3], generator=g).to(torch.uint8) for _ in range(2)]
        else:
            self.pages = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
        self.dev = [t.view(torch.uint8).to(DEV).view(t.dtype) if quantised else t.to(DEV) for t in self.pages]
        self.dev_scales = [None if s is None else s.to(DEV) for s in self.scales]

    def kw(self):
        return dict(k_pages=self.dev[0], v_pages=self.dev[1], page_table=self.table.to(DEV), k_scales=self.dev_scales[0], v_scales=self.dev_scales[1])


def cu(counts):
    c = [0]
    for n in counts:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


# ---- write --------------------------------------------------------------------------------------------------------------
def run_write(ops, qkv, pool, past, new, heads, h_kv, d, cos, sin, pos, q_out):
    ops.rope_kv_write_paged(qkv, q_out, pool.dev[0], pool.dev[1], cos, sin, pos, pool.table.to(DEV), i32(past), cu(new).to(DEV), heads, h_kv, d,
                            k_scales=pool.dev_scales[0], v_scales=pool.dev_scales[1])
    torch.cuda.synchronize()


WRITE = [
    # heads, h_kv, d, page, past, new, rows behind the last sequence
    (12, 12, 64, 16, [0], [1], 0),
    (64, 8, 128, 64, [63, 0, 130], [1, 1, 1], 2),
    (20, 4, 128, 32, [5, 31, 0, 64], [40, 0, 17, 1], 3),
    (8, 1, 64, 256, [255, 1], [3, 300], 0),
    (15, 5, 128, 128, [7] * 70, [i % 3 for i in range(70)], 1),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new,behind", WRITE)
def test_write(ops, heads, h_kv, d, page, past, new, behind, dtype, quantised):
    g = torch.Generator().manual_seed(heads * 100 + page)
    rows, cols = sum(new) + behind, (heads + 2 * h_kv) * d
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, quantised, 3)
    wide = torch.randn((rows, cols + 24), generator=g)
    wide *= torch.exp(2 * torch.randn((rows, 1), generator=g))
    wide = wide.to(dtype)
    max_pos = max(p + n for p, n in zip(past, new)) + 1
    angle = torch.rand((max_pos, d), generator=g) * 6
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    pos = torch.tensor([p + i for p, n in zip(past, new) for i in range(n)] + [0] * behind, dtype=torch.int64)
    q_out = torch.full((heads, rows, d), 7.0, dtype=dtype, device=DEV)
    run_write(ops, wide.to(DEV)[:, :cols], pool, past, new, heads, h_kv, d, cos.to(DEV), sin.to(DEV), pos.to(DEV), q_out)
    x = wide[:, :cols].double().view(rows, -1, d)
    turned = R.rope(x[:, :heads + h_kv], cos[pos].double(), sin[pos].double())
    live = sum(new)
    # the products are exact in fp32: one rounding of their sum (2^-24 of it), one to the type
    u = R.EPS[dtype]
    want = turned[:live, :heads].transpose(0, 1)
    off = (q_out[:, :live].cpu().double() - want).abs()
    assert bool((off <= (u + 2.0 ** -23) * want.abs() + R.TINY[dtype]).all())
    assert bool((q_out[:, live:] == 7.0).all()), "rows behind the last sequence changed"
    keep = torch.ones(pool.pages[0].shape[:3], dtype=torch.bool)
    t = 0
    for b, (p, n) in enumerate(zip(past, new)):
        for i in range(n):
            at = (int(pool.table[b, (p + i) // page]), slice(None), (p + i) % page)
            keep[at] = False
            for which, exact in ((0, turned[t, heads:]), (1, x[t, heads + h_kv:])):
                got = pool.dev[which].cpu()[at]
                if not quantised:
                    assert bool(((got.double() - exact).abs() <= (u + 2.0 ** -23) * exact.abs() + R.TINY[dtype]).all())
                    if which:
                        assert torch.equal(got, exact.to(dtype))
                    continue
                byte = pool.dev_scales[which].cpu()[at]
                assert torch.equal(byte.long(), R.row_scale_byte(exact.float().double(), dtype))
                # half of e4m3's step: 2^-4 of the value, 2^-10 of the scale below the normal range; the fp32 sum before it
                val = R.decode(got.view(torch.uint8), byte)
                exact = exact.clamp(-R.TOP4[dtype], R.TOP4[dtype])
                bound = torch.maximum(exact.abs() * 2.0 ** -4, torch.exp2(byte.double() - 137)[:, None]) * (1 + 2.0 ** -20) + exact.abs() * 2.0 ** -23
                assert bool(((val - exact).abs() <= bound).all())
            t += 1
    for which in (0, 1):
        assert torch.equal(bits(pool.dev[which]).view(*keep.shape, -1)[keep], bits(pool.pages[which]).view(*keep.shape, -1)[keep])
        if quantised:
            assert torch.equal(pool.dev_scales[which].cpu()[keep], pool.scales[which][keep])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
def test_write_e4m3_special_rows(ops, dtype, d):
    """Rows of zeros, of one value, of the type's largest and smallest magnitudes, with infinities and NaN: the codes are the
    nearest ones (ties to even), what is not finite reads back as NaN and leaves the others alone, nothing reads back as infinity."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal / 4
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(d), torch.full((d,), big), torch.full((d,), -small), torch.linspace(-1, 1, d) * big, torch.randn(d, generator=g),
            torch.full((d,), 448.0), torch.full((d,), 449.0), torch.full((d,), 1.75), torch.full((d,), 1.7578125)]
    mixed = torch.randn(d, generator=g)
    mixed[0], mixed[d // 2], mixed[3] = math.inf, -math.inf, math.nan
    ties = torch.tensor([448.0] + [(1 + (2 * i + 1) / 16) * 2.0 ** (i % 9) for i in range(d - 1)]).clamp(max=448.0)
    rows += [mixed, torch.full((d,), math.nan), torch.full((d,), math.inf), ties]
    v = torch.stack(rows).to(dtype)
    n = len(rows)
    qkv = torch.cat([torch.randn((n, 2 * d), generator=g).to(dtype), v], dim=1).to(DEV)
    pool = Pool([n], 1, d, 16, dtype, True, 4)
    one = torch.ones((n, d), dtype=dtype, device=DEV)
    pos = torch.arange(n, device=DEV)
    run_write(ops, qkv, pool, [0], [n], 1, 1, d, one, torch.zeros_like(one), pos, torch.empty((1, n, d), dtype=dtype, device=DEV))
    x, page = v.double(), int(pool.table[0, 0])
    byte, codes = pool.dev_scales[1].cpu()[page, 0, :n], pool.dev[1].cpu()[page, 0, :n].view(torch.uint8)
    assert torch.equal(byte.long(), R.row_scale_byte(x, dtype))
    val = R.decode(codes, byte)
    assert torch.equal(val.isnan(), ~x.isfinite())
    grid = R.e4m3_values()
    grid = grid[~grid.isnan()].unique()
    for r in range(n):
        scale = 2.0 ** (float(byte[r]) - 127)
        for j in range(d):
            if not x[r, j].isfinite():
                continue
            y = float(x[r, j].clamp(-R.TOP4[dtype], R.TOP4[dtype])) / scale
            near = (grid - y).abs()
            best = near.min()
            options = grid[near == best]
            if len(options) == 2:                      # a tie: the one whose last mantissa bit is even
                step = float((options[1] - options[0]).abs())
                options = options[(options / step).round() % 2 == 0]
            assert float(val[r, j]) / scale in [float(o) for o in options], (r, j, y)
    back = torch.empty((1, 1, n, d), dtype=dtype, device=DEV)
    ops.kv_read_paged(k_out=torch.empty_like(back), v_out=back, starts=i32([0]), counts=i32([n]), **pool.kw())
    got = back.cpu()[0, 0]
    assert not bool(got.isinf().any())
    assert torch.equal(got.isnan(), val.isnan())
    assert torch.equal(got[~got.isnan()], val.to(dtype)[~val.isnan()])


def test_write_keeps_to_its_bounds(ops):
    """Table entries outside the pool and position ids outside the tables: such rows are left out or brought inside; the others
    are written as ever."""
    d, page, dtype = 64, 16, torch.float16
    pool = Pool([40], 2, d, page, dtype, False, 8, extra=3)
    table = pool.table.clone()
    table[0, 1] = pool.n_pages                          # rows 16..31 have no page
    table[0, 2] = -1                                    # rows 32.. neither
    n = 40
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((n, 6 * d), generator=g).to(dtype)
    cos, sin = torch.ones((4, d), dtype=dtype), torch.zeros((4, d), dtype=dtype)
    pos = torch.arange(n) - 3
    pos[-1], pos[-2] = 1 << 40, -(1 << 40)
    q = torch.empty((2, n, d), dtype=dtype, device=DEV)
    ops.rope_kv_write_paged(qkv.to(DEV), q, pool.dev[0], pool.dev[1], cos.to(DEV), sin.to(DEV), pos.to(DEV), table.to(DEV), i32([0]), i32([0, n]), 2, 2, d)
    torch.cuda.synchronize()
    want = [p.clone() for p in pool.pages]
    for which in (0, 1):
        want[which][int(table[0, 0]), :, :] = qkv[:16, (2 + 2 * which) * d:(4 + 2 * which) * d].view(16, 2, d).transpose(0, 1)
        assert torch.equal(bits(pool.dev[which]), bits(want[which]))
    assert torch.equal(q.cpu(), qkv[:, :2 * d].view(n, 2, d).transpose(0, 1))


# ---- read ---------------------------------------------------------------------------------------------------------------
READ = [
    # h_kv, d, page, starts, counts, rows of the output
    (12, 64, 16, [0], [1], 1),
    (8, 128, 64, [0, 7, 100], [230, 0, 33], 240),
    (1, 64, 256, [255, 300], [258, 1], 258),
    (4, 128, 32, [31], [97], 100),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("h_kv,d,page,starts,counts,m", READ)
def test_read(ops, h_kv, d, page, starts, counts, m, dtype, quantised):
    pool = Pool([s + c for s, c in zip(starts, counts)], h_kv, d, page, dtype, quantised, 11)
    n = len(starts)
    # outputs as layers of a larger cache: the head stride is the slab's, not m * d
    ko, vo = (torch.full((n, h_kv, m + 3, d), 5.0, dtype=dtype, device=DEV)[:, :, :m] for _ in range(2))
    ops.kv_read_paged(k_out=ko, v_out=vo, starts=i32(starts), counts=i32(counts), **pool.kw())
    torch.cuda.synchronize()
    for which, out in ((0, ko.cpu()), (1, vo.cpu())):
        for b in range(n):
            want = R.stored(pool.pages[which], pool.scales[which], pool.table[b], torch.arange(starts[b], starts[b] + counts[b]))
            assert torch.equal(out[b, :, :counts[b]], want.to(dtype))
            assert bool((out[b, :, counts[b]:] == 5.0).all())
    assert bool((ko._base[:, :, m:] == 5.0).all())


def test_read_every_code_and_scale(ops):
    """All 256 codes under scales from the smallest to the largest a type's rows have."""
    d, page = 128, 16
    codes = torch.arange(256, dtype=torch.uint8)
    for dtype, lo, hi in ((torch.float16, 90, 135), (torch.bfloat16, 1, 247)):
        scales = list(range(lo, hi + 1))
        n = 2 * len(scales)
        pages_n = -(-n // page)
        pool = Pool([n], 1, d, page, dtype, True, 2)
        all_codes = codes.view(2, d).repeat(len(scales), 1)
        all_scales = torch.tensor(scales, dtype=torch.uint8).repeat_interleave(2)
        k = torch.zeros((pool.n_pages, 1, page, d), dtype=torch.uint8)
        s = torch.full((pool.n_pages, 1, page), 127, dtype=torch.uint8)
        for r in range(n):
            k[int(pool.table[0, r // page]), 0, r % page] = all_codes[r]
            s[int(pool.table[0, r // page]), 0, r % page] = all_scales[r]
        kd = k.to(DEV).view(torch.float8_e4m3fn)
        out = torch.empty((1, 1, n, d), dtype=dtype, device=DEV)
        ops.kv_read_paged(kd, kd, out, torch.empty_like(out), pool.table.to(DEV), i32([0]), i32([n]), k_scales=s.to(DEV), v_scales=s.to(DEV))
        got, want = out.cpu()[0, 0], R.decode(all_codes, all_scales).to(dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()]), dtype
        assert pages_n == pool.width


# ---- attention ----------------------------------------------------------------------------------------------------------
def run_attention(ops, pool, q, past, new, scale, behind=0, **kw):
    rows = sum(new) + behind
    h, _, d = q.shape
    out = torch.full((rows, h * d), 3.0, dtype=q.dtype, device=DEV)
    ops.paged_attention(q, pool.dev[0], pool.dev[1], out, pool.table.to(DEV), i32(past), cu(new).to(DEV), scale, k_scales=pool.dev_scales[0],
                        v_scales=pool.dev_scales[1], **kw)
    torch.cuda.synchronize()
    return out.cpu()


def check_attention(pool, q, out, past, new, scale):
    t = 0
    h, _, d = q.shape
    for b, (p, n) in enumerate(zip(past, new)):
        if not n:
            continue
        k, v = (R.stored(pool.pages[i], pool.scales[i], pool.table[b], torch.arange(p + n)) for i in (0, 1))
        want, bound = R.attention(q[:, t:t + n].double(), k, v, p, scale, q.dtype)
        got = out[t:t + n].view(n, h, d).double()
        worst = float(((got - want).abs() / bound).max())
        assert worst <= 1.0, (b, p, n, worst)
        t += n
    assert bool((out[t:] == 3.0).all()), "rows behind the last sequence changed"


ATTEND = [
    # heads, h_kv, d, page, past, new, rows behind
    (12, 12, 64, 16, [0], [1], 0),
    (12, 12, 64, 16, [143], [1], 0),
    (64, 8, 128, 64, [299, 0, 1023, 64, 63], [1, 1, 1, 0, 1], 2),
    (32, 32, 128, 32, [100, 31, 517], [7, 1, 5], 0),
    (32, 8, 128, 16, [3000], [1], 0),
    (8, 1, 64, 128, [700, 20], [3, 4], 1),
    (20, 4, 128, 256, [255, 40], [6, 33], 0),
    (16, 2, 64, 32, [0, 65], [130, 64], 5),
    (15, 5, 128, 64, [129], [200], 0),
    (4, 4, 128, 64, [0, 1, 190], [257, 128, 129], 0),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new,behind", ATTEND)
def test_attention(ops, heads, h_kv, d, page, past, new, behind, dtype, quantised):
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, quantised, 21)
    g = torch.Generator().manual_seed(9)
    q = (1.5 * torch.randn((heads, sum(new) + behind, d), generator=g)).to(dtype)
    out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, behind, max_rows=max(new), max_len=max(p + n for p, n in zip(past, new)))
    check_attention(pool, q, out, past, new, d ** -0.5)
    again = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, behind)          # the default bounds: another split, same result
    check_attention(pool, q, again, past, new, d ** -0.5)


LONG = [
    # heads, h_kv, d, page, past, new: parts of one KV head's keys in hundreds of workgroups, in two row tiles, in the tiled kernel
    (4, 1, 64, 64, [70001], [1]),
    (2, 1, 128, 16, [20000, 3], [2, 1]),
    (8, 1, 64, 32, [3000, 511], [3, 4]),
    (8, 1, 128, 256, [9000], [6]),
    (16, 2, 128, 64, [2047, 0, 600], [9, 20, 16]),
]


@pytest.mark.parametrize("dtype,quantised", [(torch.float16, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", LONG)
def test_attention_over_many_parts(ops, heads, h_kv, d, page, past, new, dtype, quantised):
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, quantised, 22)
    q = (1.5 * torch.randn((heads, sum(new), d), generator=torch.Generator().manual_seed(9))).to(dtype)
    for bounds in (dict(max_rows=max(new), max_len=max(p + n for p, n in zip(past, new))), {}):
        out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, **bounds)
        check_attention(pool, q, out, past, new, d ** -0.5)


@pytest.mark.parametrize("heads,h_kv,d,most", [(8, 8, 64, 2), (16, 2, 128, 1), (8, 1, 128, 4), (6, 2, 64, 30)])
def test_attention_of_many_sequences(ops, heads, h_kv, d, most):
    """More sequences than a wave has lanes, some without rows, lengths from nothing to many steps: every key is somebody's."""
    import random
    rng = random.Random(heads * d + most)
    n = 150
    new = [rng.choice((0, 0, 1, rng.randint(1, most))) for _ in range(n)]
    past = [rng.choice((0, rng.randint(0, 40), rng.randint(0, 900))) for _ in range(n)]
    new[0] = new[-1] = 0
    dtype = torch.float16
    pool = Pool([p + m for p, m in zip(past, new)], h_kv, d, 32, dtype, False, 23)
    q = torch.randn((heads, sum(new) + 3, d), generator=torch.Generator().manual_seed(1)).to(dtype)
    for bounds in (dict(max_rows=most, max_len=max(p + m for p, m in zip(past, new))), {}):
        out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, 3, **bounds)
        check_attention(pool, q, out, past, new, d ** -0.5)


@pytest.mark.parametrize("heads,h_kv,most", [(4, 4, 1), (8, 1, 4), (4, 1, 40)])
def test_attention_with_offsets_that_name_no_rows(ops, heads, h_kv, most):
    """Offsets outside the batch, a sequence with more rows than max_rows: such rows are left out, the other sequences' results and
    everything else stay what they are."""
    d, page, dtype = 64, 16, torch.float16
    past, new = [500, 300, 700], [most, most, most]
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, False, 24)
    rows = sum(new)
    q = torch.randn((heads, rows, d), generator=torch.Generator().manual_seed(2)).to(dtype)
    good = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, max_rows=most, max_len=740)
    for offsets in ([0, most, 2 * most, 1 << 30], [-5, most, 2 * most, rows], [0, most, 2 * most, 2 * most - 1]):
        out = torch.full((rows, heads * d), 3.0, dtype=dtype, device=DEV)
        ops.paged_attention(q.to(DEV), pool.dev[0], pool.dev[1], out, pool.table.to(DEV), i32(past), i32(offsets), d ** -0.5, max_rows=most, max_len=740)
        out = out.cpu()
        for b in range(3):
            mine = slice(b * most, (b + 1) * most)
            if offsets[b] == b * most and offsets[b + 1] == (b + 1) * most:
                worst = (out[mine].double() - good[mine].double()).abs().max()       # the shares differ, so the sums' order may
                assert float(worst) <= 2.0 ** -8, (offsets, b)
            else:
                assert bool((out[mine] == 3.0).all()), (offsets, b)
    if heads // h_kv * (most - 1) <= 32 and most > 1:
        out = torch.full((rows, heads * d), 3.0, dtype=dtype, device=DEV)
        ops.paged_attention(q.to(DEV), pool.dev[0], pool.dev[1], out, pool.table.to(DEV), i32(past), cu(new).to(DEV), d ** -0.5, max_rows=1, max_len=740)
        got = out.cpu().view(rows, heads, d)
        k, v = (R.stored(pool.pages[i], None, pool.table[0], torch.arange(501)) for i in (0, 1))
        want, bound = R.attention(q[:, :1].double(), k, v, 500, d ** -0.5, dtype)
        assert bool(((got[:1].double() - want).abs() <= bound).all())                 # the first row is there whatever the bound


@pytest.mark.parametrize("dtype,quantised", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True), (torch.bfloat16, True)])
@pytest.mark.parametrize("heads,h_kv,d,page,past,new", [
    (64, 8, 128, 64, [300, 1900, 0, 64, 63, 700, 5, 1100] * 2, [5, 6, 5, 1, 6, 0, 8, 7] * 2),       # 33 to 64 rows of shared heads
    (64, 8, 128, 64, [300, 1900, 0, 64], [5, 6, 5, 8]),                                             # (few units)
    (8, 1, 64, 16, [1000, 31, 250, 200] * 35, [12, 11, 1, 9] * 35),                                 # to 96, pages shorter than a tile
    (32, 2, 128, 32, [500, 800] * 33, [8, 7] * 33),                                                 # 128, all of a tile
    (12, 12, 64, 256, [900, 2000, 130] * 4, [40, 33, 100] * 4),                                     # no sharing
    (16, 2, 128, 128, [1500, 0] * 35, [7, 5] * 35),
])
def test_attention_of_a_few_tokens_of_shared_heads(ops, heads, h_kv, d, page, past, new, dtype, quantised):
    """33 to 128 rows a sequence and KV head: the keys of between 128 and 512 such units are shared out evenly too."""
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, quantised, 31)
    q = torch.randn((heads, sum(new) + 2, d), generator=torch.Generator().manual_seed(6)).to(dtype)
    for bounds in (dict(max_rows=max(new), max_len=max(p + n for p, n in zip(past, new))), dict(max_rows=max(new))):
        check_attention(pool, q, run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, 2, **bounds), past, new, d ** -0.5)


@pytest.mark.parametrize("quantised", [False, True])
def test_attention_of_many_sequences_with_shared_heads(ops, quantised):
    """Units of every length, none among them, fewer and more than the workgroups that fit the card."""
    rng = __import__("random").Random(7)
    n, heads, h_kv, d, dtype = 110 if quantised else 150, 24, 4, 64, torch.float16
    new = [rng.randint(0, 9) for _ in range(n)]
    past = [rng.choice((0, rng.randint(0, 70), rng.randint(200, 900))) for _ in range(n)]
    new[0] = new[-1] = 0
    pool = Pool([p + m for p, m in zip(past, new)], h_kv, d, 64, dtype, quantised, 33)
    q = torch.randn((heads, sum(new) + 3, d), generator=torch.Generator().manual_seed(2)).to(dtype)
    out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, 3, max_rows=9, max_len=max(p + m for p, m in zip(past, new)))
    check_attention(pool, q, out, past, new, d ** -0.5)


@pytest.mark.parametrize("heads,h_kv,new", [(4, 4, 3), (8, 1, 2), (2, 2, 40)])
def test_attention_of_a_length_below_zero(ops, heads, h_kv, new):
    """Rows that see nothing are zeros, also where a whole sequence has no key and its neighbours are split."""
    d, page, dtype = 64, 16, torch.float16
    past, news = [700, 0, 600], [new] * 3
    pool = Pool([p + n for p, n in zip(past, news)], h_kv, d, page, dtype, False, 25)
    q = torch.randn((heads, 3 * new, d), generator=torch.Generator().manual_seed(3)).to(dtype)
    for below in (1, new, new + 5, 1 << 30):
        out = torch.full((3 * new, heads * d), 3.0, dtype=dtype, device=DEV)
        ops.paged_attention(q.to(DEV), pool.dev[0], pool.dev[1], out, pool.table.to(DEV), i32([700, -below, 600]), cu(news).to(DEV), d ** -0.5,
                            max_rows=new, max_len=740)
        got = out.cpu()
        assert bool((got[new:new + min(below, new)] == 0).all()), below
        for b in (0, 2):
            k, v = (R.stored(pool.pages[i], None, pool.table[b], torch.arange(past[b] + new)) for i in (0, 1))
            want, bound = R.attention(q[:, b * new:(b + 1) * new].double(), k, v, past[b], d ** -0.5, dtype)
            assert bool(((got[b * new:(b + 1) * new].view(new, heads, d).double() - want).abs() <= bound).all()), (below, b)


@pytest.mark.parametrize("past,new", [([5000], [1]), ([2500, 40], [17, 2]), ([900], [150])])
def test_attention_sharp_and_flat_rows(ops, past, new):
    """Scores of hundreds (one key holds all the weight, maxima that rise late) and of 0 (every key the same weight)."""
    heads, h_kv, d, page, dtype = 8, 2, 128, 64, torch.float16
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, False, 33)
    ramp = torch.zeros_like(pool.pages[0])
    for b, t in enumerate(total):
        for j in range(t):
            ramp[int(pool.table[b, j // page]), :, j % page, 0] = 8.0 * j / t - 4.0
    pool.pages[0] = (pool.pages[0] + ramp).to(dtype)
    pool.dev[0] = pool.pages[0].to(DEV)
    g = torch.Generator().manual_seed(2)
    q = torch.randn((heads, sum(new), d), generator=g)
    q[:, :, 0] += 300.0
    q[1] = 0.0
    q = q.to(dtype)
    out = run_attention(ops, pool, q.to(DEV), past, new, d ** -0.5, max_rows=max(new), max_len=max(total))
    check_attention(pool, q, out, past, new, d ** -0.5)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,h_kv,d,past,new", [(8, 8, 128, [40], [5]), (8, 1, 64, [100, 7], [4, 9]), (4, 4, 128, [70], [140]),
                                                   (16, 2, 64, [3], [80]), (4, 4, 64, [0], [300])])
def test_attention_what_a_row_does_not_see_does_not_reach_it(ops, heads, h_kv, d, past, new, quantised):
    """Infinities and NaN in keys and values behind a sequence's end and in rows that causality hides: a row's result is what it
    would be without them, bit for bit; the rows that do see them carry them."""
    page, dtype = 16, torch.float16
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, quantised, 41, width=max(-(-t // page) for t in total) + 1)
    g = torch.Generator().manual_seed(3)
    q = torch.randn((heads, sum(new), d), generator=g).to(dtype).to(DEV)
    kw = dict(max_rows=max(new), max_len=max(total))
    clean = run_attention(ops, pool, q, past, new, d ** -0.5, **kw)
    check_attention(pool, q.cpu(), clean, past, new, d ** -0.5)
    bad = torch.tensor([0x7f, 0xff], dtype=torch.uint8) if quantised else torch.tensor([math.nan, math.inf, -math.inf]).to(dtype)

    def poison(first):
        """Every row of sequence b from first[b] on, to the end of its pages."""
        for which in (0, 1):
            t = pool.pages[which].clone().view(torch.uint8) if quantised else pool.pages[which].clone()
            for b in range(len(total)):
                for j in range(first[b], pool.width * page):
                    at = (int(pool.table[b, j // page]), slice(None), j % page, slice(j % 3, None, 5))
                    t[at] = bad[j % len(bad)]
            pool.dev[which] = t.to(DEV).view(torch.float8_e4m3fn) if quantised else t.to(DEV)

    poison(total)
    assert torch.equal(run_attention(ops, pool, q, past, new, d ** -0.5, **kw), clean)
    seen = [max(1, n // 2) for n in new]                                # the first rows see none of the poisoned ones
    poison([p + s for p, s in zip(past, seen)])
    got, t = run_attention(ops, pool, q, past, new, d ** -0.5, **kw), 0
    for n, s in zip(new, seen):
        assert torch.equal(got[t:t + s], clean[t:t + s])
        assert bool(got[t + s:t + n].isnan().view(n - s, -1).any(-1).all())
        t += n


@pytest.mark.parametrize("quantised", [False, True])
def test_attention_of_shared_keys_keeps_hidden_rows_apart(ops, quantised):
    """The same where many sequences' keys are shared out over the workgroups: behind every sequence's end, and in its last token, which
    the others of its chunk do not see."""
    heads, h_kv, d, page, dtype, past, new = 16, 2, 64, 32, torch.float16, [3, 300, 61, 127] * 17, [6, 5, 3, 8] * 17
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, quantised, 43, width=max(-(-t // page) for t in total) + 1)
    q = torch.randn((heads, sum(new), d), generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    kw = dict(max_rows=max(new), max_len=max(total))
    clean = run_attention(ops, pool, q, past, new, d ** -0.5, **kw)
    check_attention(pool, q.cpu(), clean, past, new, d ** -0.5)
    last = torch.tensor([sum(new[:b + 1]) - 1 for b in range(len(new))])
    before = torch.ones(sum(new), dtype=torch.bool)
    before[last] = False
    for back in (0, 1):                                      # from the end on, from the last token on
        for which in (0, 1):
            t = pool.pages[which].clone().view(torch.uint8) if quantised else pool.pages[which].clone()
            for b in range(len(total)):
                for j in range(total[b] - back, min(total[b] + 40, pool.width * page)):
                    t[int(pool.table[b, j // page]), :, j % page, ::5] = 0x7f if quantised else (math.inf if which else math.nan)
            pool.dev[which] = t.to(DEV).view(torch.float8_e4m3fn) if quantised else t.to(DEV)
        got = run_attention(ops, pool, q, past, new, d ** -0.5, **kw)
        if back == 0:
            assert torch.equal(got, clean)
        else:
            assert torch.equal(got[before], clean[before]) and not bool(got[last].isfinite().all(-1).any())


def test_attention_hidden_infinite_value_stays_an_infinity_where_it_is_seen(ops):
    heads, h_kv, d, page, dtype = 2, 1, 64, 16, torch.float16
    pool = Pool([20], h_kv, d, page, dtype, False, 5)
    pool.pages[1][int(pool.table[0, 1]), 0, 2, 7] = math.inf            # row 18, column 7
    pool.pages[1][int(pool.table[0, 1]), 0, 2, 9] = -math.inf
    pool.dev[1] = pool.pages[1].to(DEV)
    q = torch.randn((heads, 10, d), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    out = run_attention(ops, pool, q, [10], [10], d ** -0.5).view(10, heads, d)
    assert bool(out[:8].isfinite().all())
    assert bool((out[8:, :, 7] == math.inf).all() and (out[8:, :, 9] == -math.inf).all())
    assert bool(out[8:, :, [i for i in range(d) if i not in (7, 9)]].isfinite().all())


def test_attention_strided_queries_and_output(ops):
    heads, h_kv, d, page, dtype, past, new = 8, 2, 64, 32, torch.bfloat16, [70, 3], [5, 40]
    pool = Pool([p + n for p, n in zip(past, new)], h_kv, d, page, dtype, False, 51)
    rows = sum(new)
    g = torch.Generator().manual_seed(6)
    wide = torch.randn((rows, heads * d + 16), generator=g).to(dtype).to(DEV)
    q = wide[:, :heads * d].view(rows, heads, d).transpose(0, 1)        # rows major, as a projection leaves them
    out = torch.full((rows, heads * d + 4), 3.0, dtype=dtype, device=DEV)
    ops.paged_attention(q, out=out[:, :heads * d], seq_lens=i32(past), cu_rows=cu(new).to(DEV), scale=d ** -0.5, **pool.kw())
    check_attention(pool, q.cpu(), out.cpu()[:, :heads * d], past, new, d ** -0.5)
    assert bool((out[:, heads * d:] == 3.0).all())


def test_attention_of_one_row_and_one_head_of_any_strides(ops):
    """A dimension of one element has no stride that matters."""
    d, dtype = 64, torch.float16
    pool = Pool([300], 1, d, 16, dtype, False, 27)
    q = torch.randn((1, 1, d), generator=torch.Generator().manual_seed(5)).to(dtype)
    odd = torch.empty(512, dtype=dtype, device=DEV).as_strided((1, 1, d), (3, 5, 1)).copy_(q)
    check_attention(pool, q, run_attention(ops, pool, odd, [299], [1], d ** -0.5), [299], [1], d ** -0.5)


def test_attention_and_write_in_a_cache_past_32_bit_offsets(ops):
    """A pool of more than 2^32 bytes (and 2^31 elements): the pages at its end hold what is written and attended."""
    h_kv, d, page, dtype = 8, 128, 256, torch.float16
    n_pages = (1 << 31) // (h_kv * page * d) + 3
    k, v = (torch.empty((n_pages, h_kv, page, d), dtype=dtype, device=DEV) for _ in range(2))
    assert k.numel() > 1 << 31
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device=DEV)
    n = 300
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn((n, 3 * h_kv * d), generator=g).to(dtype)
    one = torch.ones((n, d), dtype=dtype, device=DEV)
    q = torch.empty((h_kv, n, d), dtype=dtype, device=DEV)
    ops.rope_kv_write_paged(qkv.to(DEV), q, k, v, one, torch.zeros_like(one), torch.arange(n, device=DEV), table, i32([0]), i32([0, n]), h_kv, h_kv, d)
    ko, vo = (torch.empty((1, h_kv, n, d), dtype=dtype, device=DEV) for _ in range(2))
    ops.kv_read_paged(k, v, ko, vo, table, i32([0]), i32([n]))
    parts = qkv.view(n, 3, h_kv, d).permute(1, 2, 0, 3)
    assert torch.equal(ko.cpu()[0], parts[1]) and torch.equal(vo.cpu()[0], parts[2])
    out = torch.empty((n, h_kv * d), dtype=dtype, device=DEV)
    ops.paged_attention(q, k, v, out, table, i32([0]), i32([0, n]), d ** -0.5)
    want, bound = R.attention(parts[0].double(), parts[1].double(), parts[2].double(), 0, d ** -0.5, dtype)
    assert bool(((out.cpu().view(n, h_kv, d).double() - want).abs() <= bound).all())


def test_attention_bounds_that_cut_and_bad_pages(ops):
    """max_rows and max_len are bounds of the launch: rows and keys beyond them are left out, nothing else is touched; a table
    entry outside the pool is not followed."""
    heads, h_kv, d, page, dtype = 4, 4, 64, 16, torch.float16
    pool = Pool([64, 64], h_kv, d, page, dtype, False, 61)
    q = torch.randn((heads, 20, d), generator=torch.Generator().manual_seed(1)).to(dtype)
    out = run_attention(ops, pool, q.to(DEV), [44, 44], [10, 10], d ** -0.5, max_rows=10, max_len=44)     # keys from 44 on are left out
    for b in (0, 1):
        k, v = (R.stored(pool.pages[i], None, pool.table[b], torch.arange(44)) for i in (0, 1))
        rows = slice(10 * b, 10 * b + 10)
        want, bound = R.attention(q[:, rows].double(), k, v, 44, d ** -0.5, dtype)
        assert bool(((out[rows].view(10, heads, d).double() - want).abs() <= bound).all())
    pool.table[0, 1], pool.table[0, 2] = -5, 1 << 30
    bad = run_attention(ops, pool, q.to(DEV), [44, 44], [10, 10], d ** -0.5, max_rows=10, max_len=64)
    good = torch.zeros(1)
    k, v = (R.stored(pool.pages[i], None, pool.table[1], torch.arange(54)) for i in (0, 1))
    want, bound = R.attention(q[:, 10:].double(), k, v, 44, d ** -0.5, dtype)
    assert bool(((bad[10:].view(10, heads, d).double() - want).abs() <= bound).all()) and bool(good.isfinite().all())


@pytest.mark.parametrize("past,new,heads", [([4000, 77], [1, 1], 8), ([300], [40], 8), ([900, 150, 20, 400] * 17, [11, 5, 9, 10] * 17, 8)])
def test_attention_replays_in_a_graph_with_other_lengths(ops, past, new, heads):
    """One captured launch serves every step whose bounds hold: lengths, tables and rows are read on the device; several replays
    with eager work between them, each against the eager result."""
    h_kv, d, page, dtype = 2, 128, 64, torch.bfloat16
    total = [p + n for p, n in zip(past, new)]
    pool = Pool(total, h_kv, d, page, dtype, True, 71)
    g = torch.Generator().manual_seed(4)
    q = torch.randn((heads, sum(new), d), generator=g).to(dtype).to(DEV)
    out = torch.zeros((sum(new), heads * d), dtype=dtype, device=DEV)
    lens, rows = i32(past), cu(new).to(DEV)
    kw = pool.kw()
    bounds = dict(max_rows=max(new), max_len=max(total))
    ops.paged_attention(q, out=out, seq_lens=lens, cu_rows=rows, scale=d ** -0.5, **kw, **bounds)      # loads the code
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, out=out, seq_lens=lens, cu_rows=rows, scale=d ** -0.5, **kw, **bounds)
    for step in range(4):
        lens.copy_(i32([max(0, p - 37 * step) for p in past]))
        q.copy_(torch.randn(q.shape, generator=g).to(dtype))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(out)
        ops.paged_attention(q, out=eager, seq_lens=lens, cu_rows=rows, scale=d ** -0.5, **kw, **bounds)
        assert torch.equal(out, eager) and bool(out.abs().sum() > 0)


def test_two_graphs_at_once(ops):
    """Two captured calls replayed on two streams: each graph has its own workspace."""
    h_kv, d, page, dtype = 2, 64, 32, torch.float16
    pools = [Pool([4001], h_kv, d, page, dtype, False, s) for s in (3, 4)]
    qs = [torch.randn((8, 1, d), generator=torch.Generator().manual_seed(s)).to(dtype).to(DEV) for s in (3, 4)]
    alone = [run_attention(ops, p, q, [4000], [1], d ** -0.5) for p, q in zip(pools, qs)]
    kws, lens, rows = [p.kw() for p in pools], i32([4000]), i32([0, 1])
    outs = [torch.zeros((1, 8 * d), dtype=dtype, device=DEV) for _ in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for q, o, kw in zip(qs, outs, kws):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(q, out=o, seq_lens=lens, cu_rows=rows, scale=d ** -0.5, **kw)
        graphs.append(graph)
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, a in zip(outs, alone):
            assert torch.equal(o.cpu(), a)


def test_two_streams_at_once(ops):
    """Two calls in flight on two streams, each with its own workspace: both get what they get alone."""
    h_kv, d, page, dtype = 8, 128, 64, torch.float16
    pools = [Pool([6001], h_kv, d, page, dtype, True, s) for s in (1, 2)]
    qs = [torch.randn((32, 1, d), generator=torch.Generator().manual_seed(s)).to(dtype).to(DEV) for s in (1, 2)]
    alone = [run_attention(ops, p, q, [6000], [1], d ** -0.5) for p, q in zip(pools, qs)]
    kws = [p.kw() for p in pools]
    lens, rows = i32([6000]), i32([0, 1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros((1, 32 * d), dtype=dtype, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, o, kw in zip(streams, qs, outs, kws):
            with torch.cuda.stream(s):
                ops.paged_attention(q, out=o, seq_lens=lens, cu_rows=rows, scale=d ** -0.5, **kw)
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert torch.equal(o.cpu(), a)
