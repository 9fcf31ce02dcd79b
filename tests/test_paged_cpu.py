"""Paged path without a GPU: refusals of the C entries and of the tensor front end, the host's page tables."""
from types import SimpleNamespace

import pytest
import torch

from sequoia_amd import native

CONFIG = SimpleNamespace(num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, hidden_size=256)
P = 4096          # stands for a pointer: every call below is refused before one is followed


def write(lib, **kw):
    a = dict(qkv=P, stride=512, q=P, k=P, v=P, ks=None, vs=None, cos=P, sin=P, max_pos=8, pos=P, table=P, width=2, n_pages=4, page=16, lens=P,
             cu=P, n_seqs=1, n_rows=1, heads=4, kv=2, d=64, dtype=0)
    a.update(kw)
    return lib.sq_rope_kv_write_paged(*a.values(), None)


def read(lib, **kw):
    a = dict(k=P, v=P, ks=None, vs=None, ko=P, vo=P, ss=1 << 12, hs=64 * 8, rows=8, table=P, width=2, n_pages=4, page=16, starts=P, counts=P,
             n_seqs=1, max_count=8, kv=2, d=64, dtype=0)
    a.update(kw)
    return lib.sq_kv_read_paged(*a.values(), None)


def attend(lib, **kw):
    a = dict(q=P, qh=64, qr=256, k=P, v=P, ks=None, vs=None, out=P, os=256, table=P, width=200, n_pages=4, page=16, lens=P, cu=P, n_seqs=1,
             n_rows=1, max_rows=1, max_len=3000, heads=4, kv=2, d=64, scale=0.125, dtype=0, ws=P, wsb=1 << 30)
    a.update(kw)
    return lib.sq_paged_attention(*a.values(), None)


def verify(lib, **kw):
    a = dict(t=P, ldt=100, d=P, ldd=100, tok=P, cu=P, n_seqs=1, n=2, vocab=100, ua=P, un=P, temps=None, temp=1.0, acc=P, nxt=P, dtype=0, ws=P,
             wsb=1 << 20)
    a.update(kw)
    return lib.sq_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("fn,bad", [
    (write, dict(qkv=None)), (write, dict(cos=None)), (write, dict(table=None)), (write, dict(heads=3)), (write, dict(ks=P)), (write, dict(vs=P)),
    (write, dict(stride=504)), (write, dict(stride=513)), (write, dict(max_pos=0)), (write, dict(n_rows=-1)), (write, dict(n_pages=0)),
    (write, dict(qkv=P + 8)), (write, dict(k=P + 2)),
    (read, dict(ko=None)), (read, dict(starts=None)), (read, dict(ks=P)), (read, dict(hs=64 * 7)), (read, dict(ss=4)), (read, dict(max_count=-1)),
    (read, dict(v=P + 4)), (read, dict(kv=0)),
    (attend, dict(q=None)), (attend, dict(cu=None)), (attend, dict(heads=3)), (attend, dict(scale=0.0)), (attend, dict(scale=-1.0)),
    (attend, dict(scale=float("nan"))), (attend, dict(scale=float("inf"))), (attend, dict(max_len=200 * 16 + 1)), (attend, dict(max_len=0)),
    (attend, dict(ws=None)), (attend, dict(wsb=8)), (attend, dict(ws=P + 4)), (attend, dict(qr=60)), (attend, dict(ks=P)), (attend, dict(q=P + 2)),
    (verify, dict(t=None)), (verify, dict(cu=None)), (verify, dict(d=None)), (verify, dict(tok=None)), (verify, dict(ldt=99)), (verify, dict(ldd=99)),
    (verify, dict(vocab=0)), (verify, dict(temp=-1.0)), (verify, dict(temp=float("nan"))), (verify, dict(temp=float("inf"))), (verify, dict(ws=None)),
    (verify, dict(wsb=16)), (verify, dict(n=-1)),
])
def test_c_entries_refuse_bad_arguments(fn, bad):
    assert fn(native.load(), **bad) == native.SQ_EINVAL, bad


@pytest.mark.parametrize("fn,bad", [(f, b) for f in (write, read, attend) for b in (dict(d=96), dict(page=48), dict(page=8), dict(page=512), dict(dtype=2))]
                         + [(verify, dict(dtype=3))])
def test_c_entries_name_what_they_do_not_have(fn, bad):
    assert fn(native.load(), **bad) == native.SQ_EUNSUPPORTED, bad


def test_c_entries_with_nothing_to_do():
    lib = native.load()
    assert write(lib, n_rows=0, qkv=None) == 0 and write(lib, n_seqs=0) == 0
    assert read(lib, n_seqs=0) == 0 and read(lib, max_count=0) == 0 and read(lib, rows=0, max_count=0, hs=0) == 0
    assert attend(lib, n_rows=0) == 0 and attend(lib, n_seqs=0) == 0 and attend(lib, max_rows=0) == 0
    assert verify(lib, n_seqs=0) == 0
    assert lib.sq_paged_attention_workspace_bytes(0, 1, 1, 1, 4, 2, 64) == 0 and lib.sq_verify_drafts_workspace_bytes(0, 0, 10) == 0


def test_workspace_of_the_attention():
    """Up to 32 packed rows a KV head: two places of 16 or 32 rows for each of at most 512 workgroups, and two numbers a unit.  More:
    whole parts of the key axis, at most 64 (a lane each joins them), none of fewer than 512 keys."""
    lib = native.load()
    for n_seqs in (1, 3, 64, 1000):
        for max_len in (1, 255, 257, 5000, 131072, 2_000_000):
            for max_rows in (1, 7, 129, 4096):
                for heads, kv in ((12, 12), (64, 8), (8, 1)):
                    rows, packed = max_rows * n_seqs, max_rows * heads // kv
                    got = lib.sq_paged_attention_workspace_bytes(n_seqs, rows, max_rows, max_len, heads, kv, 128)
                    if packed <= 32:
                        if max_len <= 256:
                            assert got == 0
                            continue
                        groups, left = divmod(got - n_seqs * kv * 8, 2 * (16 if packed <= 16 else 32) * 130 * 4)
                        assert left == 0 and 1 <= groups <= 512 and groups <= n_seqs * kv * -(-max_len // 256)
                    else:
                        parts, left = divmod(got, rows * heads * 130 * 4)
                        assert left == 0 and parts <= 64 and parts != 1 and (parts == 0 or max_len > 256 * (parts - 1))


def test_attention_workspace_of_a_few_tokens_of_shared_heads():
    """33 to 128 rows: two parts of a tile's rows a workgroup where the keys are shared out, nothing where every unit has its own."""
    lib = native.load()
    size = lambda seqs, rows, length: lib.sq_paged_attention_workspace_bytes(seqs, seqs * rows, rows, length, 64, 8, 128)
    for rows, tile in ((5, 64), (8, 64), (9, 96), (16, 128)):
        assert size(32, rows, 5000) == 512 * 2 * tile * 130 * 4 + 256 * 8
        assert size(64, rows, 5000) == size(32, rows, 256) == 0


def test_front_end_refuses_host_tensors():
    from sequoia_amd.ops import HipOps
    ops = HipOps()
    q, pages, table, one = torch.zeros(4, 1, 64).half(), torch.zeros(2, 2, 16, 64).half(), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    out = torch.zeros(1, 256).half()
    with pytest.raises(native.SequoiaNativeError, match="no CPU fallback"):
        ops.paged_attention(q, pages, pages, out, table, one, one, 0.1)
    with pytest.raises(native.SequoiaNativeError, match="no CPU fallback"):
        ops.rope_kv_write_paged(torch.zeros(1, 512).half(), q, pages, pages, out, out, one, table, one, one, 4, 2, 64)
    with pytest.raises(native.SequoiaNativeError, match="no CPU fallback"):
        ops.kv_read_paged(pages, pages, pages[:1], pages[:1], table, one, one)
    with pytest.raises(native.SequoiaNativeError, match="no CPU fallback"):
        ops.verify_drafts(out, out, one.long(), one, out, out, 1.0, one, one.long())


def cache(n_pages=6, page_size=16, **kw):
    from sequoia_amd.Engine.Paged_KV import PagedKVCache
    return PagedKVCache(CONFIG, n_pages, page_size, device="cpu", **kw)


def test_cache_refuses_what_the_kernels_do_not_have():
    with pytest.raises(ValueError):
        cache(page_size=24)
    with pytest.raises(ValueError):
        cache(dtype=torch.float32)
    with pytest.raises(ValueError):
        cache(n_pages=0)


def test_batches_never_share_a_page_and_lengths_roll_back():
    c = cache(n_pages=8)
    a, b = c.add_sequence(), c.add_sequence()
    x = c.batch([a, b], [20, 3])
    assert x.n_rows == 23 and x.max_rows == 20 and x.max_len == 20 and x.cu_rows.tolist() == [0, 20, 23] and x.seq_lens.tolist() == [0, 0]
    assert x.position_ids.tolist() == list(range(20)) + [0, 1, 2]
    assert len(set(x.page_table[0].tolist()) | {int(x.page_table[1, 0])}) == 3 and c.free_pages() == 5
    c.set_length(a, 20), c.set_length(b, 3)
    y = c.batch([b, a], [14, 0])
    assert y.seq_lens.tolist() == [3, 20] and y.position_ids.tolist() == list(range(3, 17)) and y.max_len == 20
    c.set_length(b, 17)
    c.set_length(a, 16)                                                 # one page comes back
    assert c.free_pages() == 5 and c.length(a) == 16
    c.free_sequence(b)
    assert c.free_pages() == 7
    with pytest.raises(KeyError):
        c.length(b)


def test_a_batch_too_large_changes_nothing():
    c = cache(n_pages=3)
    a, b = c.add_sequence(), c.add_sequence()
    c.batch([a], [16])
    c.set_length(a, 16)
    with pytest.raises(RuntimeError, match="2 free"):
        c.batch([a, b], [17, 16])
    assert c.free_pages() == 2 and c.length(a) == 16
    c.batch([a, b], [16, 16])
    for bad in (([a, a], [1, 1]), ([a], [-1]), ([], []), ([a], [1, 2])):
        with pytest.raises(ValueError):
            c.batch(*bad)
    with pytest.raises(ValueError):
        c.set_length(a, 33)
    with pytest.raises(ValueError):
        c.set_length(a, -1)


def test_layers_of_a_quantised_cache():
    c = cache(quantised=True)
    one = c.layer(1)
    assert one["k_pages"].dtype == torch.float8_e4m3fn and one["k_scales"].dtype == torch.uint8 and one["k_scales"].shape == (6, 2, 16)
    assert cache(dtype=torch.bfloat16).layer(0)["k_scales"] is None


@pytest.mark.parametrize("fn,bad", [
    (write, dict(n_rows=1 << 24)),                                        # more workgroups than a launch takes
    (read, dict(n_seqs=1 << 24)),
    (attend, dict(n_rows=1 << 24, max_rows=1 << 24, wsb=1 << 62)),
    (attend, dict(width=1 << 28, max_len=(1 << 30) + 1)),                 # keys past 30 bits
    (verify, dict(vocab=(1 << 30) + 1, ldt=1 << 31, ldd=1 << 31, wsb=1 << 62)),
    (verify, dict(n=1 << 23, wsb=1 << 62)),
])
def test_c_entries_refuse_what_a_launch_does_not_hold(fn, bad):
    assert fn(native.load(), **bad) == native.SQ_EUNSUPPORTED
