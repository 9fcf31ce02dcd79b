"""A captured step over a PagedKVCache: the step's arrays live in buffers of the program's own, at the sizes of its bounds; each batch's
are copied into them in front of a replay."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS, KV, DIM, LAYERS, PAGE = 8, 2, 64, 2, 32


@pytest.mark.parametrize("quantised", [False, True])
def test_a_captured_step_serves_the_batches_of_a_cache(quantised):
    from sequoia_amd.Engine.Llama_modules import rope_tables
    from sequoia_amd.Engine.Paged_KV import PagedKVCache
    from sequoia_amd.ops import get_ops
    ops = get_ops()
    config = SimpleNamespace(num_hidden_layers=LAYERS, num_attention_heads=HEADS, num_key_value_heads=KV, hidden_size=HEADS * DIM)
    most, width, max_rows = 6, 5, 7                                      # sequences, pages a sequence, rows a sequence brings
    cache = PagedKVCache(config, most * width, PAGE, device=DEV, quantised=quantised)
    cos, sin = rope_tables(DIM, width * PAGE, 10000.0, DEV, torch.float16)
    g = torch.Generator().manual_seed(3)
    rows = most * max_rows
    table, lens = torch.zeros((most, width), dtype=torch.int32, device=DEV), torch.zeros(most, dtype=torch.int32, device=DEV)
    cu_rows, pos = torch.zeros(most + 1, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int64, device=DEV)
    qkv = torch.zeros((LAYERS, rows, (HEADS + 2 * KV) * DIM), dtype=torch.float16, device=DEV)
    q, out = torch.zeros((HEADS, rows, DIM), dtype=torch.float16, device=DEV), torch.zeros((LAYERS, rows, HEADS * DIM), dtype=torch.float16, device=DEV)

    def step(table, lens, cu_rows, pos, qkv, q, out, max_rows, max_len):
        for i in range(LAYERS):
            one = cache.layer(i)
            ops.rope_kv_write_paged(qkv[i], q, one["k_pages"], one["v_pages"], cos, sin, pos, table, lens, cu_rows, HEADS, KV, DIM,
                                    k_scales=one["k_scales"], v_scales=one["v_scales"])
            ops.paged_attention(q, out=out[i], page_table=table, seq_lens=lens, cu_rows=cu_rows, scale=DIM ** -0.5, max_rows=max_rows, max_len=max_len, **one)

    bounds = (max_rows, width * PAGE)
    step(table, lens, cu_rows, pos, qkv, q, out, *bounds)                # loads the code; no sequence brings a row
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(table, lens, cu_rows, pos, qkv, q, out, *bounds)
    seqs = [cache.add_sequence() for _ in range(most)]
    for turn in range(7):
        if turn == 4:                                                    # one leaves, another comes: fewer sequences than the buffers hold meanwhile
            cache.free_sequence(seqs.pop(1))
        if turn == 5:
            seqs.append(cache.add_sequence())
        counts = [int(c) for c in torch.randint(0, max_rows + 1, (len(seqs),), generator=g)]
        b = cache.batch(seqs, counts)
        n, w = len(seqs), b.page_table.shape[1]
        table.zero_()
        table[:n, :w], lens[:n], cu_rows[:n + 1], pos[:b.n_rows] = b.page_table, b.seq_lens, b.cu_rows, b.position_ids
        cu_rows[n + 1:] = b.n_rows                                       # the rest of the sequences bring nothing
        qkv[:, :b.n_rows] = torch.randn((LAYERS, b.n_rows, qkv.shape[2]), generator=g).half().to(DEV)
        q.fill_(5.0), out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got, pages = (q.clone(), out.clone()), [t.view(torch.uint8).clone() for t in (cache.k_pages, cache.v_pages)]
        q2, out2 = torch.empty((HEADS, b.n_rows, DIM), dtype=torch.float16, device=DEV), torch.empty((LAYERS, b.n_rows, HEADS * DIM), dtype=torch.float16, device=DEV)
        step(b.page_table, b.seq_lens, b.cu_rows, b.position_ids, qkv[:, :b.n_rows].contiguous(), q2, out2, b.max_rows, b.max_len)
        torch.cuda.synchronize()
        assert torch.equal(got[0][:, :b.n_rows], q2) and bool((got[0][:, b.n_rows:] == 5.0).all()) and bool((got[1][:, b.n_rows:] == 5.0).all())
        for x, y in zip(pages, (cache.k_pages, cache.v_pages)):
            assert torch.equal(x, y.view(torch.uint8))
        # other bounds may share the keys out otherwise: the sums differ by roundings of fp32 and of the weights, 2^-11 each way at most of
        # sum w |v|, and by the output's own rounding
        most_v = (cache.v_pages.float().abs().max() if not quantised else qkv.float().abs().max()) * 1.07
        assert bool(((got[1][:, :b.n_rows].float() - out2.float()).abs() <= 2 * 2.0 ** -11 * (most_v + out2.float().abs()) + 1e-4).all())
        for s, c in zip(seqs, counts):
            cache.set_length(s, cache.length(s) + max(0, c - 1))
