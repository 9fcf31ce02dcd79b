"""The paged operators together, as a batch of sequences uses them: write the chunk of the last token and the drafted ones, attend,
verify, roll back by lengths; sequences come and go, their pages change hands.  Every step is held to the 64-bit forms."""
from types import SimpleNamespace

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB, HEADS, KV, DIM = 211, 8, 2, 64


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import get_ops
    o = get_ops()
    assert o.name == "hip" and o.lib.sq_device_ready() == 1
    return o


class Model:
    """One attention layer over a table of packed rows (a token's q | k | v are its row of the table: no projection's rounding)
    and a head; what it stores and attends is recomputed from the tokens."""

    def __init__(self, dtype, seed):
        from sequoia_amd.Engine.Llama_modules import rope_tables
        g = torch.Generator().manual_seed(seed)
        self.dtype = dtype
        self.table = torch.randn((VOCAB, (HEADS + 2 * KV) * DIM), generator=g).to(dtype)
        self.cos, self.sin = rope_tables(DIM, 1024, 10000.0, "cpu", dtype)
        self.head = torch.randn((HEADS * DIM, VOCAB), generator=g) * 0.15
        self.dev = {n: getattr(self, n).to(DEV) for n in ("table", "cos", "sin", "head")}

    def logits(self, out):
        return out.float() @ self.dev["head"]

    def expected(self, tokens, quantised):
        """(q rotated and rounded, k, v as stored) of a whole sequence, float64; q [H, n, D]."""
        n = len(tokens)
        x = self.table[torch.tensor(tokens)].double().view(n, -1, DIM)
        turned = R.rope(x[:, :HEADS + KV], self.cos[:n].double(), self.sin[:n].double()).float()      # exact products, one fp32 rounding
        q, k, v = turned[:, :HEADS], turned[:, HEADS:], x[:, HEADS + KV:].float()
        store = (lambda r: self.e4m3(r)) if quantised else (lambda r: r.to(self.dtype).double())
        return q.to(self.dtype).double().transpose(0, 1), store(k).transpose(0, 1), store(v).transpose(0, 1)

    def e4m3(self, rows):
        byte = R.row_scale_byte(rows.double(), self.dtype)
        codes = (rows * torch.exp2(127.0 - byte.float())[..., None]).to(torch.float8_e4m3fn)
        return R.decode(codes.view(torch.uint8), byte)


@pytest.mark.parametrize("dtype,quantised,page", [(torch.float16, False, 16), (torch.float16, True, 32), (torch.bfloat16, True, 16)])
def test_speculation_steps_of_a_changing_batch(ops, dtype, quantised, page):
    from sequoia_amd.Engine.Paged_KV import PagedKVCache
    config = SimpleNamespace(num_hidden_layers=1, num_attention_heads=HEADS, num_key_value_heads=KV, hidden_size=HEADS * DIM)
    m = Model(dtype, 5)
    cache = PagedKVCache(config, 40, page, device=DEV, dtype=dtype, quantised=quantised)
    g = torch.Generator().manual_seed(7)
    text = {}                                           # sequence -> tokens, the last one not stored yet

    def forward(seqs, chunks):
        """Stores and attends chunks[i] behind sequence seqs[i]; -> logits of all rows, checked against the 64-bit form."""
        b = cache.batch(seqs, [len(c) for c in chunks])
        ids = torch.tensor([t for c in chunks for t in c], device=DEV)
        q, out = torch.empty((HEADS, b.n_rows, DIM), dtype=dtype, device=DEV), torch.empty((b.n_rows, HEADS * DIM), dtype=dtype, device=DEV)
        one = cache.layer(0)
        ops.rope_kv_write_paged(m.dev["table"][ids], q, one["k_pages"], one["v_pages"], m.dev["cos"], m.dev["sin"], b.position_ids, b.page_table,
                                b.seq_lens, b.cu_rows, HEADS, KV, DIM, k_scales=one["k_scales"], v_scales=one["v_scales"])
        ops.paged_attention(q, out=out, page_table=b.page_table, seq_lens=b.seq_lens, cu_rows=b.cu_rows, scale=DIM ** -0.5, max_rows=b.max_rows,
                            max_len=b.max_len, **one)
        got, at = out.cpu().view(-1, HEADS, DIM).double(), 0
        for s, c in zip(seqs, chunks):
            n = len(c)
            full = text[s][:cache.length(s)] + list(c)
            eq, ek, ev = m.expected(full, quantised)
            want, bound = R.attention(eq[:, -n:], ek, ev, len(full) - n, DIM ** -0.5, dtype)
            # what the kernel read went through the same roundings; where fp32 puts a value on a border they may differ by a step
            worst = ((got[at:at + n] - want).abs() / bound).max()
            assert float(worst) <= 1.0, (s, n, float(worst))
            at += n
        return m.logits(out)

    def admit(length):
        s = cache.add_sequence()
        text[s] = torch.randint(0, VOCAB, (length,), generator=g).tolist()
        forward([s], [text[s][:-1]])
        cache.set_length(s, length - 1)
        return s

    live = [admit(n) for n in (2, 37, 90)]
    accepted = 0
    for step in range(10):
        if step == 4:
            cache.free_sequence(live.pop(0))
            live.append(admit(65))
        counts = [int(c) for c in torch.randint(0, 5, (len(live),), generator=g)]
        drafts = [torch.randint(0, VOCAB, (c,), generator=g).tolist() for c in counts]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        draft_logits = torch.zeros((sum(counts), VOCAB))
        rows = forward(live, [[text[s][-1]] + d for s, d in zip(live, drafts)])
        for i, s in enumerate(live):                    # a draft that is often right, and knows it: tokens at the target's maxima
            for j in range(counts[i]):
                draft_logits[cu[i] + j] = rows[cu[i] + i + j].cpu() + 0.3 * torch.randn(VOCAB, generator=g)
        best = [int(draft_logits[r].argmax()) for r in range(sum(counts))]
        temps = torch.tensor([0.0, 0.8, 1.3][:len(live)])
        ua, un = torch.rand((sum(counts),), generator=g), torch.rand((len(live),), generator=g)
        n_acc, nxt = torch.zeros(len(live), dtype=torch.int32, device=DEV), torch.zeros(len(live), dtype=torch.int64, device=DEV)
        tokens = torch.tensor([best[cu[i]] if j == 0 and counts[i] else drafts[i][j] for i in range(len(live)) for j in range(counts[i])], dtype=torch.int64)
        # only a chunk whose tokens were the judged ones may be committed: run the step again with them
        drafts = [tokens[cu[i]:cu[i + 1]].tolist() for i in range(len(live))]
        rows = forward(live, [[text[s][-1]] + d for s, d in zip(live, drafts)])
        ops.verify_drafts(rows, draft_logits.to(DEV), tokens.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), ua.to(DEV), un.to(DEV),
                          temps.to(DEV), n_acc, nxt)
        want_a, want_n, margin = R.verify(rows.cpu(), draft_logits, tokens.tolist(), cu, ua.tolist(), un.tolist(), temps.tolist())
        assert margin > 1e-12 and (n_acc.tolist(), nxt.tolist()) == (want_a, want_n)
        for i, s in enumerate(live):
            text[s] += drafts[i][:want_a[i]] + [want_n[i]]
            cache.set_length(s, len(text[s]) - 1)
            accepted += want_a[i]
    assert accepted > 0
    held = sum(-(-cache.length(s) // page) for s in live)
    assert cache.free_pages() == 40 - held

    # a sequence moves into the static cache
    if dtype == torch.float16:
        from sequoia_amd.Engine.Llama_KV import KV_Cache
        static = KV_Cache(config, max_length=256, device=DEV)
        s = live[0]
        cache.export(s, static)
        n = cache.length(s)
        _, k, v = m.expected(text[s][:n], quantised)
        assert static.kv_offset == n
        assert torch.equal(static.k_cache[0, 0, :, :n].cpu(), k.to(dtype)) and torch.equal(static.v_cache[0, 0, :, :n].cpu(), v.to(dtype))
        assert not bool(static.k_cache[0, 0, :, n:].any())


def test_one_captured_step_serves_a_growing_batch(ops):
    """Write, attention and verification in one graph; lengths, offsets, tokens and uniforms change between the replays, with eager
    work in between, and every replay gives what the eager calls give."""
    m, b, most = Model(torch.float16, 9), 5, 4
    g = torch.Generator().manual_seed(11)
    page, width = 32, 12
    k, v = (torch.zeros((b * width, KV, page, DIM), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((b * width, KV, page), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    table = torch.randperm(b * width, generator=g).to(torch.int32).view(b, width).to(DEV)
    rows = b * (most + 1)
    lens, cu_rows, cu = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (b, b + 1, b + 1))
    ids, pos = torch.zeros(rows, dtype=torch.int64, device=DEV), torch.zeros(rows, dtype=torch.int64, device=DEV)
    drafted = torch.zeros(b * most, dtype=torch.int64, device=DEV)
    draft = torch.randn((b * most, VOCAB), generator=g).to(DEV)
    ua, un = torch.zeros(b * most, device=DEV), torch.zeros(b, device=DEV)
    q, out = torch.zeros((HEADS, rows, DIM), dtype=torch.float16, device=DEV), torch.zeros((rows, HEADS * DIM), dtype=torch.float16, device=DEV)
    acc, nxt = torch.zeros(b, dtype=torch.int32, device=DEV), torch.zeros(b, dtype=torch.int64, device=DEV)
    pool = dict(k_scales=ks, v_scales=vs)

    def step():
        ops.rope_kv_write_paged(m.dev["table"][ids], q, k, v, m.dev["cos"], m.dev["sin"], pos, table, lens, cu_rows, HEADS, KV, DIM, **pool)
        ops.paged_attention(q, k, v, out, table, lens, cu_rows, DIM ** -0.5, max_rows=most + 1, max_len=width * page, **pool)
        ops.verify_drafts(m.logits(out), draft, drafted, cu, ua, un, 0.9, acc, nxt)

    step()                                              # loads the code, sizes the matrix product's workspace
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    length = torch.zeros(b, dtype=torch.int64)
    for _ in range(6):
        counts = torch.randint(0, most + 1, (b,), generator=g)
        at, ct = [0], [0]
        for c in counts.tolist():
            at.append(at[-1] + c)
            ct.append(ct[-1] + c + 1)
        lens.copy_(length)
        cu.copy_(torch.tensor(at))
        cu_rows.copy_(torch.tensor(ct))
        ids.copy_(torch.randint(0, VOCAB, (rows,), generator=g))
        place = [int(length[i]) + j for i in range(b) for j in range(int(counts[i]) + 1)]
        pos[:len(place)] = torch.tensor(place, device=DEV)
        drafted.copy_(torch.randint(0, VOCAB, drafted.shape, generator=g))
        ua.copy_(torch.rand(ua.shape, generator=g))
        un.copy_(torch.rand(un.shape, generator=g))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, acc, nxt, k.view(torch.uint8), ks)]
        out.zero_()
        step()
        torch.cuda.synchronize()
        for x, y in zip(got, (out, acc, nxt, k.view(torch.uint8), ks)):
            assert torch.equal(x, y)
        assert bool(out[:ct[-1]].any()) and not bool(out[ct[-1]:].any())
        length += acc.cpu() + 1
