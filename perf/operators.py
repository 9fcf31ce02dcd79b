"""The operators of batched speculative decoding over a paged KV cache, as cases that can be timed and compared.

Four operators, in the order one step of a batch uses them: the new tokens' rotary embedding with the write of their keys
and values into pages (fp16, bf16, or e4m3 with one power-of-two scale for each row of a head), the read of stored rows
back into the static slot layout, the attention of every sequence's chunk of new tokens over its pages, and the
verification of the drafted tokens against the target's probabilities from given random numbers.

`own` False: the plain form, elementary torch operations in 32 bits (the verification in 64: its outcomes are decisions,
and every comparison sits next to a border).  `own` True: the calls of `sequoia_amd.ops`.
"""
import math
import random

import torch

own = False
DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a batch of 32 through a 64-query-head, 8-KV-head layer, into an e4m3 cache
        dict(name="write 32 tokens e4m3", op="write", batch=32, new_lo=1, new_hi=1, past_lo=40, past_hi=1900, heads=64, kv=8, dim=128,
             page=64, dtype="fp16", cache="e4m3", lens=1),
        # two long prompts' chunks through the same layer, into fp16 pages
        dict(name="write prompt fp16", op="write", batch=2, new_lo=2900, new_hi=3400, past_lo=0, past_hi=500, heads=64, kv=8, dim=128,
             page=128, dtype="fp16", cache="fp16", lens=2),
        # one short sequence of a 12-head, 64-wide draft moved back into its static slots
        dict(name="read short fp16", op="read", batch=1, past_lo=230, past_hi=230, start_hi=0, kv=12, dim=64, page=16, dtype="fp16",
             cache="fp16", lens=3),
        # eight long e4m3 sequences leaving the pages, ragged, some from the middle
        dict(name="read long e4m3", op="read", batch=8, past_lo=700, past_hi=9000, start_hi=300, kv=8, dim=128, page=64, dtype="bf16",
             cache="e4m3", lens=4),
        # one token of one short sequence of the draft: nothing but latency
        dict(name="attend 1 token draft", op="attend", batch=1, new_lo=1, new_hi=1, past_lo=143, past_hi=143, heads=12, kv=12, dim=64,
             page=16, dtype="fp16", cache="fp16", lens=5),
        # one token each of a ragged batch over an e4m3 cache, 8 query heads to a KV head
        dict(name="attend batch e4m3", op="attend", batch=48, new_lo=1, new_hi=1, past_lo=300, past_hi=6000, heads=64, kv=8, dim=128,
             page=64, dtype="fp16", cache="e4m3", lens=6),
        # drafted chunks of 1 to 7 tokens checked by a 32-head target, no sharing of heads
        dict(name="attend drafted chunks", op="attend", batch=16, new_lo=1, new_hi=7, past_lo=100, past_hi=2000, heads=32, kv=32, dim=128,
             page=32, dtype="fp16", cache="fp16", lens=7),
        # one token at the end of one very long sequence: the long axis is all there is to split
        dict(name="attend long e4m3", op="attend", batch=1, new_lo=1, new_hi=1, past_lo=100000, past_hi=100000, heads=32, kv=8, dim=128,
             page=128, dtype="bf16", cache="e4m3", lens=8),
        # the second chunk of a long prompt
        dict(name="attend prompt bf16", op="attend", batch=1, new_lo=4096, new_hi=4096, past_lo=4001, past_hi=4001, heads=64, kv=8,
             dim=128, page=64, dtype="bf16", cache="bf16", lens=9),
        # one sequence's five drafted tokens
        dict(name="verify one sequence", op="verify", batch=1, new_lo=5, new_hi=5, vocab=32000, dtype="fp16", greedy=False, lens=10),
        # a batch with 0 to 8 drafted tokens each, a third of the sequences greedy
        dict(name="verify batch", op="verify", batch=64, new_lo=0, new_hi=8, vocab=32000, dtype="fp16", greedy=True, lens=11),
        # a large vocabulary of odd size, rows that no 16-byte load fits
        dict(name="verify wide vocabulary", op="verify", batch=24, new_lo=2, new_hi=6, vocab=128261, dtype="bf16", greedy=False, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "attend", "verify"))
    lens = rng.randrange(1 << 30)
    if op == "verify":
        vocab = _log(rng, 1000, 130000)
        hi = _log(rng, 1, 12)
        batch = min(_log(rng, 1, 96), max(1, 18_000_000 // (vocab * (hi + 1))))
        return dict(op=op, batch=batch, new_lo=rng.randrange(0, hi + 1), new_hi=hi, vocab=vocab, dtype=rng.choice(("fp16", "bf16", "fp32")),
                    greedy=rng.random() < 0.4, lens=lens)
    dim = rng.choice((64, 128))
    kv, group = rng.choice(((12, 1), (16, 1), (32, 1), (8, 8), (8, 4), (2, 8), (1, 8), (4, 5), (5, 3)))
    page = rng.choice((16, 32, 64, 128, 256))
    dtype = rng.choice(("fp16", "bf16"))
    cache = rng.choice((dtype, "e4m3"))
    base = dict(op=op, heads=kv * group, kv=kv, dim=dim, page=page, dtype=dtype, cache=cache, lens=lens)
    if op == "read":
        hi = _log(rng, 1, 9000)
        batch = min(_log(rng, 1, 64), max(1, 60_000 * 8 * 128 // (hi * kv * dim)))
        base.pop("heads")
        return dict(base, batch=batch, past_lo=rng.randrange(0, hi + 1), past_hi=hi, start_hi=rng.randrange(0, hi + 1))
    if op == "write":
        hi = _log(rng, 1, 3400)
        batch = min(_log(rng, 1, 128), max(1, 5800 // hi))
        return dict(base, batch=batch, new_lo=rng.randrange(0, hi + 1), new_hi=hi, past_lo=0, past_hi=_log(rng, 1, 3000))
    # attention: decode, drafted chunks, prompts; the products of the sizes stay under those of the largest listed cases
    new_hi = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 4000)))
    past_hi = _log(rng, 1, 60000 if new_hi <= 16 else 4000)
    rows = new_hi * (past_hi + new_hi)
    batch = min(_log(rng, 1, 96), max(1, 290_000 * 8 * 128 // ((past_hi + new_hi) * kv * dim)), max(1, 4096 * 8097 * 64 // (rows * kv * group)))
    return dict(base, batch=batch, new_lo=rng.randrange(0, new_hi + 1), new_hi=new_hi, past_lo=rng.randrange(0, past_hi + 1), past_hi=past_hi)


def _lengths(case):
    """(new tokens, tokens already stored) of every sequence: part of the case, not of the seed."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case.get("new_lo", 0), case.get("new_hi", 0)) for _ in range(case["batch"])]
    past = [rng.randint(case.get("past_lo", 0), case.get("past_hi", 0)) for _ in range(case["batch"])]
    if "new_hi" in case and not any(new) and case["op"] != "verify":
        new[0] = max(1, case["new_hi"])
    if case["op"] == "read" and not any(past):
        past[0] = max(1, case["past_hi"])
    return new, past


def _starts(case, past):
    rng = random.Random(case["lens"] + 1)
    return [rng.randint(0, min(case["start_hi"], max(0, p - 1))) for p in past]


def work(case):
    new, past = _lengths(case)
    if case["op"] == "verify":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = 2 * sum(new) + case["batch"]
        return {"bytes": rows * case["vocab"] * size + sum(new) * 12 + case["batch"] * 24, "flops": 0}
    kv, dim = case["kv"], case["dim"]
    row = dim + 1 if case["cache"] == "e4m3" else 2 * dim                # one stored row of a head
    if case["op"] == "read":
        n = sum(p - s for p, s in zip(past, _starts(case, past)))
        return {"bytes": 2 * n * kv * (row + 2 * dim) + 4 * n // case["page"], "flops": 0}
    heads, t = case["heads"], sum(new)
    if case["op"] == "write":
        moved = t * (heads + 2 * kv) * dim * 2 + t * heads * dim * 2 + 2 * t * kv * row + t * (2 * dim * 2 + 8)
        if case["cache"] == "e4m3":
            moved += 2 * t * kv * (row + 2 * dim)                         # the rows read back
        return {"bytes": moved, "flops": 0}
    seen = [p + n if n else 0 for n, p in zip(new, past)]
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return {"bytes": 2 * sum(seen) * kv * row + 2 * t * heads * dim * 2, "flops": 4 * pairs * heads * dim}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _quantise(x, dtype):
    """Rows of `x` (float32) as e4m3 codes and the exponent byte of their scale: the smallest power of two that brings the
    row's largest finite magnitude to 448 or less."""
    top = 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)          # the largest value of the type with four significant bits
    x = torch.where(x.isfinite(), x.clamp(-top, top), torch.nan)
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))                  # m in [0.5, 1): amax = 2m 2^(e-1), 448 = 1.75 * 2^8
    byte = torch.where(m > 0, (e - 9 + (m > 0.875).int() + 127).clamp(1, 254), 1)
    inv = torch.ldexp(torch.ones_like(m), 127 - byte)
    return (x * inv[..., None]).to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _dequantise(codes, byte):
    return codes.view(torch.float8_e4m3fn).float() * torch.ldexp(torch.ones((), device=codes.device), byte.int() - 127)[..., None]


def _pages(case, total, gen):
    """A pool of pages in a random order, as a cache that has served a while holds it: every sequence's table, and pages with
    keys and values of what was stored before (rows behind a sequence's end hold what an earlier one left)."""
    p = case["page"]
    width = max(1, max((n + p - 1) // p for n in total))
    need = case["batch"] * width
    table = torch.randperm(need + 3, generator=gen, device=DEV)[:need].to(torch.int32).view(case["batch"], width)
    dtype = DTYPES[case["dtype"]]
    s = {"page_table": table}
    for name in ("k", "v"):
        rows = torch.randn((need + 3, case["kv"], p, case["dim"]), generator=gen, device=DEV, dtype=dtype)
        rows *= torch.exp(0.5 * torch.randn((need + 3, case["kv"], p, 1), generator=gen, device=DEV)).to(dtype)    # rows of unlike size
        if case["cache"] == "e4m3":
            s[name + "_pages"], s[name + "_scales"] = _quantise(rows.float(), dtype)
        else:
            s[name + "_pages"], s[name + "_scales"] = rows, None
        del rows
    return s


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _int(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    new, past = _lengths(case)
    if case["op"] == "verify":
        return _prepare_verify(case, new, gen)
    dtype, dim, kv = DTYPES[case["dtype"]], case["dim"], case["kv"]
    s = dict(case=case)
    if case["op"] == "read":
        start = _starts(case, past)
        s.update(_pages(case, past, gen))
        counts = [p - b for p, b in zip(past, start)]
        rows = max(counts) + 5                                            # rows behind a sequence's count stay as they are
        s.update(start=_int(start), count=_int(counts), max_count=max(counts),
                 k_out=torch.zeros((case["batch"], kv, rows, dim), dtype=dtype, device=DEV),
                 v_out=torch.zeros((case["batch"], kv, rows, dim), dtype=dtype, device=DEV))
        return s
    heads, t = case["heads"], sum(new)
    total = [n + p for n, p in zip(new, past)]
    s.update(_pages(case, total, gen))
    s.update(seq_lens=_int(past), cu_rows=_int(_offsets(new)), max_rows=max(new), max_len=max(total))
    owner = [b for b, n in enumerate(new) for _ in range(n)]
    local = [i for n in new for i in range(n)]
    s.update(owner=_int(owner, torch.int64), local=_int(local, torch.int64))
    if case["op"] == "attend":
        s["q"] = 1.5 * torch.randn((heads, t, dim), generator=gen, device=DEV, dtype=dtype)
        s["out"] = torch.zeros((t, heads * dim), dtype=dtype, device=DEV)
        return s
    top = max(total)
    freq = 10000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
    angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * freq
    angle = torch.cat((angle, angle), dim=-1)
    s.update(cos=angle.cos().to(dtype), sin=angle.sin().to(dtype), qkv=torch.randn((t, (heads + 2 * kv) * dim), generator=gen, device=DEV, dtype=dtype),
             position_ids=s["seq_lens"].long()[s["owner"]] + s["local"], q_out=torch.zeros((heads, t, dim), dtype=dtype, device=DEV))
    if case["cache"] == "e4m3":
        s.update(count=_int(new), k_out=torch.zeros((case["batch"], kv, max(new), dim), dtype=dtype, device=DEV),
                 v_out=torch.zeros((case["batch"], kv, max(new), dim), dtype=dtype, device=DEV))
    return s


def _prepare_verify(case, new, gen):
    n, b, vocab, dtype = sum(new), case["batch"], case["vocab"], DTYPES[case["dtype"]]
    owner = _int([i for i, c in enumerate(new) for _ in range(c)], torch.int64)
    local = _int([i for c in new for i in range(c)], torch.int64)
    cu = _int(_offsets(new))
    target = 2.5 * torch.randn((n + b, vocab), generator=gen, device=DEV)
    rows = torch.arange(n, device=DEV) + owner                            # the target row that judges each drafted token
    draft = target[rows] + torch.randn((n, vocab), generator=gen, device=DEV)
    target[torch.rand((n + b, vocab), generator=gen, device=DEV) < 0.02] = -math.inf        # what a nucleus filter took out
    target, draft = target.to(dtype), draft.to(dtype)
    temperature = torch.full((b,), 0.6, device=DEV)
    temperature += 0.5 * torch.rand((b,), generator=gen, device=DEV)
    if case["greedy"]:
        temperature[::3] = 0.0
    t = temperature[owner][:, None]
    noise = -torch.log(-torch.log(torch.rand((n, vocab), generator=gen, device=DEV).clamp(1e-9, 1 - 1e-7)))
    tokens = torch.where(t[:, 0] > 0, (draft.float() / t.clamp(min=1e-3) + noise).argmax(-1) if n else owner, draft.float().argmax(-1) if n else owner)
    greedy_rows = torch.rand((n,), generator=gen, device=DEV) < 0.7       # a greedy draft that mostly agrees
    tokens = torch.where((t[:, 0] == 0) & greedy_rows, target[rows].float().argmax(-1) if n else owner, tokens)
    return dict(case=case, target=target, draft=draft, tokens=tokens, cu=cu, owner=owner, local=local, rows=rows, temperature=temperature,
                u_accept=torch.rand((n,), generator=gen, device=DEV), u_next=torch.rand((b,), generator=gen, device=DEV), longest=max(new),
                accepted=torch.zeros((b,), dtype=torch.int32, device=DEV), next_tokens=torch.zeros((b,), dtype=torch.int64, device=DEV))


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(s):
    return {"write": _write, "read": _read, "attend": _attend, "verify": _verify}[s["case"]["op"]](s)


def _ops():
    from sequoia_amd.ops import get_ops
    return get_ops()


def _write(s):
    c = s["case"]
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    quantised = c["cache"] == "e4m3"
    if own:
        _ops().rope_kv_write_paged(s["qkv"], s["q_out"], s["k_pages"], s["v_pages"], s["cos"], s["sin"], s["position_ids"], s["page_table"],
                                   s["seq_lens"], s["cu_rows"], heads, kv, dim, k_scales=s["k_scales"], v_scales=s["v_scales"])
        if not quantised:
            return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}
        _ops().kv_read_paged(s["k_pages"], s["v_pages"], s["k_out"], s["v_out"], s["page_table"], s["seq_lens"], s["count"],
                             max_count=s["max_rows"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    x = s["qkv"].float().view(-1, heads + 2 * kv, dim)
    cos, sin = s["cos"][s["position_ids"]].float()[:, None], s["sin"][s["position_ids"]].float()[:, None]
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    turned = torch.cat((-qk[..., dim // 2:], qk[..., :dim // 2]), dim=-1)
    qk = qk * cos + turned * sin
    q, k = qk[:, :heads], qk[:, heads:]
    dtype = s["q_out"].dtype
    s["q_out"].copy_(q.transpose(0, 1))
    slot = s["seq_lens"].long()[s["owner"]] + s["local"]
    page, at = s["page_table"][s["owner"], slot // c["page"]].long(), slot % c["page"]
    for name, rows in (("k", k), ("v", v)):
        if quantised:
            codes, byte = _quantise(rows, dtype)
            s[name + "_pages"].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            s[name + "_scales"][page, :, at] = byte
            s[name + "_out"][s["owner"], :, s["local"]] = _dequantise(s[name + "_pages"].view(torch.uint8)[page, :, at],
                                                                       s[name + "_scales"][page, :, at]).to(dtype)
        else:
            s[name + "_pages"][page, :, at] = rows.to(dtype)
    where = "_out" if quantised else "_pages"
    return {"q": s["q_out"], "k": s["k" + where], "v": s["v" + where]}


def _gather(s, name, position):
    """Rows at `position` [batch, n] of every sequence, float32 [batch, n, kv, dim]."""
    p = s["case"]["page"]
    page = torch.gather(s["page_table"].long(), 1, (position // p).clamp(max=s["page_table"].shape[1] - 1))
    at = position % p
    if s[name + "_scales"] is None:
        return s[name + "_pages"][page, :, at].float()
    return _dequantise(s[name + "_pages"].view(torch.uint8)[page, :, at], s[name + "_scales"][page, :, at])


def _read(s):
    if own:
        _ops().kv_read_paged(s["k_pages"], s["v_pages"], s["k_out"], s["v_out"], s["page_table"], s["start"], s["count"],
                             max_count=s["max_count"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"k": s["k_out"], "v": s["v_out"]}
    n = torch.arange(s["k_out"].shape[2], device=DEV)
    valid = (n < s["count"][:, None])[:, None, :, None]
    for name in ("k", "v"):
        rows = _gather(s, name, n + s["start"].long()[:, None]).transpose(1, 2).to(s["k_out"].dtype)
        s[name + "_out"].copy_(torch.where(valid, rows, s[name + "_out"]))
    return {"k": s["k_out"], "v": s["v_out"]}


def _attend(s):
    c = s["case"]
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    scale = dim ** -0.5
    if own:
        _ops().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["out"], s["page_table"], s["seq_lens"], s["cu_rows"], scale,
                               max_rows=s["max_rows"], max_len=s["max_len"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return s["out"]
    b, group, rows = c["batch"], heads // kv, s["max_rows"]
    i = torch.arange(rows, device=DEV)
    at = (s["cu_rows"].long()[:-1, None] + i).clamp(max=max(0, s["q"].shape[1] - 1))
    q = s["q"][:, at].float().view(kv, group, b, rows, dim).permute(2, 0, 1, 3, 4).reshape(b, kv, group * rows, dim)
    j = torch.arange(s["max_len"], device=DEV)
    position = j.expand(b, -1)
    score = torch.matmul(q, _gather(s, "k", position).permute(0, 2, 3, 1).contiguous()).view(b, kv, group, rows, -1)
    score *= scale
    hidden = j > (s["seq_lens"].long()[:, None] + i)[..., None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    v = _gather(s, "v", position).transpose(1, 2)
    v = torch.where((j < (s["seq_lens"] + s["cu_rows"].diff())[:, None])[:, None, :, None], v, 0.0).contiguous()
    o = torch.matmul(score.view(b, kv, group * rows, -1), v).view(b, kv, group, rows, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, rows, heads * dim)
    s["out"].copy_(o[s["owner"], s["local"]])
    return s["out"]


def _verify(s):
    if own:
        _ops().verify_drafts(s["target"], s["draft"], s["tokens"], s["cu"], s["u_accept"], s["u_next"], s["temperature"], s["accepted"],
                             s["next_tokens"])
        return {"accepted": s["accepted"], "next": s["next_tokens"]}
    b, n, vocab = s["case"]["batch"], s["tokens"].shape[0], s["case"]["vocab"]
    seq = torch.arange(b, device=DEV)

    def probabilities(logits, t):
        x, t = logits.double(), t.double()[:, None]
        e = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0))
        best = torch.nn.functional.one_hot(x.argmax(-1), vocab)
        return torch.where(t > 0, e / e.sum(-1, keepdim=True), best.double())

    taken = torch.zeros((b, s["longest"] + 1), dtype=torch.bool, device=DEV)
    if n:
        t = s["temperature"][s["owner"]]
        p = probabilities(s["target"][s["rows"]], t).gather(1, s["tokens"][:, None])[:, 0]
        q = probabilities(s["draft"], t).gather(1, s["tokens"][:, None])[:, 0]
        taken[s["owner"], s["local"]] = torch.where(t > 0, s["u_accept"].double() * q < p, p > 0)
    accepted = taken.int().cumprod(-1).sum(-1)
    count = s["cu"].diff()
    at = s["cu"].long()[:-1] + accepted
    p = probabilities(s["target"][at + seq], s["temperature"])
    rest = p
    if n:
        q = probabilities(s["draft"][at.clamp(max=n - 1)], s["temperature"])
        rest = torch.where((accepted < count)[:, None] & (s["temperature"] > 0)[:, None], (p - q).clamp(min=0.0), p)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    mass = rest.cumsum(-1)
    token = (mass > (s["u_next"].double() * mass[:, -1])[:, None]).int().argmax(-1)
    s["accepted"].copy_(accepted)
    s["next_tokens"].copy_(token)
    return {"accepted": s["accepted"], "next": s["next_tokens"]}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](s, case)


def _stored(s, name, b, position):
    """Stored rows of sequence b in 64 bits, [kv, n, dim]: a code has four bits of exponent (bias 7) and three of mantissa."""
    p = s["case"]["page"]
    page, at = s["page_table"][b, position // p].long(), position % p
    rows = s[name + "_pages"][page, :, at]
    if s[name + "_scales"] is None:
        return rows.double().transpose(0, 1)
    code = rows.view(torch.uint8).long()
    sign, e, m = 1.0 - 2.0 * (code >> 7).double(), (code >> 3) & 15, (code & 7).double()
    value = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * torch.exp2((e - 7).double()))
    value = torch.where((code & 127) == 127, math.nan, sign * value)
    return (value * torch.exp2(s[name + "_scales"][page, :, at].double() - 127.0)[..., None]).transpose(0, 1)


def _to_e4m3(x, largest):
    """What rows hold after they were stored in 8 bits, in 64 bits: at most four significant bits, steps no finer than 2^-9
    of the row's scale, ties to the even one."""
    x = x.clamp(-largest, largest)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
    scale = torch.exp2((e - 8 + (top > 1.75 * torch.exp2(e)).double()).clamp(-126, 127))
    y = x / scale
    ey = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(ey - 3)
    return torch.round(y / step) * step * scale


def _exact_write(s, c):
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, dim)
    half = dim // 2
    cos, sin = s["cos"][s["position_ids"], None, :half].double(), s["sin"][s["position_ids"], None, :half].double()
    a, b = x[:, :heads + kv, :half], x[:, :heads + kv, half:]
    r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    q, k, v = r[:, :heads].transpose(0, 1), r[:, heads:], x[:, heads + kv:]
    if c["cache"] == "e4m3":
        largest = 61440.0 if c["dtype"] == "fp16" else 1.875 * 2.0 ** 127
        out = []
        for rows in (k, v):
            o = torch.zeros(s["k_out"].shape, dtype=torch.float64, device=DEV)
            o[s["owner"], :, s["local"]] = _to_e4m3(rows, largest)
            out.append(o)
        return {"q": q, "k": out[0], "v": out[1]}
    out = []
    slot = s["seq_lens"].long()[s["owner"]] + s["local"]
    for name, rows in (("k", k), ("v", v)):
        o = s[name + "_pages"].double()
        o[s["page_table"][s["owner"], slot // c["page"]].long(), :, slot % c["page"]] = rows
        out.append(o)
    return {"q": q, "k": out[0], "v": out[1]}


def _exact_read(s, c):
    out = []
    for name in ("k", "v"):
        o = torch.zeros(s["k_out"].shape, dtype=torch.float64, device=DEV)
        for b, (first, n) in enumerate(zip(s["start"].tolist(), s["count"].tolist())):
            o[b, :, :n] = _stored(s, name, b, torch.arange(first, first + n, device=DEV))
        out.append(o)
    return {"k": out[0], "v": out[1]}


def _exact_attend(s, c):
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    group = heads // kv
    at, past = s["cu_rows"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros((at[-1], heads, dim), dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        n = at[b + 1] - at[b]
        if not n:
            continue
        j = torch.arange(past[b] + n, device=DEV)
        k, v = _stored(s, "k", b, j), _stored(s, "v", b, j)
        hidden = j[None, :] > past[b] + torch.arange(n, device=DEV)[:, None]
        for h in range(kv):
            q = s["q"][h * group:(h + 1) * group, at[b]:at[b + 1]].double()
            w = torch.einsum("gnd,md->gnm", q, k[h]) / math.sqrt(dim)
            w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
            out[at[b]:at[b + 1], h * group:(h + 1) * group] = torch.einsum("gnm,md->ngd", w, v[h])
    return out.view(at[-1], heads * dim)


def _exact_verify(s, c):
    at, temperature = s["cu"].tolist(), s["temperature"].tolist()
    tokens, u, last = s["tokens"].tolist(), s["u_accept"].tolist(), s["u_next"].tolist()
    accepted, following = [], []
    for b in range(c["batch"]):
        n, t, k = at[b + 1] - at[b], temperature[b], 0

        def dist(row):
            if t == 0:
                d = torch.zeros(row.shape, dtype=torch.float64, device=DEV)
                d[torch.nonzero(row == row.max())[0, 0]] = 1.0
                return d
            return torch.softmax(row.double() / t, dim=-1)

        while True:
            p = dist(s["target"][at[b] + b + k])
            if k == n:
                break
            token = tokens[at[b] + k]
            if t == 0:
                if p[token] == 0:
                    break
            else:
                q = dist(s["draft"][at[b] + k])
                if not u[at[b] + k] * float(q[token]) < float(p[token]):
                    r = (p - q).clamp(min=0.0)
                    p = r if float(r.sum()) > 0 else p
                    break
            k += 1
        mass = torch.cumsum(p, dim=-1)
        accepted.append(k)
        following.append(int(torch.nonzero(mass > last[b] * mass[-1])[0, 0]))
    return {"accepted": _int(accepted), "next": _int(following, torch.int64)}
