"""Plain 64-bit forms of the paged-cache operators and of the draft verification (test infrastructure), with the bounds their
results may be off by."""
import math

import numpy as np
import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}        # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}                               # half of the smallest step
TOP4 = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0 ** 127}                          # largest value with four significant bits


def e4m3_values():
    """The 256 codes' values, from the format: 4 bits of exponent (bias 7), 3 of mantissa, no infinities."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if c & 127 == 127 else (m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out[c] = -v if c & 128 else v
    return torch.from_numpy(out)


def row_scale_byte(rows, dtype):
    """rows float64 [..., D] -> exponent byte: smallest x >= 1 with max finite magnitude (at most TOP4) / 2^(x - 127) <= 448."""
    a = torch.where(rows.isfinite(), rows.abs().clamp(max=TOP4[dtype]), 0.0).amax(-1)
    byte = torch.ones(a.shape, dtype=torch.int64)
    for x in range(1, 255):
        byte = torch.where(a > 448.0 * 2.0 ** (x - 127), torch.tensor(x + 1), byte)
    return byte


def decode(codes, byte):
    """codes uint8 [..., D], byte uint8 [...] -> float64."""
    return e4m3_values()[codes.long()] * torch.exp2(byte.double() - 127.0)[..., None]


def stored(pages, scales, table_row, positions):
    """float64 [H_kv, n, D]: rows `positions` of one sequence (all on the CPU)."""
    p = pages.shape[2]
    page, at = table_row[positions // p].long(), positions % p
    if scales is None:
        return pages[page, :, at].double().transpose(0, 1)
    return decode(pages.view(torch.uint8)[page, :, at], scales[page, :, at]).transpose(0, 1)


def rope(x, cos, sin):
    """x [n, heads, D], cos / sin [n, D], float64."""
    half = x.shape[-1] // 2
    c, s = cos[:, None], sin[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]), dim=-1)


def attention(q, k, v, past, scale, dtype):
    """q [H, n, D], k / v [H_kv, past + n, D] float64 -> (o [n, H, D], bound): row i sees keys [0, past + i].

    The bound, element by element (u = half a step of the element type, e = 2^-24, w_j the softmax weights):
      the output's rounding                          u |o|
      the weights' rounding for the second product   u sum w_j |v_j|, and below the type's normal range TINY each
      where the sum is taken of the rounded weights, sum w_j (1 + a_j) v_j / sum w_j (1 + a_j) with |a_j| <= u is off by
      sum w_j a_j (v_j - o) / sum w_j (1 + a_j): u |o| more, and TINY |o| each
      a score's fp32 sum of D exact products and its scaling, an exponential of 2 units in the last place, the exponent's own
      subtraction: each weight off by a factor 1 + d, d = 2 (D + 4) e scale sum |q_i k_ij| + 4 e |s| + 4 e; numerator and denominator
      fp32 sums over n keys (in blocks, but at worst) 2 (n + 8) e sum w_j |v_j|"""
    h, n, d = q.shape
    group = h // k.shape[0]
    kk, vv = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    hidden = torch.arange(kk.shape[1])[None, :] > past + torch.arange(n)[:, None]
    s = torch.matmul(q, kk.transpose(1, 2).contiguous()) * scale
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    w = w / total
    vz, va = vv, vv.abs()
    o = torch.matmul(w, vz)
    e = 2.0 ** -24
    mag = torch.matmul(q.abs(), kk.abs().transpose(1, 2).contiguous()).masked_fill(hidden, 0.0) * scale
    off = (2 * (d + 4) * e * mag + 4 * e * s.masked_fill(hidden, 0.0).abs()).amax(-1, keepdim=True) + 4 * e
    wv = torch.matmul(w, va)
    u = EPS[dtype]
    keys = kk.shape[1]
    bound = 2 * u * o.abs() * (1 + 2 * u) + (u + 2 * off + 2 * (keys + 8) * e) * wv * (1 + 2 * u) + TINY[dtype]
    seen = (~hidden).double().expand_as(w)
    bound = bound + TINY[dtype] * (torch.matmul(seen, va) + seen.sum(-1, keepdim=True) * o.abs()) / total
    return o.transpose(0, 1), bound.transpose(0, 1)


def verify(target, draft, tokens, cu, u_accept, u_next, temps):
    """One sequence after the other, float64; lists in, (accepted, next) out, and the narrowest margin any outcome had."""
    accepted, following, margin = [], [], math.inf
    target, draft = target.double(), draft.double()
    vocab = target.shape[1]

    def dist(row, t):
        if row.isnan().any() or (row == math.inf).any() or (row == -math.inf).all():
            return torch.full_like(row, math.nan)
        if t == 0:
            d = torch.zeros_like(row)
            d[int(torch.nonzero(row == row.max())[0, 0])] = 1.0
            return d
        return torch.softmax(row / t, dim=0)

    for b in range(len(cu) - 1):
        n, t, k, rest = cu[b + 1] - cu[b], temps[b], 0, None
        while k < n:
            p, tok = dist(target[cu[b] + b + k], t), tokens[cu[b] + k]
            inside = 0 <= tok < vocab
            if t == 0:
                ok = inside and float(p[tok]) > 0
            else:
                q = dist(draft[cu[b] + k], t)
                lhs, rhs = (u_accept[cu[b] + k] * float(q[tok]), float(p[tok])) if inside else (0.0, 0.0)
                ok = lhs < rhs
                if inside and lhs == lhs and rhs == rhs and max(lhs, rhs) > 0:
                    margin = min(margin, abs(lhs - rhs) / max(lhs, rhs))
            if not ok:
                rest = p
                if t > 0:
                    r = torch.where(p - q < 0, torch.zeros_like(p), p - q)
                    rest = p if float(r.sum()) == 0 else r
                break
            k += 1
        if rest is None:
            rest = dist(target[cu[b] + b + n], t)
        accepted.append(k)
        mass = torch.cumsum(rest, 0)
        if not float(mass[-1]) > 0:
            following.append(-1)
            continue
        goal = u_next[b] * float(mass[-1])
        hit = torch.nonzero(mass > goal)
        following.append(int(hit[0, 0]) if len(hit) else int(torch.nonzero(rest > 0)[-1, 0]))
        margin = min(margin, float((mass - goal).abs().min() / mass[-1]) if goal > 0 else margin)
    return accepted, following, margin
