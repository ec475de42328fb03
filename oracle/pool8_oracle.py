"""Plain float64 restatements of the 8-bit pool and of attention behind a sliding window (CPU; test infrastructure only)."""
import math

import torch


def e4m3_values():
    """The finite values of OCP e4m3 by byte 0..126, from the format's definition: 4 exponent bits of bias 7, 3 mantissa bits."""
    out = []
    for byte in range(127):
        e, m = byte >> 3, byte & 7
        out.append((m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def round_e4m3(x):
    """Nearest e4m3 value of float64 |x| <= 448, ties to the even byte."""
    v = e4m3_values()
    a = x.abs()
    hi = torch.searchsorted(v, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    d_lo, d_hi = a - v[lo], v[hi] - a
    up = (d_hi < d_lo) | ((d_hi == d_lo) & (hi % 2 == 0))
    return torch.where(up, v[hi], v[lo]) * torch.where(torch.signbit(x), -1.0, 1.0).double()


def quantise(x):
    """(e4m3 values as float64, exponent + 127) of rows [.., head_dim]: the least e with max |x| <= 448 * 2^e, at least -126."""
    x = x.double()
    fin = torch.isfinite(x)
    amax = torch.where(fin, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(amax.shape, -126, dtype=torch.int64)
    for k in range(-126, 130):
        e = torch.where(amax > 448.0 * 2.0 ** k, torch.full_like(e, k + 1), e)
    q = round_e4m3(torch.where(fin, x / torch.pow(2.0, e.double())[..., None], torch.zeros_like(x)))
    return torch.where(fin, q, torch.full_like(q, math.nan)), e + 127


def visible_positions(n, window, sinks):
    """Positions that the last of n tokens sees (window None: all)."""
    j = torch.arange(max(n, 0))
    return j if window is None else j[(j >= n - window) | (j < sinks)]


def decode(q, k, v, table, b_req, b_len, window=None, sinks=0, num_slots=None):
    """(o, lse, tolerance of o, tolerance of lse) in float64 for k, v [slots, Hkv, D] given as the values they stand for.  Table entries outside
    [0, num_slots) do not exist.

    The tolerances are worst cases of a float32 computation (eps = 2^-24, half a step): a score is a sum of D products, off by at most (D + 8) eps
    of the sum of their magnitudes S (the softmax scale, the token's scale and the exponent's argument among the 8); that
    is the relative error of exp(s), once for the numerator and once for the sum; exp2 itself and the parts that P is kept in
    (2^-22) add 8 eps; a sum of n weights in blocks of 32 tokens adds at most (n / 32 + 40) eps twice."""
    B, Hq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    num_slots = k.shape[0] if num_slots is None else num_slots
    o = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros(B, Hq, 1, dtype=torch.float64), torch.zeros(B, Hq, dtype=torch.float64)
    eps = 2.0 ** -24
    for b in range(B):
        slots = table[int(b_req[b]), visible_positions(int(b_len[b]), window, sinks)].long()
        slots = slots[(slots >= 0) & (slots < num_slots)]
        if len(slots) == 0:
            continue
        kk, vv = k[slots].double().repeat_interleave(G, 1), v[slots].double().repeat_interleave(G, 1)  # [n, Hq, D]
        qq = q[b].double()
        s = torch.einsum("hd,nhd->hn", qq, kk) / math.sqrt(D)
        size = torch.einsum("hd,nhd->hn", qq.abs(), kk.abs()).amax(-1) / math.sqrt(D)
        lse[b] = torch.logsumexp(s, -1)
        o[b] = torch.einsum("hn,nhd->hd", torch.exp(s - lse[b][:, None]), vv)
        n = len(slots)
        rel = 2 * ((D + 8) * eps * size + 8 * eps + (n / 32 + 40) * eps)
        tol_o[b, :, 0] = rel * vv.abs().amax((0, 2))
        tol_l[b] = rel + 8 * eps * lse[b].abs()
    return o, lse, tol_o, tol_l


def prefill(q, k, v, q_len, q_first, k_len, k_first, peers, window, sinks):
    """(o, lse, tolerance of o before its rounding, tolerance of lse): a step for one sequence: query m at position q_first + m * peers sees key n at kpos = k_first + n * peers iff
    kpos <= qpos and (kpos > qpos - window or kpos < sinks).  P is kept in fp16 for the product with V (2^-11 of each weight at most); the rest as in decode()."""
    D, G = q.shape[-1], q.shape[1] // k.shape[1]
    qp = q_first + torch.arange(q_len) * peers
    kp = k_first + torch.arange(k_len) * peers
    seen = (kp[None] <= qp[:, None]) & ((kp[None] > qp[:, None] - window) | (kp[None] < sinks))
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("mhd,nhd->mhn", q.double(), kk) / math.sqrt(D)
    size = torch.einsum("mhd,nhd->mhn", q.double().abs(), kk.abs()) / math.sqrt(D)
    s = s.masked_fill(~seen[:, None], -math.inf)
    size = torch.where(seen[:, None].expand_as(size), size, torch.zeros_like(size))
    if k_len == 0:
        return (torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64),
                torch.zeros(*q.shape[:2], 1, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))[..., None])
    o = torch.einsum("mhn,nhd->mhd", p, vv)
    eps = 2.0 ** -24
    rel = 2 * ((D + 8) * eps * size.amax(-1) + 8 * eps + (k_len / 32 + 40) * eps)
    weight = torch.einsum("mhn,nhd->mhd", p, vv.abs()).amax(-1)
    return o, lse, ((rel + 2.0 ** -11) * weight)[..., None], rel + 8 * eps * lse.abs().nan_to_num(0, 0, 0)
