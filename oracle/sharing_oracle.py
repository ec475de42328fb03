"""Plain restatements of attention over shared prefixes (float64) and of forks, releases and compaction of a pool (CPU; test infrastructure only)."""
import math

import torch

EPS32 = 2.0 ** -24
# what a weight of the prefix may be off by, relative to itself: rounded to fp16, or kept in two parts of bfloat16 (the second rounded)
EPS_P = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -16}
EPS_OUT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attend(q, k, v, eps_p):
    """(o, lse, tolerance of o before its rounding, tolerance of lse) of rows q [m, Hq, D] that all see k, v [n, Hkv, D].

    The tolerances are worst cases (eps = 2^-24, half a step of float32): a score is a sum of D products, off by at most (D + 8) eps of the sum of their magnitudes
    (scale, difference and the exponent's argument among the 8), which is the relative error of exp(s), once for the numerator and once for the sum; exp2 adds 8 eps; a
    sum of n weights in blocks of 32 adds at most (n / 32 + 40) eps twice, and joining up to 2048 partials (2048 + 40) eps less than that per partial, counted as 64 eps more.
    A weight held in fewer bits is off by eps_p of itself, in the numerator and in the sum that divides it; below fp16's normal range (2^-14, where the largest is 2^9 or more) by
    2^-25, n of them by n 2^-34 of the sum."""
    m, Hq, D = q.shape
    n, G = k.shape[0], Hq // k.shape[1]
    if n == 0:
        return (torch.zeros(q.shape, dtype=torch.float64), torch.full((m, Hq), -math.inf, dtype=torch.float64), torch.zeros(m, Hq, 1, dtype=torch.float64),
                torch.zeros(m, Hq, dtype=torch.float64))
    kk, vv, qq = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1), q.double()
    s = torch.einsum("mhd,nhd->mhn", qq, kk) / math.sqrt(D)
    size = torch.einsum("mhd,nhd->mhn", qq.abs(), kk.abs()).amax(-1) / math.sqrt(D)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    o = torch.einsum("mhn,nhd->mhd", p, vv)
    weight = torch.einsum("mhn,nhd->mhd", p, vv.abs()).amax(-1)
    rel = 2 * ((D + 8) * EPS32 * size + 8 * EPS32 + (n / 32 + 104) * EPS32)
    tol = rel * vv.abs().amax((0, 2))[None] + 2 * eps_p * weight + n * 2.0 ** -34 * vv.abs().amax((0, 2))[None]
    return o, lse, tol[..., None], rel + 8 * EPS32 * lse.abs()


def members(g_start, g_size, g_req, g_prefix, rows, num_reqs, most):
    """(group or -1, prefix) of every row: groups in order, the first that names a row has it."""
    owner = [-1] * rows
    end = 0
    for g, (s, n) in enumerate(zip(g_start, g_size)):
        s = min(max(s, 0), rows)
        e = min(s + max(n, 0), rows)
        for b in range(max(s, end), e):
            owner[b] = g
        end = max(end, e)
    prefix = [0 if g < 0 or not 0 <= g_req[g] < num_reqs else min(max(g_prefix[g], 0), most) for g in owner]
    return owner, prefix


def valid(slots, num_slots):
    slots = slots.long()
    return slots[(slots >= 0) & (slots < num_slots)]


def decode(q, k, v, table, b_req, b_len, g_start, g_size, g_req, g_prefix, max_prefix, out_dtype):
    """(o, lse, tolerances) of every request: its group's prefix, then its own row behind it."""
    R, S = table.shape
    owner, prefix = members(g_start, g_size, g_req, g_prefix, len(b_req), R, min(max_prefix, S))
    parts = []
    for b in range(len(b_req)):
        n = min(max(int(b_len[b]), 0), S) if 0 <= int(b_req[b]) < R else 0
        p = prefix[b] if prefix[b] <= n else 0
        slots = table.new_zeros(0) if n == 0 else table[int(b_req[b]), p:n]
        if p:
            slots = torch.cat([table[g_req[owner[b]], :p], slots])
        slots = valid(slots, k.shape[0])
        parts.append(attend(q[b:b + 1], k[slots], v[slots], EPS_P[q.dtype]))
    o, lse, to, tl = (torch.cat(x) for x in zip(*parts))
    return o, lse, to + EPS_OUT[out_dtype] * (o.abs() + to) + 2.0 ** -25, tl


def prompt(q, k, v, table, g_start, g_size, g_req, g_prefix, max_prefix, eps_p):
    """(o, lse, tolerances, which rows see a key) of the step from the empty state; rows of no group have lse = -inf."""
    R, S = table.shape
    owner, prefix = members(g_start, g_size, g_req, g_prefix, len(q), R, min(max_prefix, S))
    o, lse, to, tl = attend(q, k[:0], v[:0], eps_p)
    for g in set(owner) - {-1}:
        rows = torch.tensor([b for b in range(len(q)) if owner[b] == g])
        slots = valid(table[g_req[g], :prefix[rows[0]]], k.shape[0]) if prefix[rows[0]] else table.new_zeros(0).long()
        o[rows], lse[rows], to[rows], tl[rows] = attend(q[rows], k[slots], v[slots], eps_p)
    return o, lse, to, tl


def fork(table, src, dst, lens, most, state=None):
    """(table, state): entries as they are and a reference on each slot; no slot (2147483647) where the source is no row of the table, or the slot is free."""
    table, state = table.clone(), None if state is None else state.clone()
    old, held = table.clone(), None if state is None else state.clone()
    for a, b, n in zip(src, dst, lens):
        n = min(n, most, table.shape[1])
        if not 0 <= b < len(table) or n <= 0:
            continue
        row = old[a, :n].clone() if 0 <= a < len(table) else torch.full((n,), 2147483647, dtype=table.dtype)
        if state is not None:
            inside = (row >= 0) & (row < len(state))
            row[inside & (held[row.clamp(0, len(state) - 1).long()] == 0)] = 2147483647
            for s in row.tolist():
                if 0 <= s < len(state):
                    state[s] += 1
        table[b, :n] = row
    return table, state


def release(table, req, lens, most, state):
    """(state, freed, wrong)"""
    state = state.clone()
    freed = wrong = 0
    for r, n in zip(req, lens):
        for s in table[r, :min(n, most, table.shape[1])].tolist() if 0 <= r < len(table) else [-1] * min(n, most, table.shape[1]):
            if not 0 <= s < len(state) or state[s] <= 0:
                wrong += 1
                continue
            state[s] -= 1
            freed += int(state[s] == 0)
    return state, freed, wrong


def compact(state, table, req, lens, most):
    """(state, table, remap, sources, holes)"""
    state, table = state.clone(), table.clone()
    values = state.tolist()
    used = [i for i, n in enumerate(values) if n != 0]
    U = len(used)
    source = [i for i in used if i >= U]
    hole = [i for i in range(U) if values[i] == 0]
    remap = torch.full((len(state),), -1, dtype=torch.int32)
    remap[used] = torch.tensor(used, dtype=torch.int32)
    for a, b in zip(source, hole):
        values[b], values[a] = values[a], 0
    remap[source] = torch.tensor(hole, dtype=torch.int32)[:len(source)]
    state = torch.tensor(values, dtype=torch.int32)
    for r, n in zip(req, lens):
        for i in range(min(n, most, table.shape[1])):
            s = int(table[r, i])
            if 0 <= s < len(state) and remap[s] >= 0:
                table[r, i] = remap[s]
    return state, table, remap, source, hole
