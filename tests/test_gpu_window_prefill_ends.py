"""The prefill step behind a window at its ends: one key that outweighs thousands, no keys at all, every request of a full launch."""
import math

import numpy as np
import pytest
import torch

from oracle import pool8_oracle as orc
from tests.test_gpu_window_prefill import DT, Step, _rows, _vec, rows  # noqa: F401 (a fixture: both shapes of 128-wide heads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,D,q_len", [(4, 2, 128, 40), (2, 2, 64, 33), (2, 1, 32, 20), (3, 3, 16, 17), (32, 32, 128, 1200)])
def test_a_first_key_that_outweighs_the_others(lsa, rows, dtype, Hq, Hkv, D, q_len):
    """A sink whose score lies 20 to 22 binary orders above those of 4000 others, which are alike: their weights keep 11 bits each (the oracle's
    tolerance), whatever share of a row they make up.  V is 0 at the sink, so that nothing hides them."""
    n = 4000 + q_len
    for bits in (20.03, 22.03):
        s = Step([(q_len, 4000, n, 0)], Hq, Hkv, D, DT[dtype], seed=31)
        ks = s.k_start[0]
        s.q.zero_(), s.kv[ks:ks + n, :Hkv].zero_()
        s.q[..., 0] = 16.0
        s.kv[ks, :Hkv, 0] = bits * math.log(2) * math.sqrt(D) / 16.0
        s.kv[ks, Hkv:] = 0
        s.kv[ks + 1:ks + n, Hkv:] = s.kv[ks + 1:ks + n, Hkv:].abs() + 0.5
        got = s.run(lsa, 5000, 1, o_dtype=torch.float32)
        q0, m = s.q_start[0], min(q_len, 64)  # (float64 over the first rows)
        want, lse, tol_o, tol_l = orc.prefill(s.q[q0:q0 + m], s.kv[ks:ks + n, :Hkv], s.kv[ks:ks + n, Hkv:], m, 4000, n, 0, 1, 5000, 1)
        assert ((got[0][q0:q0 + m].cpu().double() - want).abs() <= tol_o).all(), ((got[0][q0:q0 + m].cpu().double() - want).abs() / tol_o).max()
        assert ((got[1][q0:q0 + m].cpu().double() - lse).abs() <= tol_l).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("o_dtype", [None, torch.float32])
def test_no_keys_at_all(lsa, rows, dtype, D, o_dtype):
    """K and V without rows, as an instance of a ring has them whose part of a prompt is empty: the empty partial, on the rows that requests name."""
    s = Step([(70, 9, 0, 0), (0, 0, 0, 0), (3, 500, 0, 0)], 4, 2, D, DT[dtype], seed=33)
    none = s.kv[:0].cuda()
    s.check(s.run(lsa, 20, 2, o_dtype=o_dtype, kv=none), 20, 2)
    s.check(s.run(lsa, 20, 2, o_dtype=o_dtype, kv=none, lse=False, total_q_len=73), 20, 2)
    with pytest.raises(ValueError, match="window"):
        s.run(lsa, 0, 2, kv=none)


@pytest.mark.gpu
def test_an_empty_partial_joins(lsa):
    s = Step([(40, 60, 100, 0)], 4, 2, 128, torch.float16, seed=34)
    o, l = s.run(lsa, 50, 3, o_dtype=torch.float32)
    o0, l0 = s.run(lsa, 50, 3, o_dtype=torch.float32, kv=s.kv[:0].cuda())
    q0 = s.q_start[0]
    got = lsa.lse_merge([(o0[q0:].contiguous(), l0[q0:].contiguous()), (o[q0:].contiguous(), l[q0:].contiguous())])
    assert torch.equal(got[0], o[q0:]) and torch.equal(got[1], l[q0:])


@pytest.mark.gpu
def test_lengths_and_windows_as_numpy_integers(lsa):
    """What a scheduler that keeps its lengths in numpy passes."""
    s = Step([(40, 60, 100, 0), (9, 0, 9, 0)], 4, 2, 128, torch.float16, seed=35)
    n = np.int64
    for total in (None, n(49)):
        got = s.run(lsa, n(50), np.int32(3), total_q_len=total)
        s.check(got, 50, 3)
    o = torch.zeros(s.q.shape, dtype=torch.float16, device="cuda")
    q, kv, v = s.q.cuda(), s.kv.cuda(), [_vec(s.q_start), _vec([40, 9]), _vec([60, 0]), _vec(s.k_start), _vec([100, 9]), _vec([0, 0])]
    lsa.window_attention_fwd(q, kv[:, :2], kv[:, 2:], o, *v, n(1), n(40), n(50), n(3))
    q0 = s.q_start[0]
    assert torch.equal(o[q0:q0 + 40], got[0][q0:q0 + 40])
    with pytest.raises(ValueError, match="window"):
        s.run(lsa, n(0), 2)
    with pytest.raises(TypeError):
        s.run(lsa, 4.5, 2)


def _step64(q, k, v, qp, kp, window, sinks):
    """(o, lse, mean of |v|, largest sum of a score's magnitudes) in float64 on the GPU: queries at positions qp, keys at kp."""
    G = q.shape[1] // k.shape[1]
    qd, kd, vd = (t.cuda().double().transpose(0, 1).contiguous() for t in (q, k, v))  # [heads, rows, D]
    kd, vd = kd.repeat_interleave(G, 0), vd.repeat_interleave(G, 0)
    qp, kp = qp.cuda()[:, None], kp.cuda()[None]
    unseen = ~((kp <= qp) & ((kp > qp - window) | (kp < sinks)))
    kt = kd.transpose(1, 2).contiguous()
    s = (torch.matmul(qd, kt) / math.sqrt(q.shape[2])).masked_fill(unseen, -math.inf)
    size = (torch.matmul(qd.abs(), kt.abs()) / math.sqrt(q.shape[2])).masked_fill(unseen, 0.0).amax(-1)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    o, mean = torch.matmul(p, vd), torch.matmul(p, vd.abs()).amax(-1)
    return o.transpose(0, 1).cpu(), lse.T.cpu(), mean.T.cpu()[..., None], size.T.cpu()[..., None]


EPS = 2.0 ** -24


def _rel(D, n, size):
    """As in the oracle: float32 sums of D products and of n weights in blocks of 32, twice."""
    return 2 * ((D + 8) * EPS * size + 8 * EPS + (n / 32 + 40) * EPS)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,D,lens", [(32, 8, 128, [700, 333, 900]), (32, 32, 128, [400, 400]), (32, 4, 64, [900, 1000])])
def test_every_request_of_a_launch_that_fills_the_chip(lsa, rows, dtype, Hq, Hkv, D, lens):
    """Many workgroups, 32 positions per wave, the requests in bunches or one after the other: all of them against float64."""
    s = Step([(n, 0, n, 0) for n in lens] * (8 if D == 128 else 5), Hq, Hkv, D, DT[dtype], seed=36)
    half = 2.0 ** -11 if s.dtype == torch.float16 else 2.0 ** -8
    for window, sinks in ((128, 4), (250, 0)):
        got = [t.cpu().double() for t in s.run(lsa, window, sinks)]
        for (n, _, _, _), qs, ks in zip(s.seqs, s.q_start, s.k_start):
            kv = s.kv[ks:ks + n]
            o, lse, mean, size = _step64(s.q[qs:qs + n], kv[:, :Hkv], kv[:, Hkv:], torch.arange(n), torch.arange(n), window, sinks)
            rel = _rel(D, n, size)
            tol = (rel + 2.0 ** -11) * mean
            assert ((got[0][qs:qs + n] - o).abs() <= tol + half * (o.abs() + tol) + 2.0 ** -24).all()
            assert ((got[1][qs:qs + n] - lse).abs() <= rel[..., 0] + 8 * EPS * lse.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,P,W,S", [(300, 3, 70, 8), (1000, 2, 333, 0), (500, 4, 1, 5)])
def test_striped_chunks_join_row_by_row(lsa, rows, dtype, n, P, W, S):
    """P instances hold every P-th token; one instance's partials over all chunks, merged, against the step over all keys, each row by its own bound: a
    partial's weight is exp of its log-sum-exp, off by a partial's tolerance in the numerator and in the sum."""
    q, kv = _rows((n, 4, 128), 1, DT[dtype]), _rows((n, 4, 128), 2, DT[dtype])
    for mine in range(P):
        qs = q[mine::P].contiguous()
        o, lse, mean, size = _step64(qs, kv[:, :2], kv[:, 2:], torch.arange(mine, n, P), torch.arange(n), W, S)
        parts = []
        for r in range(P):
            rows_r = kv[r::P].contiguous().cuda()
            po, pl = torch.empty(qs.shape, device="cuda"), torch.empty(qs.shape[:2], device="cuda")
            lsa.window_attention_fwd(qs.cuda(), rows_r[:, :2], rows_r[:, 2:], po, _vec([0]), _vec([len(qs)]), _vec([mine]), _vec([0]), _vec([len(rows_r)]),
                                     _vec([r]), P, len(qs), W, S, lse=pl)
            parts.append((po, pl))
        got = [t.cpu().double() for t in lsa.lse_merge(parts)]
        rel = _rel(128, n, size)
        of_a_part = rel + 8 * EPS * (size + math.log(n)) + 16 * EPS
        assert ((got[0] - o).abs() <= (rel + 2.0 ** -11 + 2 * of_a_part) * mean + 2.0 ** -24).all()
        assert ((got[1] - lse).abs() <= of_a_part[..., 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("o_dtype", [None, torch.float32])
@pytest.mark.parametrize("lens", [[130, 301], [1700, 900]])
def test_outputs_and_queries_inside_wider_rows(lsa, rows, dtype, D, o_dtype, lens):
    """q and o as slices of wider rows and heads: the same bits as packed, nothing written beside them."""
    Hq, Hkv = 16, 4
    s = Step([(n, 0, n, 0) for n in lens], Hq, Hkv, D, DT[dtype], seed=41)
    want = s.run(lsa, 90, 3, o_dtype=o_dtype)
    n = s.q.shape[0]
    wide_q = torch.full((n, Hq + 5, D + 16), 3.0, dtype=s.dtype, device="cuda")
    wide_q[:, 2:2 + Hq, 8:8 + D] = s.q.cuda()
    wide_o = torch.full((n, Hq + 3, D + 8), 7.0, dtype=o_dtype or s.dtype, device="cuda")
    o, l = wide_o[:, 1:1 + Hq, 8:], torch.full((n, Hq), 7.0, device="cuda")
    col = lambda i: _vec([t[i] for t in s.seqs])  # noqa: E731
    kv = s.kv.cuda()
    lsa.window_attention_fwd(wide_q[:, 2:2 + Hq, 8:8 + D], kv[:, :Hkv], kv[:, Hkv:], o, _vec(s.q_start), col(0), col(1), _vec(s.k_start), col(2), col(3), 1, max(lens), 90, 3,
                             lse=l)
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    wide_o[:, 1:1 + Hq, 8:] = 7.0
    assert (wide_o == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_padded_batch_of_many_requests(lsa, rows, D):
    """Three hundred requests, most of them without rows."""
    r = torch.Generator().manual_seed(42)
    lens = [int(torch.randint(1, 90, (1,), generator=r)) if i % 7 == 3 else 0 for i in range(300)]
    s = Step([(n, i % 40, n + i % 40, 0) if n else (0, 0, i % 5, 0) for i, n in enumerate(lens)], 4, 2, D, torch.float16, seed=43)
    s.check(s.run(lsa, 33, 4), 33, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_past_four_gigabytes(lsa, rows, dtype):
    """K/V rows more than 2^33 bytes, q and o rows more than 2^32 bytes behind the first."""
    Hq, Hkv, D, nq, nk, n = 32, 8, 128, 600000, 2200000, 333
    q, kv = (torch.empty(m, h, D, dtype=DT[dtype], device="cuda") for m, h in ((nq, Hq), (nk, 2 * Hkv)))
    o, l = torch.full((nq, Hq, D), 7.0, dtype=DT[dtype], device="cuda"), torch.full((nq, Hq), 7.0, device="cuda")
    qs, kvs = _rows((n, Hq, D), 5, DT[dtype]), _rows((n, 2 * Hkv, D), 6, DT[dtype])
    q[nq - n:], kv[nk - n:] = qs.cuda(), kvs.cuda()
    lsa.window_attention_fwd(q, kv[:, :Hkv], kv[:, Hkv:], o, _vec([nq - n]), _vec([n]), _vec([0]), _vec([nk - n]), _vec([n]), _vec([0]), 1, n, 100, 2, lse=l)
    want, lse, mean, size = _step64(qs, kvs[:, :Hkv], kvs[:, Hkv:], torch.arange(n), torch.arange(n), 100, 2)
    rel = _rel(D, n, size)
    tol = (rel + 2.0 ** -11) * mean
    half = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
    assert ((o[nq - n:].cpu().double() - want).abs() <= tol + half * (want.abs() + tol) + 2.0 ** -24).all()
    assert ((l[nq - n:].cpu().double() - lse).abs() <= rel[..., 0] + 8 * EPS * lse.abs()).all()
    assert (o[:nq - n:997] == 7).all() and (o[nq - n - 400:nq - n] == 7).all() and (l[:nq - n] == 7).all()
